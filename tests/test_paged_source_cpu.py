"""Rules of order between lanes that the paged attention's source has to ask for itself.  A breach need not show in what a compiler makes of it
today, and is not to be tried on a GPU: these tests read the source."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ternaryllm_amd", "csrc", "tl_paged.hip")


def body(name):
    """The text from a function's name on to the brace that ends it at the left margin."""
    with open(SOURCE) as f:
        text = f.read()
    at = re.search(r"\b%s\([^;{]*\)\n\{" % name, text)
    assert at, name
    return text[at.start():text.index("\n}\n", at.start())]


def test_the_walks_sums_have_one_writer():
    """Two stores under conditions of different lanes are in no order: a thread makes one of them at most."""
    assert len(re.findall(r"\bsums\[\w+\] = ", body("begin_walk"))) == 1
