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


def test_values_cross_lanes_in_order():
    """Single tokens: a wave's lanes write a tile's values into LDS, others of its lanes read them by columns, and the next tile is written.  Between each
    two of these stands what orders them.  Likewise the marks of spoiled keys of a chunk's tile, cleared by some lanes and set by others."""
    loop = body("tl_paged_few")
    loop = loop[loop.index("for (int t = first_tile;"):loop.index("// ---- the waves meet")]
    written, read = loop.rindex("reinterpret_cast<u32x4*>(own"), loop.index("column_read(")
    assert "wave_exchange();" in loop[written:read] and "wave_exchange();" in loop[loop.rindex("column_read("):]
    put = body("tl_paged_rows")
    put = put[put.index("auto put = "):]
    cleared = put.index("spoiled[buf][wave * KW + lane] = 0;")
    assert "wave_exchange();" in put[cleared:put.index("] = 1;")]
    exchange = body("wave_exchange")
    assert '__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront")' in exchange and "__builtin_amdgcn_wave_barrier()" in exchange


def instructions(name):
    """The instructions of the one asm statement of a function."""
    statements = re.findall(r'asm volatile\(((?:\s*"(?:[^"\\]|\\.)*")+)', body(name))
    assert len(statements) == 1
    text = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', statements[0]))
    return [i.strip() for i in re.split(r"\\n|\\t", text) if i.strip() and not i.endswith(":")]


def wait_states(lines):
    """An instruction is one, s_nop n is n + 1."""
    return sum(int(i.split()[1]) + 1 if i.startswith("s_nop") else 1 for i in lines)


def test_loads_written_as_assembly_wait_for_their_scalars():
    """A memory instruction may read a scalar register five wait states after a vector instruction wrote it, m0 one after a move."""
    lines = instructions("buffer_to_lds")
    load = next(i for i, line in enumerate(lines) if line.startswith("buffer_load"))
    assert wait_states(lines[:load]) >= 5
    moved = next(i for i, line in enumerate(lines) if "m0" in line)
    assert wait_states(lines[moved + 1:load]) >= 1


def test_sums_scaled_in_assembly_wait_for_their_products():
    """A vector instruction may read what a matrix product wrote 19 wait states after the longest of them, and a product what a vector instruction
    wrote two after it."""
    lines = instructions("scale_if")
    branch = next(i for i, line in enumerate(lines) if line.startswith("s_cbranch"))
    scaled = [i for i, line in enumerate(lines) if line.startswith("v_")]
    assert wait_states(lines[branch + 1:scaled[0]]) >= 19 and wait_states(lines[scaled[-1] + 1:]) >= 2
