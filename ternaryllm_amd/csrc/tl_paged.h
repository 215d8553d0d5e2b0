// What the kernels of a paged cache share: the batch and the pages as kernels take them, where a row of a batch lies, and
// the checks in front of a launch.
#pragma once
#include <initializer_list>

#include "tl_device.h"
#include "tl_rope.h"

namespace tl {

struct Pages {
    void *k, *v;
    unsigned char *k_exp, *v_exp;           // null: fp16
    long long page_stride, head_stride, slot_stride;
    unsigned pages;
    int shift, kv_heads, hd;                // 1 << shift slots to a page
};

struct Batch {
    const int *table, *starts, *lengths;
    long long table_stride;
    int table_pages, seqs, tokens;
};

// Where a row of the batch belongs: its sequence (-1: none) and its index there (negative where the sequence is said to be
// shorter than its rows), and how long that is.
struct Place {
    int seq, index, length;
};

// By a whole wave, for one row that is the same in all lanes: 64 starts are compared at a time.
__device__ __forceinline__ Place place_of(const Batch& b, int token)
{
    const int lane = (int)(threadIdx.x & 63u);
    int below = 0;                                              // starts that are not behind the row
    for (int first = 0; first <= b.seqs; first += 64) {
        const int i = first + lane;
        const int more = __popcll(__builtin_amdgcn_ballot_w64(i <= b.seqs && b.starts[min(i, b.seqs)] <= token));
        below += more;
        if (more < 64) break;
    }
    const int seq = below - 1;
    if (seq < 0 || seq >= b.seqs) return Place{-1, 0, 0};
    const int length = b.lengths[seq];
    return Place{seq, length - b.starts[seq + 1] + token, length};
}

// Page and slot of a token of a sequence; page -1: the table has none that is a page, or does not hold the sequence.
struct Slot {
    int page, slot;
};

__device__ __forceinline__ Slot slot_of(const Pages& p, const Batch& b, const Place& at)
{
    const int column = at.index >> p.shift;
    if (at.seq < 0 || at.index < 0 || column >= b.table_pages || at.length > b.table_pages << p.shift) return Slot{-1, 0};
    const int page = b.table[at.seq * b.table_stride + column];
    return Slot{(unsigned)page < p.pages ? page : -1, at.index & ((1 << p.shift) - 1)};
}

// Host: whether an address and strides (of elements of `es` bytes) are whole 16-byte pieces.
inline bool in_pieces(const void* p, std::initializer_list<int64_t> strides, int64_t es)
{
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
    for (int64_t s : strides)
        if (s * es % 16) return false;
    return true;
}

// Host: launches of at most 2^23 workgroups that make up `groups`, each told its first.  (A launch has fewer than 2^32 threads; of more, the excess over
// 2^32 would run, without an error.)
template <typename F>
void in_launches(int64_t groups, F launch)
{
    constexpr int64_t kMost = 1 << 23;
    for (int64_t first = 0; first < groups; first += kMost) launch((int)first, dim3((unsigned)std::min(groups - first, kMost)));
}

// Host: the caller's pages and batch as the kernels take them, or an error.
int take_pages(const tl_pages* pages, const tl_page_batch* batch, int64_t tokens, Pages* p, Batch* b);

}  // namespace tl
