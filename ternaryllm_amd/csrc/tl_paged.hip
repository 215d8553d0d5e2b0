// Causal softmax attention of a ragged batch's new tokens over everything their sequences have in the pages of a cache, on the
// matrix cores (the reference's eager matmul / softmax / matmul, ternaryLLM_GPU/TernaryLLM/TernaryAttn.py:100-113, for sequences of
// different lengths).
//
// The work is a list of units: a sequence's key head, and as many of its rows -- (token, query head of the group) pairs, tokens
// first -- as a workgroup holds.  A unit costs about as many steps as its last row sees keys.  The list's whole cost is cut into
// equal parts, one to a workgroup, whatever the lengths are: a part may end inside a unit, whose keys then are shared out among
// neighbouring workgroups.  What such a workgroup leaves are pieces (unnormalised sums, their maximum and sum of exponentials), which
// a second launch joins.  Every workgroup finds its part by itself from the lengths on the device: the host knows nothing of them,
// and a captured call serves any.
#include <climits>

#include "tl_matrix.h"
#include "tl_paged.h"

using namespace tl;

namespace {

constexpr int kRound = 64;                       // keys: units are cut at multiples
constexpr int kSeqsOfThread = 4;                 // of a pass over the lengths
constexpr float kNone = -__builtin_huge_valf();

// The unit that begins in a workgroup and goes on behind it: last is the workgroup that ends it, -1: none does.
struct Shared {
    int seq, head, tile, last;
};

struct PagedAttn {
    const __half* q;
    long long q_t, q_h;
    __half* out;
    Pages pages;
    Batch batch;
    int heads, group;
    int tile_heads, blocks, tile_tokens;         // query heads and tokens of a unit, units that a group's heads are shared out among
    float scale_log2;                            // of the scores, times log2(e)
    int fixed;                                   // cost of a unit beside its keys
    int least;                                   // cost of a workgroup's part, 1 or more
    int uncut;                                   // units go to one workgroup whole
    float* pieces;                               // [workgroups][2][rows][head_dim + 4]
    Shared* shared;                              // [workgroups]
};

__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long long scalar(long long v)
{
    return (long long)(((unsigned long long)(uint32_t)scalar((int)(v >> 32)) << 32) | (uint32_t)scalar((int)v));
}

// A sequence as the walk over the units takes it.
struct Seq {
    int start, n, length, tiles;
    int before;                                  // its keys that every row sees, 0 at least
    bool wrong;                                  // the table does not hold its length
};

__device__ __forceinline__ Seq sequence(const PagedAttn& a, int b)
{
    Seq s;
    s.start = a.batch.starts[b];
    const int end = min(a.batch.starts[b + 1], a.batch.tokens);
    s.n = s.start >= 0 ? max(end - s.start, 0) : 0;
    const int length = a.batch.lengths[b], room = a.batch.table_pages << a.pages.shift;
    s.wrong = length > room;
    s.length = min(max(length, 0), room);
    s.tiles = (s.n + a.tile_tokens - 1) / a.tile_tokens;
    s.before = max(s.length - s.n, 0);
    return s;
}

// The same for a sequence that all lanes look at.
__device__ __forceinline__ Seq scalar(Seq s)
{
    return Seq{scalar(s.start), scalar(s.n), scalar(s.length), scalar(s.tiles), scalar(s.before), scalar((int)s.wrong) != 0};
}

// Cost of a key head's first `tiles` units: unit i costs fixed + before + (i + 1) * tile_tokens.
__device__ __forceinline__ long long tiles_cost(const PagedAttn& a, int before, int tiles)
{
    return (long long)tiles * (a.fixed + before) + (long long)a.tile_tokens * tiles * (tiles + 1ll) / 2;
}

// The workgroup's part of the list, and where it stands in it.
struct Walk {
    int wg, wgs;                                 // this workgroup, and how many have a part
    long long total, from, to;                   // the part
    long long at;                                // where the present unit begins
    int b, head, tile;                           // the unit: sequence, key head and block of query heads, rows
    Seq s;
};

__device__ __forceinline__ long long unit_cost(const PagedAttn& a, const Walk& w) { return a.fixed + (long long)w.s.before + (w.tile + 1ll) * a.tile_tokens; }

// a * b / c rounded down, for a * b < 2^53 (exact then: a quotient below an integer by 1 / c at least does not round to it; a division of 64-bit
// integers takes several times as long).
__device__ __forceinline__ long long share_of(long long a, long long b, long long c) { return (long long)((double)(a * b) / (double)c); }

__device__ __forceinline__ bool next_unit(const PagedAttn& a, Walk& w, long long cost);

// By a whole workgroup of 256 threads.  False where it has no part.
__device__ __forceinline__ bool begin_walk(const PagedAttn& a, Walk& w)
{
    __shared__ long long sums[4];
    __shared__ long long found_at;
    __shared__ int found_b;
    __shared__ Seq found;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr int kPass = 256 * kSeqsOfThread;
    const int seqs = a.batch.seqs, heads = a.pages.kv_heads * a.blocks;
    Seq s[kSeqsOfThread];
    long long cost[kSeqsOfThread], upto = 0, total = 0, pass = 0;
    // this thread's sequences from `first` on, what they cost, and the sum of all before and of its own
    auto look = [&](int first) {
        long long own = 0;
#pragma unroll
        for (int i = 0; i < kSeqsOfThread; ++i) {
            const int b = first + tid * kSeqsOfThread + i;
            cost[i] = 0;
            if (b < seqs) {
                s[i] = sequence(a, b);
                cost[i] = tiles_cost(a, s[i].before, s[i].tiles) * heads;
            }
            own += cost[i];
        }
        upto = own;
        const bool one = seqs - first <= kSeqsOfThread;   // thread's
        if (!one) {
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const long long below = __shfl_up(upto, off, 64);
                if (lane >= off) upto += below;
            }
        }
        if (seqs > kPass) __syncthreads();       // the pass before is done with the sums
        if (one ? tid == 0 : lane == 63) sums[wave] = upto;   // (one writer each: of two, neither is the last)
        __syncthreads();
        pass = sums[0];
        if (seqs - first > 64 * kSeqsOfThread) {
#pragma unroll
            for (int i = 0; i < 4; ++i) upto += i < wave ? sums[i] : 0;
            pass += sums[1] + sums[2] + sums[3];
        }
    };
    for (int first = 0; first < seqs; first += kPass) {
        look(first);
        total += pass;
    }
    total = scalar(total);
    // as many parts as there are workgroups, but none of less than `least`; neighbours of the list stay in one part of the chip, whose
    // cache they share
    w.wgs = (int)min(share_of(total + a.least - 1, 1, a.least), (long long)gridDim.x);
    const int eighth = (w.wgs + 7) / 8, inside = (int)blockIdx.x / 8;
    w.wg = inside < eighth ? ((int)blockIdx.x & 7) * eighth + inside : (int)blockIdx.x;
    if (w.wg >= w.wgs) {
        if (tid == 0) a.shared[w.wg].last = -1;
        return false;
    }
    w.total = total;
    w.from = scalar(share_of(total, w.wg, w.wgs));
    w.to = scalar(share_of(total, w.wg + 1, w.wgs));
    long long below = 0;
    for (int first = 0;; first += kPass) {
        if (seqs > kPass) look(first);
        long long begins = below + upto;
#pragma unroll
        for (int i = kSeqsOfThread - 1; i >= 0; --i) {
            const long long ends = begins;
            begins -= cost[i];
            if (begins <= w.from && w.from < ends) found_b = first + tid * kSeqsOfThread + i, found_at = begins, found = s[i];
        }
        below += pass;
        if (w.from < below) break;               // (the same for all: the list ends behind the part)
    }
    __syncthreads();
    w.b = scalar(found_b);
    w.at = scalar(found_at);
    w.s = scalar(found);
    const long long head_cost = tiles_cost(a, w.s.before, w.s.tiles);
    w.head = scalar((int)((double)(w.from - w.at) / (double)head_cost));
    w.at += w.head * head_cost;
    int low = 0, high = w.s.tiles - 1;           // the last unit that begins no later
    while (low < high) {
        const int middle = (low + high + 1) / 2;
        if (w.at + tiles_cost(a, w.s.before, middle) <= w.from) low = middle;
        else high = middle - 1;
    }
    w.tile = low;
    w.at += tiles_cost(a, w.s.before, low);
    // units that are not cut belong to the part in which they begin
    return !(a.uncut && w.at < w.from) || next_unit(a, w, unit_cost(a, w));
}

// On to the next unit; false behind the last of the part.
__device__ __forceinline__ bool next_unit(const PagedAttn& a, Walk& w, long long cost)
{
    w.at += cost;
    if (w.at >= w.to) return false;
    if (++w.tile < w.s.tiles) return true;
    w.tile = 0;
    if (++w.head < a.pages.kv_heads * a.blocks) return true;
    w.head = 0;
    do {
        if (++w.b >= a.batch.seqs) return false;
        w.s = scalar(sequence(a, w.b));
    } while (w.s.tiles == 0);
    return true;
}

// A walk as it was put into LDS, for all lanes alike: it is needed between units only, and would fill the scalar registers while one is worked on.
__device__ __forceinline__ Walk scalar(const Walk& k)
{
    return Walk{scalar(k.wg), scalar(k.wgs), scalar(k.total), scalar(k.from), scalar(k.to), scalar(k.at), scalar(k.b), scalar(k.head), scalar(k.tile), scalar(k.s)};
}

// The present unit as one workgroup has it.
struct Unit {
    long long cost;
    int first_key, end_key;                      // its share of the keys
    int first_token, kv_head, first_head;        // rows: tokens of the sequence, query heads of the group
    bool whole, begins;
    float* piece;
};

template <int ROWS, int HD>
__device__ __forceinline__ Unit unit_of(const PagedAttn& a, const Walk& w)
{
    Unit u;
    u.cost = unit_cost(a, w);
    u.first_token = w.tile * a.tile_tokens;
    u.kv_head = w.head / a.blocks;
    u.first_head = (w.head - u.kv_head * a.blocks) * a.tile_heads;
    const int seen = max(w.s.length - w.s.n + min(u.first_token + a.tile_tokens, w.s.n), 0);   // by its last row
    u.begins = a.uncut || w.at >= w.from;
    const bool ends = a.uncut || w.at + u.cost <= w.to;
    u.whole = u.begins && ends;
    // (its keys in proportion to its cost)
    auto cut = [&](long long at) { return min((int)(share_of(at - w.at, seen, u.cost) + kRound - 1) / kRound * kRound, seen); };
    u.first_key = u.begins ? 0 : cut(w.from);
    u.end_key = ends ? seen : cut(w.to);
    u.piece = a.pieces + ((long long)w.wg * 2 + (u.begins ? 1 : 0)) * ROWS * (HD + 4);
    return u;
}

// By one thread, once it has the last unit of its part: what the second launch has to join.
__device__ __forceinline__ void tell_shared(const PagedAttn& a, const Walk& w, const Unit& u)
{
    Shared s{w.b, w.head, w.tile, -1};
    if (u.begins && !u.whole) {
        const long long end = w.at + u.cost;
        s.last = (int)share_of(end, w.wgs, w.total);              // or one beside it: the last whose part begins before the unit's end
        while (s.last + 1 < w.wgs && share_of(w.total, s.last + 1, w.wgs) < end) ++s.last;
        while (share_of(w.total, s.last, w.wgs) >= end) --s.last;
    }
    a.shared[w.wg] = s;
}

__device__ __forceinline__ bool last_unit(const Walk& w, const Unit& u) { return w.at + u.cost >= w.to; }

// Rows of a unit: row r is token r / tile_heads of its tokens, query head r % tile_heads of its heads.
struct Row {
    int token, head;                             // of the sequence, of all
    bool there;
};

__device__ __forceinline__ Row row_of(const PagedAttn& a, const Walk& w, const Unit& u, int r)
{
    const int t = r / a.tile_heads, h = r - t * a.tile_heads;
    Row x;
    x.token = u.first_token + t;
    x.there = t < a.tile_tokens && x.token < w.s.n && u.first_head + h < a.group;
    x.head = u.kv_head * a.group + u.first_head + h;
    return x;
}

typedef short short4v __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));

// Between what lanes of a wave put into LDS and what others of it read there, and between those reads and what is put there next.  (No instruction:
// LDS takes a wave's requests in order, and this holds the compiler to that order, which it sees no reason for in a lane of its own.)
__device__ __forceinline__ void wave_exchange()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Four 16-bit values of this lane's column from four rows of LDS: lanes 4 j + c of sixteen name row j, values 4 c .. 4 c + 3, and
// lane i of the sixteen gets column i.
__device__ __forceinline__ uint2 column_read(const unsigned char* p)
{
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wold-style-cast"
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p));
#pragma clang diagnostic pop
}

// Sixteen 8-bit codes as sixteen fp16 values, times a power of two.
__device__ __forceinline__ void sixteen_halves(u32x4 codes, float scale, u32x4* lo, u32x4* hi)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[i], scale, false));
        const uint32_t y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[i], scale, true));
        if (i < 2) (*lo)[2 * i] = x, (*lo)[2 * i + 1] = y;
        else (*hi)[2 * i - 4] = x, (*hi)[2 * i - 3] = y;
    }
}

// Eight fp16 values with those that are not finite made 0; whether there were any.  (A value that a row does not see weighs 0, which would make NaN of it.)
__device__ __forceinline__ bool make_finite(u32x4* x)
{
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t bad = (((*x)[i] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;   // the exponent's bits all set, in either half
        (*x)[i] &= ~((bad >> 15) * 0xffffu);
        any |= bad;
    }
    return any != 0;
}

// The running softmax of a row: its reference is a maximum that it has seen (in units of the scores), which probabilities are taken
// against; limit is how far a score may lie above it.  The reference moves only where a score passes the limit, kSlack in the exponent of 2, and the
// sums, which are fp32, hardly ever have to be scaled.  The reference's own probability is 2^kAbove, so that the largest is 2^15, the last power of two that fp16
// has.  Then its lower end rounds off 2^-32 of the largest a key at most, less than fp32 sums do (2^-29, where each addition brings 32 keys that are alike).
// (From 1 on, it was 2^-25: all of what lies 17.4 below the largest score, 0.4 % of a row over 131072 such keys.)
constexpr float kSlack = 8.0f, kAbove = 7.0f;

struct Running {
    float top, limit, base, sum;                 // base: of probabilities, an exponent of 2 (0 while there is no top); sum: of this lane's keys
};

// top as an exponent of 2 is rounded, and a score's difference from it is then off by as much, for all keys alike: that cancels in the quotient, but
// but where sums with other references are joined; and from 2^30 on the rounding alone takes probabilities out of the range of any format.  From kFar on,
// where it reaches 2^-12, top is taken from the scores themselves, before they are scaled.
constexpr float kFar = 4096.0f;

// The weight of sums taken against `top` among those against `now`, which is no less.  (Both -inf: there are none.)
__device__ __forceinline__ float weight_of(float top, float now, float scale_log2)
{
    return __builtin_amdgcn_exp2f((top - (now == kNone ? 0.f : now)) * scale_log2);
}

constexpr Running kNothing{kNone, kNone, 0.f, 0.f};

// Eight sums times `by` where `moves` says so.  (As assembly with a branch of its own: around a branch of the compiler's it keeps the sums in two
// sets of registers and copies all of them from the one to the other at every tile.  The compiler does not see what reads the sums here: a vector
// instruction may 19 wait states after the longest matrix product that writes them, which are waited for where sums are scaled at all.  Products that
// follow want two between a write and their read.)
__device__ __forceinline__ void scale_if(int moves, float by, f32x4& x, f32x4& y)
{
    float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    asm volatile("s_cmp_eq_u32 %8, 0\n\ts_cbranch_scc1 .Lkeep%=\n\ts_nop 15\n\ts_nop 2\n\t"
                 "v_mul_f32 %0, %9, %0\n\tv_mul_f32 %1, %9, %1\n\tv_mul_f32 %2, %9, %2\n\tv_mul_f32 %3, %9, %3\n\t"
                 "v_mul_f32 %4, %9, %4\n\tv_mul_f32 %5, %9, %5\n\tv_mul_f32 %6, %9, %6\n\tv_mul_f32 %7, %9, %7\n.Lkeep%=:\n\ts_nop 1"
                 : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]), "+v"(v[4]), "+v"(v[5]), "+v"(v[6]), "+v"(v[7]) : "s"(moves), "v"(by) : "scc");
    x = f32x4{v[0], v[1], v[2], v[3]};
    y = f32x4{v[4], v[5], v[6], v[7]};
}

// Scores of QF rows and COUNT fragments of 16 keys in, probabilities out (as the operand of the product with the values).  far: whether some row of the
// wave has a reference past kFar, 0 at the start.  MAY_BE: also at the start of this step; else that is looked at where a reference moves only (a branch
// of its own at every tile cost 4.5 % of a chunk's time).
template <bool MAY_BE, int QF, int COUNT, int DF>
__device__ __forceinline__ void softmax_step(f32x4 (&sc)[QF][COUNT], float scale_log2, Running (&run)[QF], int& far, f32x4 (&o)[QF][DF], u32x4 (&px)[QF][COUNT / 2])
{
    float most[QF];
    bool past = false;
#pragma unroll
    for (int f = 0; f < QF; ++f) {
        most[f] = sc[f][0][0];
#pragma unroll
        for (int n = 0; n < COUNT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) most[f] = fmaxf(most[f], sc[f][n][i]);
        past |= most[f] > run[f].limit;
    }
    auto from_top = [&] {
#pragma unroll
        for (int f = 0; f < QF; ++f) {
            const float top = run[f].top == kNone ? 0.f : run[f].top;
#pragma unroll
            for (int n = 0; n < COUNT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[f][n][i] -= top;
        }
    };
    const int moves = scalar((int)__popcll(__builtin_amdgcn_ballot_w64(past)));
    float shrink[QF];
#pragma unroll
    for (int f = 0; f < QF; ++f) shrink[f] = 1.0f;
    if (moves) {
        const float slack = kSlack / scale_log2;
        bool is_far = false;
#pragma unroll
        for (int f = 0; f < QF; ++f) {
            const float now = fmaxf(run[f].top, with_other_rows(most[f], [](float x, float y) { return fmaxf(x, y); }));
            shrink[f] = weight_of(run[f].top, now, scale_log2);
            run[f].top = now;
            const float base = now == kNone ? 0.f : now * scale_log2;             // (nothing but -inf so far)
            run[f].base = base - kAbove;
            run[f].sum *= shrink[f];
            is_far |= fabsf(base) > kFar;
        }
        far |= scalar((int)__popcll(__builtin_amdgcn_ballot_w64(is_far)));
#pragma unroll
        for (int f = 0; f < QF; ++f) {
            run[f].limit = far || run[f].top == kNone ? run[f].top : run[f].top + slack;   // (far: of numbers so large the sum may be rounded up)
        }
        if (far) {
#pragma unroll
            for (int f = 0; f < QF; ++f) run[f].base = -kAbove;
            if constexpr (!MAY_BE) from_top();
        }
    }
    if constexpr (MAY_BE)
        if (far) from_top();
#pragma unroll
    for (int f = 0; f < QF; ++f)
#pragma unroll
        for (int d = 0; d < DF; d += 2) scale_if(moves, shrink[f], o[f][d], o[f][d + 1]);
#pragma unroll
    for (int f = 0; f < QF; ++f) {
        float sum = 0.f;                                          // of this step's keys, as many as a lane has: a sum of all keys has few additions
#pragma unroll
        for (int n = 0; n < COUNT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float2v e;
#pragma unroll
                for (int j = 0; j < 2; ++j) e[j] = __builtin_amdgcn_exp2f(fmaf(sc[f][n][2 * i + j], scale_log2, -run[f].base));
                const half2v two = __builtin_convertvector(e, half2v);
                sum = __builtin_amdgcn_fdot2(two, half2v{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
                px[f][n >> 1][(n & 1) * 2 + i] = __builtin_bit_cast(uint32_t, two);
            }
        run[f].sum += sum;
    }
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is a register that the compiler reserves; named all the same, as this writes it)
// 16 bytes per lane from a buffer's byte `offset` + `more` into LDS at `lds` + 16 * lane, zeros past the buffer's end.  (As assembly, because the
// compiler would wait for all such loads before any read of LDS; here they are waited for by hand.  The compiler does not see a load here either: the buffer's
// description comes from the vector unit (v_readfirstlane), which a load may read five wait states later -- the move to m0 and the s_nop's four.)
__device__ __forceinline__ void buffer_to_lds(uint32_t lds, u32x4 buffer, uint32_t offset, uint32_t more)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(lds), "v"(offset), "s"(buffer), "s"(more) : "memory", "m0");
}
#pragma clang diagnostic pop

// The description of a buffer of `bytes` bytes for such loads.
__device__ __forceinline__ u32x4 buffer_at(const void* base, int bytes)
{
    const unsigned long long at = reinterpret_cast<unsigned long long>(base);
    return u32x4{(uint32_t)scalar((int)(uint32_t)at), (uint32_t)scalar((int)(uint32_t)(at >> 32) & 0xffff), (uint32_t)scalar(bytes), 0x00020000u};
}

// A workgroup of four waves holds 64 * QF rows, a wave QF fragments of 16, and walks its units' keys in tiles of KT, one pass.
// The scores are computed transposed, keys x rows: a lane then holds, for ONE row (lane % 16), four neighbouring keys of every
// fragment -- what it holds is already its operand of the second product (values^T x probabilities), and no probability crosses lanes.
// The values lie in LDS as they come, rows of a key, and are read by columns (column_read).
// LDS: two buffers of a tile of keys (pieces of 16 bytes swizzled so that the 16 keys of a read hit all banks) and of values (32-byte
// pairs swizzled so that the eight keys of a read do); one barrier a tile.  A wave brings a quarter of a tile's keys, which share a page.
// fp16 rows go from memory into LDS by themselves, from lane offsets that do not change: a tile costs a wave a page number and two
// buffer descriptions, and what lies past the sequence's end, outside the buffer, is zero (a key there weighs 0, which would make NaN of a value
// that is not finite).  8-bit rows pass through registers, where they become fp16: exactly for
// exponents from -15 on, of smaller ones rounded to its 2^-24.
// Measured with the join (15 us), 4096 rows over 4096 keys, 32 heads on 8 of 128: 402 us, 1025 TFLOP/s (425 on other cards); the matrix cores are busy for
// 48 % of it, the vector unit for 31 % and 18 % (exponentials) beside them.  64 rows: 526.  8-bit pages: 472 (64 rows: 665).  Heads of 64: 291, of 256: 1107.
template <int HD, int QF, bool BYTES>
__global__ __launch_bounds__(256, 2) void tl_paged_rows(PagedAttn a)
{
    constexpr int ROWS = 64 * QF, KT = HD == 256 ? 32 : 64, NF = KT / 16, KS = HD / 32, DF = HD / 16;
    constexpr int KB = KT * HD * 2, BUF = 2 * KB, KW = KT / 4;    // KW: keys that a wave brings
    constexpr int VALUES = BYTES ? 16 : 8, PIECES = HD / VALUES, KL = KW * PIECES / 64, KEYS = 64 / PIECES;   // of a load
    __shared__ __align__(16) unsigned char lds[2 * BUF];
    __shared__ int wrong_somewhere;
    __shared__ Walk kept;
    __shared__ int spoiled[2][KT];                                // keys of a buffer whose values were not finite
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6);
    const int g = lane >> 4, r16 = lane & 15;
    Walk w;
    if (!begin_walk(a, w)) return;
    auto key_place = [](int key, int p) { return HD == 64 ? p ^ ((key >> 1) & 7) : p ^ (key & 15); };
    auto value_place = [](int key, int pair) { return HD == 64 ? pair ^ ((key >> 1) & 3) : pair ^ (key & 7); };
    const int mask = (1 << a.pages.shift) - 1;
    // fp16: this lane's bytes within the wave's keys, for each load: where what comes to its place in LDS lies in the page
    uint32_t key_from[KL], value_from[KL];
    if constexpr (!BYTES) {
#pragma unroll
        for (int i = 0; i < KL; ++i) {
            const int key = wave * KW + i * KEYS + lane / PIECES, p = lane % PIECES;
            key_from[i] = (uint32_t)(lane / PIECES) * (uint32_t)a.pages.slot_stride * 2u + (uint32_t)key_place(key, p) * 16u;
            value_from[i] = (uint32_t)(lane / PIECES) * (uint32_t)a.pages.slot_stride * 2u + (uint32_t)(value_place(key, p >> 1) * 2 + (p & 1)) * 16u;
        }
    }
    const uint32_t lds_at = (uint32_t)(uintptr_t)lds;             // (the low half of such an address is the offset in LDS)
    for (;;) {
        Unit u = unit_of<ROWS, HD>(a, w);
        const int first_tile = (u.first_key + KT - 1) / KT, tiles = (u.end_key + KT - 1) / KT;   // (a share may be empty)
        bool wrong = w.s.wrong;
        const int length = w.s.length;
        // Tiles with tokens that some of the unit's rows do not see: values there that are not finite must not meet the weights of 0.  They are made 0
        // in LDS, and the rows that do see their key are NaN.
        const int all_see = length - w.s.n + u.first_token;       // the last key that every row sees
        const int first_mixed = all_see < length - 1 ? max(all_see + 1, 0) / KT : INT_MAX;   // ... are the last
        // ---- tiles on their way ----
        const long long head_at = u.kv_head * a.pages.head_stride;
        // page of this wave's keys of the tile after the next (by a vector load: a scalar one would be waited for with the first read of LDS)
        const int* ids = a.batch.table + w.b * a.batch.table_stride;
        int ahead = 0;
        auto ask = [&](int t) { ahead = ids[min(t * KT + wave * KW, length - 1) >> a.pages.shift]; };
        u32x4 kreg[KL], vreg[KL];
        int kexp[KL], vexp[KL];
        auto fetch = [&](int t, int buf) {
            const int number = scalar(ahead);
            const bool known = (unsigned)number < a.pages.pages;
            wrong |= !known;
            const int page = known ? number : 0, first = t * KT + wave * KW;
            const long long at = page * a.pages.page_stride + head_at;
            if constexpr (BYTES) {
                const long long exp_at = ((long long)page * a.pages.kv_heads + u.kv_head) << a.pages.shift;
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    const int key = first + i * KEYS + lane / PIECES, slot = min(key, length - 1) & mask;
                    const unsigned within = (unsigned)slot * (unsigned)a.pages.slot_stride + (unsigned)(lane % PIECES) * VALUES;
                    kreg[i] = *reinterpret_cast<const u32x4*>(static_cast<const unsigned char*>(a.pages.k) + at + within);
                    vreg[i] = *reinterpret_cast<const u32x4*>(static_cast<const unsigned char*>(a.pages.v) + at + within);
                    kexp[i] = a.pages.k_exp[exp_at + slot];
                    vexp[i] = a.pages.v_exp[exp_at + slot];
                }
            } else {
                const int there = min(max(length - first, 0), KW), step = (int)a.pages.slot_stride * 2;
                const long long from = (at + (long long)(there ? first & mask : 0) * a.pages.slot_stride) * 2;
                const u32x4 kbuf = buffer_at(static_cast<const char*>(a.pages.k) + from, there * step), vbuf = buffer_at(static_cast<const char*>(a.pages.v) + from, there * step);
                const uint32_t to = (uint32_t)scalar((int)(lds_at + buf * BUF + wave * KW * HD * 2));
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    buffer_to_lds(to + i * 1024, kbuf, key_from[i], (uint32_t)(i * KEYS * step));
                    buffer_to_lds(to + KB + i * 1024, vbuf, value_from[i], (uint32_t)(i * KEYS * step));
                }
            }
        };
        auto put = [&](auto may_mix, int t, int buf) {            // what fetch has asked for is in LDS
            const bool mixed = decltype(may_mix)::value && t >= first_mixed;
            if (mixed) {
                if (lane < KW) spoiled[buf][wave * KW + lane] = 0;
                wave_exchange();
            }
            if constexpr (BYTES) {
                unsigned char* kd = lds + buf * BUF;
                unsigned char* vd = kd + KB;
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    const int key = wave * KW + i * KEYS + lane / PIECES, p = lane % PIECES;
                    u32x4 lo, hi;
                    sixteen_halves(kreg[i], __uint_as_float((uint32_t)kexp[i] << 23), &lo, &hi);
                    *reinterpret_cast<u32x4*>(kd + key * HD * 2 + key_place(key, 2 * p) * 16) = lo;
                    *reinterpret_cast<u32x4*>(kd + key * HD * 2 + key_place(key, 2 * p + 1) * 16) = hi;
                    sixteen_halves(vreg[i], __uint_as_float((uint32_t)vexp[i] << 23), &lo, &hi);
                    if (t * KT + key >= length) lo = hi = u32x4{0u, 0u, 0u, 0u};
                    if (mixed) {
                        const bool low = make_finite(&lo), high = make_finite(&hi);
                        if (low || high) spoiled[buf][key] = 1;
                    }
                    u32x4* v = reinterpret_cast<u32x4*>(vd + key * HD * 2 + value_place(key, p) * 32);
                    v[0] = lo;
                    v[1] = hi;
                }
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                if (mixed) {
#pragma unroll
                    for (int i = 0; i < KL; ++i) {
                        u32x4* at = reinterpret_cast<u32x4*>(lds + buf * BUF + KB + wave * KW * HD * 2 + i * 1024 + lane * 16);
                        u32x4 x = *at;
                        if (make_finite(&x)) *at = x, spoiled[buf][wave * KW + i * KEYS + lane / PIECES] = 1;
                    }
                }
            }
        };
        if (first_tile < tiles) ask(first_tile);

        // ---- the wave's rows ----
        u32x4 qx[QF][KS];
        int last[QF];                                             // the last key that this lane's row sees
        int wave_last = -1, wave_first = INT_MAX;                 // ... any of the wave's, and all of them
        f32x4 o[QF][DF];
        Running run[QF];
        int far = 0;
#pragma unroll
        for (int f = 0; f < QF; ++f) {
            const Row x = row_of(a, w, u, wave * 16 * QF + f * 16 + r16);
            last[f] = x.there ? w.s.length - w.s.n + x.token : -1;
            const __half* row = a.q + (long long)(w.s.start + x.token) * a.q_t + x.head * a.q_h + g * 8;
#pragma unroll
            for (int s = 0; s < KS; ++s) qx[f][s] = x.there ? *reinterpret_cast<const u32x4*>(row + s * 32) : u32x4{0u, 0u, 0u, 0u};
            run[f] = kNothing;
#pragma unroll
            for (int d = 0; d < DF; ++d) o[f][d] = f32x4{0.f, 0.f, 0.f, 0.f};
            wave_last = max(wave_last, last[f]);
            wave_first = min(wave_first, last[f]);
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) {
            wave_last = max(wave_last, __shfl_xor(wave_last, off, 64));
            wave_first = min(wave_first, __shfl_xor(wave_first, off, 64));
        }
        wave_last = scalar(wave_last);
        wave_first = scalar(wave_first);

        __syncthreads();                                          // the unit before is done with LDS
        if (tid == 0) wrong_somewhere = 0, kept = w;
        if (first_tile < tiles) {
            fetch(first_tile, 0);
            if (first_tile + 1 < tiles) ask(first_tile + 1);
            put(std::true_type{}, first_tile, 0);
        }
        __syncthreads();
#pragma unroll
        for (int f = 0; f < QF; ++f)
#pragma unroll
            for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qx[f][s]));   // (here before the loop: waited for inside it, the next tile's loads are too)

        // the next tile on its way, and in LDS; the tiles of which the wave's rows see nothing, which come last, are brought and no more
        auto before = [&](int t) {
            if (t + 1 < tiles) {
                fetch(t + 1, (t + 1 - first_tile) & 1);
                if (t + 2 < tiles) ask(t + 2);
            }
        };
        auto behind = [&](auto may_mix, int t) {
            if (t + 1 < tiles) {
                put(may_mix, t + 1, (t + 1 - first_tile) & 1);             // (read last before the barrier of the turn before)
                __syncthreads();
            }
        };
        const int seen_tiles = min(tiles, wave_last / KT + (wave_last >= 0 ? 1 : 0));
        auto work = [&](auto may_mix, int t) {
            before(t);
            const unsigned char* ks = lds + ((t - first_tile) & 1) * BUF;
            const unsigned char* vs = ks + KB;
            f32x4 sc[QF][NF];
            // NF fragments of keys a step, the next ones read while these are multiplied.  (Left to the compiler all reads move to the front and
            // fill the registers, until it copies the sums at every branch.)
            u32x4 kx[2][NF];
            auto keys = [&](int s, u32x4* to) {
#pragma unroll
                for (int n = 0; n < NF; ++n) to[n] = *reinterpret_cast<const u32x4*>(ks + (n * 16 + r16) * HD * 2 + key_place(r16, s * 4 + g) * 16);
            };
            keys(0, kx[0]);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if (s + 1 < KS) keys(s + 1, kx[(s + 1) & 1]);
#pragma unroll
                for (int n = 0; n < NF; ++n)
#pragma unroll
                    for (int f = 0; f < QF; ++f) sc[f][n] = matrix_step<false>(kx[s & 1][n], qx[f][s], s == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[f][n]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (t * KT + KT - 1 > wave_first) {               // some row of the wave does not see all of the tile
#pragma unroll
                for (int f = 0; f < QF; ++f) {
                    const int seen = last[f] - t * KT - g * 4;
#pragma unroll
                    for (int n = 0; n < NF; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[f][n][i] = n * 16 + i <= seen ? sc[f][n][i] : kNone;
                }
            }
            u32x4 px[QF][NF / 2];
            softmax_step<decltype(may_mix)::value>(sc, a.scale_log2, run, far, o, px);
            if (decltype(may_mix)::value && t >= first_mixed) {
                const unsigned long long keys_spoiled = __builtin_amdgcn_ballot_w64(lane < KT && spoiled[(t - first_tile) & 1][lane & (KT - 1)] != 0);
                if (keys_spoiled != 0) {
#pragma unroll
                    for (int f = 0; f < QF; ++f) {
                        const int seen = last[f] - t * KT;
                        if (seen >= 0 && (keys_spoiled & (~0ull >> (63 - min(seen, 63)))) != 0) run[f].sum = __builtin_nanf("");
                    }
                }
            }
            constexpr int VG = 4, GROUPS = NF / 2 * DF / VG;  // values: VG fragments a step
            u32x4 vx[2][VG];
            auto values = [&](int i, u32x4* to) {
#pragma unroll
                for (int j = 0; j < VG; ++j) {
                    const int key = i * VG / DF * 32 + g * 4 + (r16 >> 2), d = i * VG % DF + j;
                    const unsigned char* from = vs + key * HD * 2 + value_place(g * 4 + (r16 >> 2), d) * 32 + (r16 & 3) * 8;
                    const uint2 x = column_read(from), y = column_read(from + 16 * HD * 2);   // (16 keys on: the same swizzle)
                    to[j] = u32x4{x.x, x.y, y.x, y.y};
                }
            };
            values(0, vx[0]);
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) {
                if (i + 1 < GROUPS) values(i + 1, vx[(i + 1) & 1]);
#pragma unroll
                for (int j = 0; j < VG; ++j)
#pragma unroll
                    for (int f = 0; f < QF; ++f) o[f][i * VG % DF + j] = matrix_step<false>(vx[i & 1][j], px[f][i * VG / DF], o[f][i * VG % DF + j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            behind(may_mix, t);
        };
        int t = first_tile;
        for (; t < min(seen_tiles, first_mixed - 1) && !far; ++t) work(std::false_type{}, t);   // (nor is the next one mixed)
        for (; t < seen_tiles; ++t) work(std::true_type{}, t);
        for (; t < tiles; ++t) {
            before(t);
            behind(std::true_type{}, t);
        }
        if (wrong && lane == 0) wrong_somewhere = 1;
        __syncthreads();
        wrong = wrong_somewhere != 0;
        w = scalar(kept);
        u = unit_of<ROWS, HD>(a, w);
#pragma unroll
        for (int f = 0; f < QF; ++f) {
            const int r = wave * 16 * QF + f * 16 + r16;
            const Row x = row_of(a, w, u, r);
            float all = with_other_rows(run[f].sum, [](float v, float y) { return v + y; });
            if (wrong) all = __builtin_nanf("");
            if (!x.there) continue;
            if (u.whole) {
                const float inv = all == 0.f ? 0.f : 1.0f / all;  // (no key: 0)
                __half* row = a.out + ((long long)(w.s.start + x.token) * a.heads + x.head) * HD + g * 4;
#pragma unroll
                for (int d = 0; d < DF; ++d) {
                    __half h[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[i] = __float2half(o[f][d][i] * inv);
                    *reinterpret_cast<uint2*>(row + d * 16) = *reinterpret_cast<const uint2*>(h);
                }
            } else {
                float* row = u.piece + r * (HD + 4);
#pragma unroll
                for (int d = 0; d < DF; ++d) *reinterpret_cast<f32x4*>(row + d * 16 + g * 4) = o[f][d];
                if (g == 0) row[HD] = run[f].top, row[HD + 1] = all;
            }
        }
        if (last_unit(w, u)) {
            if (tid == 0) tell_shared(a, w, u);
            return;
        }
        if (!next_unit(a, w, u.cost)) return;
    }
}

// 16 rows: single tokens, or the few of a group of query heads.  Bound by the pages' bytes.  A workgroup's four waves share out a unit's
// keys, tile by tile of 32 each, every wave with a softmax of its own; at the unit's end they meet in LDS.  No wave waits for another
// before: a wave's keys go from memory straight into the registers that its products want, its values through LDS of its own (to be read
// by columns).  The next tile is asked for as soon as this one's registers are free.  8-bit rows are loaded 16 values to a lane, and
// the order of the values within a score is free: the queries are loaded to match.
// Measured, with the join: 32 sequences of 4096, 32 heads on 8 of 128: 102 us, 5.3 TB/s (8-bit pages 58, 4.7); heads of 256, whose registers allow one
// workgroup a compute unit, 104 for the same bytes (241 while they spilled).
template <int HD, bool BYTES>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void tl_paged_few(PagedAttn a)
{
    constexpr int ROWS = 16, KT = 32, KS = HD / 32, DF = HD / 16;
    constexpr int KL = BYTES ? HD / 64 : KS;                      // 16-byte pieces of a key that a lane loads
    constexpr int VALUES = BYTES ? 16 : 8, PIECES = HD / VALUES, VL = KT * PIECES / 64, VKEYS = 64 / PIECES;   // keys of one load of values
    constexpr int LD = HD + 4;
    __shared__ __align__(16) unsigned char lds[4 * ROWS * LD * 4];                                              // >= 4 * KT * HD * 2
    __shared__ float tops[4][ROWS], sums[4][ROWS];
    __shared__ int wrong_somewhere;
    __shared__ Walk kept;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6);
    const int g = lane >> 4, r16 = lane & 15;
    Walk w;
    if (!begin_walk(a, w)) return;
    unsigned char* own = lds + wave * KT * HD * 2;
    auto value_place = [](int key, int pair) { return HD == 64 ? pair ^ ((key >> 1) & 3) : pair ^ (key & 7); };
    for (;;) {
        Unit u = unit_of<ROWS, HD>(a, w);
        if (tid == 0) kept = w;
        const int tiles = (u.end_key + KT - 1) / KT, first_tile = (u.first_key + KT - 1) / KT + wave;
        bool wrong = w.s.wrong;
        const int length = w.s.length;
        const long long head_at = u.kv_head * a.pages.head_stride;
        const int* ids = a.batch.table + w.b * a.batch.table_stride;
        u32x4 kreg[2][KL], vreg[VL];
        int kexp[2], vexp[VL];
        int ahead[2];                                             // pages of the next tile's keys
        auto ask = [&](int t) {
#pragma unroll
            for (int n = 0; n < 2; ++n) ahead[n] = (int)as_const(reinterpret_cast<const uint32_t*>(ids))[scalar(min(t * KT + n * 16, length - 1) >> a.pages.shift)];
        };
        auto fetch = [&](int t) {
            long long at[2], exp_at[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const bool known = (unsigned)ahead[n] < a.pages.pages;
                wrong |= !known;
                const int page = known ? ahead[n] : 0;
                at[n] = page * a.pages.page_stride + head_at;
                exp_at[n] = ((long long)page * a.pages.kv_heads + u.kv_head) << a.pages.shift;
            }
            const int mask = (1 << a.pages.shift) - 1;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int slot = min(t * KT + n * 16 + r16, length - 1) & mask;
                const unsigned within = (unsigned)slot * (unsigned)a.pages.slot_stride + (unsigned)g * VALUES;
#pragma unroll
                for (int s = 0; s < KL; ++s) {
                    if constexpr (BYTES) kreg[n][s] = *reinterpret_cast<const u32x4*>(static_cast<const unsigned char*>(a.pages.k) + at[n] + within + s * 64);
                    else kreg[n][s] = *reinterpret_cast<const u32x4*>(static_cast<const __half*>(a.pages.k) + at[n] + within + s * 32);
                }
                if constexpr (BYTES) kexp[n] = a.pages.k_exp[exp_at[n] + slot];
            }
#pragma unroll
            for (int i = 0; i < VL; ++i) {
                const int n = i * VKEYS / 16, slot = min(t * KT + i * VKEYS + lane / PIECES, length - 1) & mask;
                const unsigned within = (unsigned)slot * (unsigned)a.pages.slot_stride + (unsigned)(lane % PIECES) * VALUES;
                if constexpr (BYTES) {
                    vreg[i] = *reinterpret_cast<const u32x4*>(static_cast<const unsigned char*>(a.pages.v) + at[n] + within);
                    vexp[i] = a.pages.v_exp[exp_at[n] + slot];
                } else {
                    vreg[i] = *reinterpret_cast<const u32x4*>(static_cast<const __half*>(a.pages.v) + at[n] + within);
                }
            }
        };
        if (first_tile < tiles) {
            ask(first_tile);
            fetch(first_tile);
            if (first_tile + 4 < tiles) ask(first_tile + 4);
        }
        const Row x = row_of(a, w, u, r16);
        const int last = x.there ? w.s.length - w.s.n + x.token : -1;
        u32x4 qx[KS];
        const __half* row = a.q + (long long)(w.s.start + x.token) * a.q_t + x.head * a.q_h;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = BYTES ? s / 2 * 64 + g * 16 + s % 2 * 8 : s * 32 + g * 8;
            qx[s] = x.there ? *reinterpret_cast<const u32x4*>(row + d) : u32x4{0u, 0u, 0u, 0u};
        }
        f32x4 o[1][DF];
        Running run[1] = {kNothing};
        int far = 0;
#pragma unroll
        for (int d = 0; d < DF; ++d) o[0][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int all_see = w.s.length - w.s.n + u.first_token;   // the last key that every row sees

        auto spoil = [&](unsigned long long lanes, int first) {   // lanes whose pieces of values were not finite, of keys from `first` on
            for (int k = 0; lanes != 0 && k < VKEYS; ++k)
                if ((lanes >> (k * PIECES) & (~0ull >> (64 - PIECES))) != 0 && first + k <= last) run[0].sum = __builtin_nanf("");
        };
        for (int t = first_tile; t < tiles; t += 4) {
            const bool ends = t * KT + KT > length;
            // a tile with tokens that some rows do not see: values that are not finite become 0, and the rows that see their key NaN
            const bool mixed = all_see < length - 1 && t * KT + KT - 1 > all_see;
#pragma unroll
            for (int i = 0; i < VL; ++i) {
                const int key = i * VKEYS + lane / PIECES, p = lane % PIECES;
                // (a key past the end weighs 0, which would make NaN of a value that is not finite)
                if (ends && t * KT + key >= length) vreg[i] = u32x4{0u, 0u, 0u, 0u};
                if constexpr (BYTES) {
                    u32x4 lo, hi;
                    sixteen_halves(vreg[i], __uint_as_float((uint32_t)vexp[i] << 23), &lo, &hi);
                    if (mixed) {
                        const bool low = make_finite(&lo), high = make_finite(&hi);
                        spoil(__builtin_amdgcn_ballot_w64(low || high), t * KT + i * VKEYS);
                    }
                    u32x4* v = reinterpret_cast<u32x4*>(own + key * HD * 2 + value_place(key, p) * 32);
                    v[0] = lo;
                    v[1] = hi;
                } else {
                    if (mixed) spoil(__builtin_amdgcn_ballot_w64(make_finite(&vreg[i])), t * KT + i * VKEYS);
                    *reinterpret_cast<u32x4*>(own + key * HD * 2 + value_place(key, p >> 1) * 32 + (p & 1) * 16) = vreg[i];
                }
            }
            wave_exchange();
            f32x4 sc[1][2];
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    u32x4 kx;
                    if constexpr (BYTES) {
                        u32x4 both[2];
                        if (s % 2 == 0) sixteen_halves(kreg[n][s / 2], __uint_as_float((uint32_t)kexp[n] << 23), &both[0], &both[1]), kreg[n][s / 2] = both[1], kx = both[0];
                        else kx = kreg[n][s / 2];
                    } else {
                        kx = kreg[n][s];
                    }
                    sc[0][n] = matrix_step<false>(kx, qx[s], s == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[0][n]);
                }
            if (t + 4 < tiles) {
                fetch(t + 4);
                if (t + 8 < tiles) ask(t + 8);
            }
            if (t * KT + KT - 1 > all_see) {
                const int seen = last - t * KT - g * 4;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[0][n][i] = n * 16 + i <= seen ? sc[0][n][i] : kNone;
            }
            u32x4 px[1][1];
            softmax_step<true>(sc, a.scale_log2, run, far, o, px);
#pragma unroll
            for (int d = 0; d < DF; ++d) {
                const int key = g * 4 + (r16 >> 2);
                const unsigned char* from = own + key * HD * 2 + value_place(key, d) * 32 + (r16 & 3) * 8;
                const uint2 lo = column_read(from), hi = column_read(from + 16 * HD * 2);   // (16 keys on: the same swizzle)
                o[0][d] = matrix_step<false>(u32x4{lo.x, lo.y, hi.x, hi.y}, px[0][0], o[0][d]);
            }
            wave_exchange();
        }
        // ---- the waves meet ----
        const float sum = with_other_rows(run[0].sum, [](float v, float y) { return v + y; });
        if (tid == 0) wrong_somewhere = 0;
        __syncthreads();                                          // every wave is done with its values
        w = scalar(kept);
        u = unit_of<ROWS, HD>(a, w);
        float* mine = reinterpret_cast<float*>(lds) + (wave * ROWS + r16) * LD;
        if (x.there) {
#pragma unroll
            for (int d = 0; d < DF; ++d) *reinterpret_cast<f32x4*>(mine + d * 16 + g * 4) = o[0][d];
            if (g == 0) tops[wave][r16] = run[0].top, sums[wave][r16] = sum;
        }
        if (wrong && lane == 0) wrong_somewhere = 1;
        __syncthreads();
        {
            constexpr int EACH = HD / 16;                         // values of a thread
            const int r = tid >> 4, d = (tid & 15) * 4;           // four values, and those 64 on
            const Row y = row_of(a, w, u, r);
            if (y.there) {
                float most = tops[0][r];
#pragma unroll
                for (int i = 1; i < 4; ++i) most = fmaxf(most, tops[i][r]);
                f32x4 v[EACH / 4];
#pragma unroll
                for (int j = 0; j < EACH / 4; ++j) v[j] = f32x4{0.f, 0.f, 0.f, 0.f};
                float all = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float weight = weight_of(tops[i][r], most, a.scale_log2);
                    all = fmaf(sums[i][r], weight, all);
                    const float* theirs = reinterpret_cast<const float*>(lds) + (i * ROWS + r) * LD + d;
#pragma unroll
                    for (int j = 0; j < EACH / 4; ++j) {
                        const f32x4 z = *reinterpret_cast<const f32x4*>(theirs + j * 64);
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[j][e] = fmaf(z[e], weight, v[j][e]);
                    }
                }
                if (wrong_somewhere) all = __builtin_nanf("");
                if (u.whole) {
                    const float inv = all == 0.f ? 0.f : 1.0f / all;   // (no key: 0)
                    __half* to = a.out + ((long long)(w.s.start + y.token) * a.heads + y.head) * HD + d;
#pragma unroll
                    for (int j = 0; j < EACH / 4; ++j) {
                        __half h[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) h[e] = __float2half(v[j][e] * inv);
                        *reinterpret_cast<uint2*>(to + j * 64) = *reinterpret_cast<const uint2*>(h);
                    }
                } else {
                    float* to = u.piece + r * LD;
#pragma unroll
                    for (int j = 0; j < EACH / 4; ++j) *reinterpret_cast<f32x4*>(to + d + j * 64) = v[j];
                    if (d == 0) to[HD] = most, to[HD + 1] = all;
                }
            }
        }
        if (last_unit(w, u)) {
            if (tid == 0) tell_shared(a, w, u);
            return;
        }
        if (!next_unit(a, w, u.cost)) return;
        __syncthreads();                                          // the unit is done with LDS
    }
}

// Joins the pieces of the units that were shared out: blockIdx.x is the workgroup in which one begins.  HD / 4 lanes take a row, four
// values each.  Of a unit of a few pieces as many rows as there are such groups of lanes are joined at a time; where they are many, as of a single long sequence, one row by as many
// groups of lanes, which share the pieces out.
template <int ROWS>
constexpr int kJoinThreads = ROWS > 16 ? 512 : 256;

template <int HD, int ROWS>
__global__ __launch_bounds__(kJoinThreads<ROWS>) void tl_paged_join(PagedAttn a)
{
    constexpr int THREADS = kJoinThreads<ROWS>, LANES = HD / 4, AT_ONCE = THREADS / LANES, FEW = ROWS > 16 ? 64 : 8;
    __shared__ float4 part[THREADS];
    __shared__ float tops[AT_ONCE], sums[AT_ONCE];
    Shared sh = a.shared[blockIdx.x];
    sh.last = scalar(sh.last);
    if (sh.last < 0) return;
    Walk w{};
    w.b = scalar(sh.seq), w.head = scalar(sh.head), w.tile = scalar(sh.tile);
    w.s = scalar(sequence(a, w.b));
    const Unit u = unit_of<ROWS, HD>(a, w);
    const int first = (int)blockIdx.x, count = sh.last - first + 1;
    const int lane = (int)threadIdx.x % LANES, own = (int)threadIdx.x / LANES;
    float4 o;
    float top, sum;
    auto start = [&] { o = make_float4(0.f, 0.f, 0.f, 0.f), top = kNone, sum = 0.f; };
    // pieces i, i + step, ... of a row, several on their way at a time
    auto add = [&](auto fly, int i, int step, int r) {
        constexpr int FLY = decltype(fly)::value;
        for (; i < count; i += FLY * step) {
            float m[FLY], l[FLY];
            float4 v[FLY];
#pragma unroll
            for (int k = 0; k < FLY; ++k) {
                const int n = min(i + k * step, count - 1);
                const float* piece = a.pieces + (((long long)(first + n) * 2 + (n == 0 ? 1 : 0)) * ROWS + r) * (HD + 4);
                m[k] = piece[HD], l[k] = piece[HD + 1];
                v[k] = *reinterpret_cast<const float4*>(piece + lane * 4);
            }
            if constexpr (FLY > 4) __builtin_amdgcn_sched_barrier(0);   // (or the compiler asks for them one after the other)
#pragma unroll
            for (int k = 0; k < FLY; ++k) {
                if (i + k * step >= count) break;
                const float now = fmaxf(top, m[k]);
                const float old = weight_of(top, now, a.scale_log2), fresh = weight_of(m[k], now, a.scale_log2);
                o = make_float4(o.x * old + v[k].x * fresh, o.y * old + v[k].y * fresh, o.z * old + v[k].z * fresh, o.w * old + v[k].w * fresh);
                sum = sum * old + l[k] * fresh;
                top = now;
            }
        }
    };
    auto finish = [&](const Row& x) {
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;          // (no key: 0)
        const __half h[4] = {__float2half(o.x * inv), __float2half(o.y * inv), __float2half(o.z * inv), __float2half(o.w * inv)};
        *reinterpret_cast<uint2*>(a.out + ((long long)(w.s.start + x.token) * a.heads + x.head) * HD + lane * 4) = *reinterpret_cast<const uint2*>(h);
    };
    if (count <= FEW) {
        for (int r = (int)blockIdx.y * AT_ONCE + own; r < ROWS; r += (int)gridDim.y * AT_ONCE) {
            const Row x = row_of(a, w, u, r);
            if (!x.there) continue;
            start();
            add(std::integral_constant<int, 4>{}, 0, 1, r);
            finish(x);
        }
        return;
    }
    for (int r = (int)blockIdx.y; r < ROWS; r += (int)gridDim.y) {
        const Row x = row_of(a, w, u, r);
        if (!x.there) continue;                                   // (the same for all)
        start();
        if (ROWS > 16 || count <= 4 * AT_ONCE) add(std::integral_constant<int, 4>{}, own, AT_ONCE, r);
        else add(std::integral_constant<int, (ROWS > 16 ? 4 : 8)>{}, own, AT_ONCE, r);
        __syncthreads();                                          // the row before is done with LDS
        part[threadIdx.x] = o;
        if (lane == 0) tops[own] = top, sums[own] = sum;
        __syncthreads();
        if (own == 0) {
            float most = tops[0];
#pragma unroll
            for (int i = 1; i < AT_ONCE; ++i) most = fmaxf(most, tops[i]);
            start();
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const float weight = weight_of(tops[i], most, a.scale_log2);
                const float4 v = part[i * LANES + lane];
                o = make_float4(o.x + v.x * weight, o.y + v.y * weight, o.z + v.z * weight, o.w + v.w * weight);
                sum += sums[i] * weight;
            }
            finish(x);
        }
    }
}

// What a call takes: rows of a unit, workgroups at most, the cost of a unit beside its keys, the cost below which a part is not cut, and whether units
// are not cut at all.
struct Plan {
    int rows, workgroups, fixed, least, uncut;
};

Plan plan_of(int64_t tokens, int heads, const tl_pages* pages, const tl_page_batch* batch, int64_t most_rows)
{
    const int group = heads / pages->kv_heads, hd = pages->head_dim;
    const int64_t keys = (int64_t)batch->table_pages * pages->page_size;   // of a sequence, at most
    auto workgroups = [](int each) { return (int)ceil_div(each * compute_units(), 8) * 8; };
    // units of few keys are not cut, which saves the second launch (us uncut / cut: one sequence of 600, 32 heads, 12.7 / 15.7; 8 of 300, 32 heads on 8,
    // 10.9 / 15.4; 256 of up to 200 25.3 / 31.6; 64 of 1000 51.3 / 53.4).  At the edge a few units alone would be quicker cut: one sequence of 1000, 32 heads,
    // 17.1 / 15.4; 8 heads on one 16.1 / 12.0, of 600 12.7 / 12.2.  (The lengths are on the device: the table's width is what the host knows.)
    const int uncut = keys <= 1024;
    if (most_rows * group <= 16) return Plan{16, workgroups(hd == 256 ? 1 : 2), 128, 128, uncut};
    // 128 rows to a workgroup read half as much from LDS for a product, 64 have twice as many units: from 2048 keys of 128 rows to a workgroup on, as
    // far as the host can tell (us with 128 / 64: 4096 rows over 4096, 32 heads on 8: 402 / 526; 723 rows of 8 sequences of up to 3500, 14
    // heads of 64 on 2: 37 / 34; 64 rows over 32768, 32 heads on 8: 92 / 78).
    const bool tall = hd < 256 && most_rows * group >= 128 && tokens * heads / 128 * keys >= workgroups(2) * 2048ll;
    return Plan{tall ? 128 : 64, workgroups(2), 128, 512, uncut};
}

int64_t workspace_of(const Plan& p, int hd)
{
    return (int64_t)p.workgroups * (2 * p.rows * (hd + 4) * (int64_t)sizeof(float) + (int64_t)sizeof(Shared));
}

int check_heads(int heads, const tl_pages* pages)
{
    if (!pages) return fail(TL_ERR_ARG, "null pointer");
    if (pages->head_dim != 64 && pages->head_dim != 128 && pages->head_dim != 256) return fail(TL_ERR_UNSUPPORTED, "head_dim=%d (64, 128 or 256 supported)", pages->head_dim);
    if (heads <= 0 || heads > (1 << 16) || pages->kv_heads <= 0 || heads % pages->kv_heads) return fail(TL_ERR_SHAPE, "kv_heads=%d must divide heads=%d", pages->kv_heads, heads);
    return TL_OK;
}

template <int HD, int ROWS>
void launch_join(const PagedAttn& a, const Plan& p, hipStream_t st)
{
    if (!p.uncut) hipLaunchKernelGGL((tl_paged_join<HD, ROWS>), dim3((unsigned)p.workgroups, 8), dim3(kJoinThreads<ROWS>), 0, st, a);
}

template <int HD, bool BYTES>
void launch_attention(const PagedAttn& a, const Plan& p, hipStream_t st)
{
    const dim3 grid((unsigned)p.workgroups), block(256);
    if (p.rows == 16) {
        hipLaunchKernelGGL((tl_paged_few<HD, BYTES>), grid, block, 0, st, a);
        launch_join<HD, 16>(a, p, st);
        return;
    }
    if constexpr (HD < 256) {
        if (p.rows == 128) {
            hipLaunchKernelGGL((tl_paged_rows<HD, 2, BYTES>), grid, block, 0, st, a);
            launch_join<HD, 128>(a, p, st);
            return;
        }
    }
    hipLaunchKernelGGL((tl_paged_rows<HD, 1, BYTES>), grid, block, 0, st, a);
    launch_join<HD, 64>(a, p, st);
}

}  // namespace

extern "C" int tl_paged_attention_workspace(int64_t tokens, int heads, const tl_pages* pages, const tl_page_batch* batch, int64_t most_rows, int64_t* bytes)
{
    if (int rc = check_heads(heads, pages)) return rc;
    if (!bytes || !batch || most_rows < 0 || tokens < 0) return fail(TL_ERR_ARG, "a pointer is null, or tokens or most_rows negative");
    *bytes = workspace_of(plan_of(tokens, heads, pages, batch, most_rows), pages->head_dim);
    return TL_OK;
}

extern "C" int tl_paged_attention(const void* q, int64_t q_token, int64_t q_head, int dtype, int64_t tokens, int heads, const tl_pages* pages,
                                  const tl_page_batch* batch, int64_t most_rows, float scale, void* out, void* workspace, int64_t workspace_bytes, void* stream)
{
    if (int rc = check_dtype(dtype, "q")) return rc;
    if (dtype != TL_F16) return fail(TL_ERR_UNSUPPORTED, "fp16 queries only");
    PagedAttn a{};
    if (int rc = check_heads(heads, pages)) return rc;
    if (int rc = take_pages(pages, batch, tokens, &a.pages, &a.batch)) return rc;
    if (tokens == 0 || a.batch.seqs == 0) return TL_OK;
    if (!q || !out || !workspace) return fail(TL_ERR_ARG, "device pointer is null");
    if (most_rows < 0) return fail(TL_ERR_ARG, "most_rows is negative");
    if (!(scale > 0.f) || scale > 1e30f) return fail(TL_ERR_ARG, "scale=%g is not a positive number up to 1e30", (double)scale);
    if (!in_pieces(q, {q_token, q_head}, 2) || !in_pieces(out, {}, 2) || !in_pieces(workspace, {}, 1)) return fail(TL_ERR_ALIGN, "addresses and strides must be whole 16-byte pieces");
    const Plan p = plan_of(tokens, heads, pages, batch, most_rows);
    if (workspace_bytes < workspace_of(p, pages->head_dim))
        return fail(TL_ERR_SIZE, "workspace has %lld bytes, %lld needed", (long long)workspace_bytes, (long long)workspace_of(p, pages->head_dim));
    a.q = static_cast<const __half*>(q), a.q_t = q_token, a.q_h = q_head;
    a.out = static_cast<__half*>(out);
    a.heads = heads, a.group = heads / pages->kv_heads;
    a.tile_heads = std::min(a.group, p.rows);
    a.blocks = (int)ceil_div(a.group, a.tile_heads);
    a.tile_tokens = p.rows / a.tile_heads;
    // the walk's products of costs stay below 2^53
    const int64_t keys = (int64_t)batch->table_pages * pages->page_size;
    const int64_t units = (ceil_div(tokens, a.tile_tokens) + batch->seqs) * pages->kv_heads * a.blocks;
    if (keys > (1 << 26) || units > (1ll << 42) / (keys + tokens + p.fixed + a.tile_tokens))
        return fail(TL_ERR_SHAPE, "%lld rows over up to %lld keys are more than one call takes", (long long)tokens, (long long)keys);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.fixed = p.fixed;
    a.least = p.least;
    a.uncut = p.uncut;
    a.shared = static_cast<Shared*>(workspace);
    a.pieces = reinterpret_cast<float*>(a.shared + p.workgroups);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool bytes = pages->dtype == TL_E4M3;
    switch (pages->head_dim) {
        case 64: bytes ? launch_attention<64, true>(a, p, st) : launch_attention<64, false>(a, p, st); break;
        case 128: bytes ? launch_attention<128, true>(a, p, st) : launch_attention<128, false>(a, p, st); break;
        default: bytes ? launch_attention<256, true>(a, p, st) : launch_attention<256, false>(a, p, st);
    }
    return finish_launch();
}
