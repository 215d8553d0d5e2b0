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
    int least;                                   // cost of a workgroup's part, 1 or more
    float* pieces;                               // [workgroups][2][rows][head_dim + 4]
    Shared* shared;                              // [workgroups]
};

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

// Cost of a key head's first `tiles` units: unit i costs before + (i + 1) * tile_tokens.
__device__ __forceinline__ long long tiles_cost(const PagedAttn& a, int before, int tiles)
{
    return (long long)tiles * before + (long long)a.tile_tokens * tiles * (tiles + 1ll) / 2;
}

__device__ __forceinline__ long long seq_cost(const PagedAttn& a, int b)
{
    if (b >= a.batch.seqs) return 0;
    const Seq s = sequence(a, b);
    return tiles_cost(a, s.before, s.tiles) * (a.pages.kv_heads * a.blocks);
}

// The workgroup's part of the list, and where it stands in it.
struct Walk {
    int wg, wgs;                                 // this workgroup, and how many have a part
    long long total, from, to;                   // the part
    long long at;                                // where the present unit begins
    int b, head, tile;                           // the unit: sequence, key head and block of query heads, rows
    Seq s;
};

__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long long scalar(long long v)
{
    return (long long)(((unsigned long long)(uint32_t)scalar((int)(v >> 32)) << 32) | (uint32_t)scalar((int)v));
}

// By a whole workgroup of 256 threads.  False where it has no part.
__device__ __forceinline__ bool begin_walk(const PagedAttn& a, Walk& w)
{
    __shared__ long long sums[4];
    __shared__ long long found_at;
    __shared__ int found_b;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr int kPass = 256 * kSeqsOfThread;
    const int seqs = a.batch.seqs;
    long long cost[kSeqsOfThread], upto = 0, total = 0, pass = 0;
    // costs of this thread's sequences from `first` on, and the sum of all before and of its own
    auto look = [&](int first) {
        long long own = 0;
#pragma unroll
        for (int i = 0; i < kSeqsOfThread; ++i) own += cost[i] = seq_cost(a, first + tid * kSeqsOfThread + i);
        upto = own;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const long long below = __shfl_up(upto, off, 64);
            if (lane >= off) upto += below;
        }
        __syncthreads();
        if (lane == 63) sums[wave] = upto;
        __syncthreads();
        pass = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i < wave) upto += sums[i];
            pass += sums[i];
        }
    };
    for (int first = 0; first < seqs; first += kPass) {
        look(first);
        total += pass;
    }
    total = scalar(total);
    // as many parts as there are workgroups, but none of less than `least`; neighbours of the list stay in one part of the chip, whose
    // cache they share
    w.wgs = (int)min((total + a.least - 1) / a.least, (long long)gridDim.x);
    const int eighth = (w.wgs + 7) / 8, inside = (int)blockIdx.x / 8;
    w.wg = inside < eighth ? ((int)blockIdx.x & 7) * eighth + inside : (int)blockIdx.x;
    if (w.wg >= w.wgs) {
        if (tid == 0) a.shared[w.wg].last = -1;
        return false;
    }
    w.total = total;
    w.from = total * w.wg / w.wgs;
    w.to = total * (w.wg + 1) / w.wgs;
    long long below = 0;
    for (int first = 0;; first += kPass) {
        if (seqs > kPass) look(first);
        long long begins = below + upto;
#pragma unroll
        for (int i = kSeqsOfThread - 1; i >= 0; --i) {
            const long long ends = begins;
            begins -= cost[i];
            if (begins <= w.from && w.from < ends) found_b = first + tid * kSeqsOfThread + i, found_at = begins;
        }
        below += pass;
        if (w.from < below) break;               // (the same for all: the list ends behind the part)
    }
    __syncthreads();
    w.b = scalar(found_b);
    w.at = scalar(found_at);
    w.s = sequence(a, w.b);
    const long long head_cost = tiles_cost(a, w.s.before, w.s.tiles);
    w.head = (int)((w.from - w.at) / head_cost);
    w.at += w.head * head_cost;
    int low = 0, high = w.s.tiles - 1;           // the last unit that begins no later
    while (low < high) {
        const int middle = (low + high + 1) / 2;
        if (w.at + tiles_cost(a, w.s.before, middle) <= w.from) low = middle;
        else high = middle - 1;
    }
    w.tile = low;
    w.at += tiles_cost(a, w.s.before, low);
    return true;
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
        w.s = sequence(a, w.b);
    } while (w.s.tiles == 0);
    return true;
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
    u.cost = (long long)w.s.before + (w.tile + 1ll) * a.tile_tokens;
    u.first_token = w.tile * a.tile_tokens;
    u.kv_head = w.head / a.blocks;
    u.first_head = (w.head - u.kv_head * a.blocks) * a.tile_heads;
    const int seen = max(w.s.length - w.s.n + min(u.first_token + a.tile_tokens, w.s.n), 0);   // by its last row
    u.begins = w.at >= w.from;
    const bool ends = w.at + u.cost <= w.to;
    u.whole = u.begins && ends;
    auto cut = [&](long long at) { return (int)min((at - w.at + kRound - 1) / kRound * kRound, (long long)seen); };
    u.first_key = u.begins ? 0 : cut(w.from);
    u.end_key = ends ? seen : cut(w.to);
    u.piece = a.pieces + ((long long)w.wg * 2 + (u.begins ? 1 : 0)) * ROWS * (HD + 4);
    return u;
}

// By one thread, once it has the last unit of its part: what the second launch has to join.
__device__ __forceinline__ void tell_shared(const PagedAttn& a, const Walk& w, const Unit& u)
{
    Shared s{w.b, w.head, w.tile, -1};
    if (u.begins && !u.whole) s.last = (int)(((w.at + u.cost) * w.wgs + w.total - 1) / w.total) - 1;
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

// The running softmax of one fragment of 16 rows over COUNT fragments of 16 keys: scores in, probabilities out (as the operand of the
// product with the values), the sums so far shrunk where the maximum moved.
template <int COUNT, int DF>
__device__ __forceinline__ void softmax_step(f32x4 (&sc)[COUNT], float scale_log2, float& top, float& sum, f32x4 (&o)[DF], u32x4 (&px)[COUNT / 2])
{
    float most = sc[0][0];
#pragma unroll
    for (int n = 0; n < COUNT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) most = fmaxf(most, sc[n][i]);
    most = with_other_rows(most, [](float x, float y) { return fmaxf(x, y); });
    const float now = fmaxf(top, most);
    const float base = now == kNone ? 0.f : now * scale_log2;      // (nothing but -inf so far)
    const float shrink = __builtin_amdgcn_exp2f(fmaf(top, scale_log2, -base));
    top = now;
    float part = 0.f;
#pragma unroll
    for (int n = 0; n < COUNT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float2v e;
#pragma unroll
            for (int j = 0; j < 2; ++j) e[j] = __builtin_amdgcn_exp2f(fmaf(sc[n][2 * i + j], scale_log2, -base));
            part += e[0];
            part += e[1];
            px[n >> 1][(n & 1) * 2 + i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(e, half2v));
        }
    sum = fmaf(sum, shrink, part);
    if (__builtin_amdgcn_ballot_w64(shrink != 1.0f) != 0) {
#pragma unroll
        for (int d = 0; d < DF; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] *= shrink;
    }
}

// A workgroup of four waves holds 64 * QF rows, a wave QF fragments of 16, and walks its units' keys in tiles of KT, one pass.
// The scores are computed transposed, keys x rows: a lane then holds, for ONE row (lane % 16), four neighbouring keys of every
// fragment -- the maximum and sum take two cross-lane steps a tile, and what it holds is already its operand of the second product
// (values^T x probabilities).  The values lie in LDS as they come, rows of a key, and are read by columns (column_read).
// LDS: two buffers of a tile of keys (pieces of 16 bytes swizzled so that the 16 keys of a read hit all banks) and of values (32-byte
// pairs swizzled so that the eight keys of a read do).  8-bit rows are turned into fp16 between the load and LDS, exactly.  The next
// tile is on its way into registers while this one is worked on; one barrier a tile.
template <int HD, int QF, bool BYTES>
__global__ __launch_bounds__(256, 2) void tl_paged_rows(PagedAttn a)
{
    constexpr int ROWS = 64 * QF, KT = HD == 256 ? 32 : 64, NF = KT / 16, KS = HD / 32, DF = HD / 16;
    constexpr int KB = KT * HD * 2, BUF = 2 * KB;
    constexpr int VALUES = BYTES ? 16 : 8, PIECES = HD / VALUES, KL = KT * PIECES / 256;    // of 16 bytes in the pages
    __shared__ __align__(16) unsigned char lds[2 * BUF];
    __shared__ int wrong_somewhere;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6);
    const int g = lane >> 4, r16 = lane & 15;
    Walk w;
    if (!begin_walk(a, w)) return;
    auto key_place = [](int key, int p) { return HD == 64 ? p ^ ((key >> 1) & 7) : p ^ (key & 15); };
    auto value_place = [](int key, int pair) { return HD == 64 ? pair ^ ((key >> 1) & 3) : pair ^ (key & 7); };
    for (;;) {
        const Unit u = unit_of<ROWS, HD>(a, w);
        const int first_tile = (u.first_key + KT - 1) / KT, tiles = (u.end_key + KT - 1) / KT;   // (a share may be empty)
        bool wrong = w.s.wrong;
        // ---- tiles on their way ----
        const long long head_at = u.kv_head * a.pages.head_stride;
        const int* ids = a.batch.table + w.b * a.batch.table_stride;
        u32x4 kreg[KL], vreg[KL];
        int kexp[KL], vexp[KL];
        auto fetch = [&](int t) {
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const int group_key = t * KT + (i * 256 + wave * 64) / PIECES;              // a wave's rows of one i share a page
                int page = ids[min(group_key, w.s.length - 1) >> a.pages.shift];
                page = scalar(page);
                const bool known = (unsigned)page < a.pages.pages;
                wrong |= !known;
                page = known ? page : 0;
                const int key = group_key + lane / PIECES, slot = min(key, w.s.length - 1) & ((1 << a.pages.shift) - 1);
                const long long at = page * a.pages.page_stride + head_at;
                const unsigned within = (unsigned)slot * (unsigned)a.pages.slot_stride + (unsigned)(lane % PIECES) * VALUES;
                const bool there = key < w.s.length;
                if constexpr (BYTES) {
                    kreg[i] = *reinterpret_cast<const u32x4*>(static_cast<const unsigned char*>(a.pages.k) + at + within);
                    vreg[i] = there ? *reinterpret_cast<const u32x4*>(static_cast<const unsigned char*>(a.pages.v) + at + within) : u32x4{0u, 0u, 0u, 0u};
                    const long long e = (((long long)page * a.pages.kv_heads + u.kv_head) << a.pages.shift) + slot;
                    kexp[i] = a.pages.k_exp[e];
                    vexp[i] = a.pages.v_exp[e];
                } else {
                    kreg[i] = *reinterpret_cast<const u32x4*>(static_cast<const __half*>(a.pages.k) + at + within);
                    // (a key past the end weighs 0, which would make NaN of a value that is not finite)
                    vreg[i] = there ? *reinterpret_cast<const u32x4*>(static_cast<const __half*>(a.pages.v) + at + within) : u32x4{0u, 0u, 0u, 0u};
                }
            }
        };
        auto put = [&](int buf) {
            unsigned char* kd = lds + buf * BUF;
            unsigned char* vd = kd + KB;
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const int id = i * 256 + tid, key = id / PIECES, p = id % PIECES;
                if constexpr (BYTES) {
                    u32x4 lo, hi;
                    sixteen_halves(kreg[i], __uint_as_float((uint32_t)kexp[i] << 23), &lo, &hi);
                    *reinterpret_cast<u32x4*>(kd + key * HD * 2 + key_place(key, 2 * p) * 16) = lo;
                    *reinterpret_cast<u32x4*>(kd + key * HD * 2 + key_place(key, 2 * p + 1) * 16) = hi;
                    sixteen_halves(vreg[i], __uint_as_float((uint32_t)vexp[i] << 23), &lo, &hi);
                    u32x4* v = reinterpret_cast<u32x4*>(vd + key * HD * 2 + value_place(key, p) * 32);
                    v[0] = lo;
                    v[1] = hi;
                } else {
                    *reinterpret_cast<u32x4*>(kd + key * HD * 2 + key_place(key, p) * 16) = kreg[i];
                    *reinterpret_cast<u32x4*>(vd + key * HD * 2 + value_place(key, p >> 1) * 32 + (p & 1) * 16) = vreg[i];
                }
            }
        };
        if (first_tile < tiles) fetch(first_tile);

        // ---- the wave's rows ----
        u32x4 qx[QF][KS];
        int last[QF];                                             // the last key that this lane's row sees
        int wave_last = -1;
        f32x4 o[QF][DF];
        float top[QF], sum[QF];
#pragma unroll
        for (int f = 0; f < QF; ++f) {
            const Row x = row_of(a, w, u, wave * 16 * QF + f * 16 + r16);
            last[f] = x.there ? w.s.length - w.s.n + x.token : -1;
            const __half* row = a.q + (long long)(w.s.start + x.token) * a.q_t + x.head * a.q_h + g * 8;
#pragma unroll
            for (int s = 0; s < KS; ++s) qx[f][s] = x.there ? *reinterpret_cast<const u32x4*>(row + s * 32) : u32x4{0u, 0u, 0u, 0u};
            top[f] = kNone;
            sum[f] = 0.f;
#pragma unroll
            for (int d = 0; d < DF; ++d) o[f][d] = f32x4{0.f, 0.f, 0.f, 0.f};
            wave_last = max(wave_last, last[f]);
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) wave_last = max(wave_last, __shfl_xor(wave_last, off, 64));
        wave_last = scalar(wave_last);
        int wave_first = INT_MAX;                                 // the last key that all its rows see
#pragma unroll
        for (int f = 0; f < QF; ++f) wave_first = min(wave_first, last[f]);
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) wave_first = min(wave_first, __shfl_xor(wave_first, off, 64));
        wave_first = scalar(wave_first);

        __syncthreads();                                          // the unit before is done with LDS
        if (tid == 0) wrong_somewhere = 0;
        if (first_tile < tiles) put(0);
        __syncthreads();
#pragma unroll
        for (int f = 0; f < QF; ++f)
#pragma unroll
            for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qx[f][s]));   // (here before the loop: waited for inside it, the next tile's loads are too)

        for (int t = first_tile; t < tiles; ++t) {
            if (t + 1 < tiles) fetch(t + 1);
            const unsigned char* ks = lds + ((t - first_tile) & 1) * BUF;
            const unsigned char* vs = ks + KB;
            if (t * KT <= wave_last) {                            // (a tile of which the wave's rows see nothing is skipped)
                f32x4 sc[QF][NF];
#pragma unroll
                for (int i = 0; i < NF * KS; ++i) {
                    const int s = HD == 64 ? i % KS : i / NF, n = HD == 64 ? i / KS : i % NF, key = n * 16 + r16;
                    const u32x4 kx = *reinterpret_cast<const u32x4*>(ks + key * HD * 2 + key_place(key, s * 4 + g) * 16);
#pragma unroll
                    for (int f = 0; f < QF; ++f) sc[f][n] = matrix_step<false>(kx, qx[f][s], s == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[f][n]);
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
#pragma unroll
                for (int f = 0; f < QF; ++f) softmax_step(sc[f], a.scale_log2, top[f], sum[f], o[f], px[f]);
#pragma unroll
                for (int s = 0; s < NF / 2; ++s)
#pragma unroll
                    for (int d = 0; d < DF; ++d) {
                        const int key = s * 32 + g * 4 + (r16 >> 2);
                        const unsigned char* from = vs + key * HD * 2 + value_place(key, d) * 32 + (r16 & 3) * 8;
                        const uint2 x = column_read(from), y = column_read(from + 16 * HD * 2);   // (16 keys on: the same swizzle)
                        const u32x4 vx{x.x, x.y, y.x, y.y};
#pragma unroll
                        for (int f = 0; f < QF; ++f) o[f][d] = matrix_step<false>(vx, px[f][s], o[f][d]);
                    }
            }
            if (t + 1 < tiles) {
                put((t + 1 - first_tile) & 1);                    // (read last before the barrier of the turn before)
                __syncthreads();
            }
        }
        if (wrong && lane == 0) wrong_somewhere = 1;
        __syncthreads();
        wrong = wrong_somewhere != 0;
#pragma unroll
        for (int f = 0; f < QF; ++f) {
            const int r = wave * 16 * QF + f * 16 + r16;
            const Row x = row_of(a, w, u, r);
            float all = with_other_rows(sum[f], [](float v, float y) { return v + y; });
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
                if (g == 0) row[HD] = top[f], row[HD + 1] = all;
            }
        }
        if (last_unit(w, u)) {
            if (tid == 0) tell_shared(a, w, u);
            return;
        }
        if (!next_unit(a, w, u.cost)) return;
    }
}

// Joins the pieces of the units that were shared out: blockIdx.x is the workgroup in which one begins.  HD / 4 lanes take a row, four
// values each, and 1024 / HD of them at a time its pieces.
template <int HD, int ROWS>
__global__ __launch_bounds__(256) void tl_paged_join(PagedAttn a)
{
    constexpr int LANES = HD / 4, AT_ONCE = 256 / LANES;
    __shared__ float4 part[256];
    __shared__ float tops[AT_ONCE], sums[AT_ONCE];
    const Shared sh = a.shared[blockIdx.x];
    if (sh.last < 0) return;
    Walk w{};
    w.b = sh.seq, w.head = sh.head, w.tile = sh.tile;
    w.s = sequence(a, w.b);
    const Unit u = unit_of<ROWS, HD>(a, w);
    const int first = (int)blockIdx.x, count = sh.last - first + 1;
    const int lane = (int)threadIdx.x % LANES, own = (int)threadIdx.x / LANES;
    for (int r = (int)blockIdx.y; r < ROWS; r += (int)gridDim.y) {
        const Row x = row_of(a, w, u, r);
        if (!x.there) continue;                                   // (the same for all)
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = kNone, sum = 0.f;
        for (int i = own; i < count; i += AT_ONCE) {
            const float* piece = a.pieces + (((long long)(first + i) * 2 + (i == 0 ? 1 : 0)) * ROWS + r) * (HD + 4);
            const float m = piece[HD], l = piece[HD + 1];
            const float4 v = *reinterpret_cast<const float4*>(piece + lane * 4);
            const float now = fmaxf(top, m), base = now == kNone ? 0.f : now * a.scale_log2;
            const float old = __builtin_amdgcn_exp2f(fmaf(top, a.scale_log2, -base)), fresh = __builtin_amdgcn_exp2f(fmaf(m, a.scale_log2, -base));
            o = make_float4(o.x * old + v.x * fresh, o.y * old + v.y * fresh, o.z * old + v.z * fresh, o.w * old + v.w * fresh);
            sum = sum * old + l * fresh;
            top = now;
        }
        __syncthreads();                                          // the row before is done with LDS
        part[threadIdx.x] = o;
        if (lane == 0) tops[own] = top, sums[own] = sum;
        __syncthreads();
        if (own == 0) {
            float most = tops[0];
#pragma unroll
            for (int i = 1; i < AT_ONCE; ++i) most = fmaxf(most, tops[i]);
            const float base = most == kNone ? 0.f : most * a.scale_log2;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            float all = 0.f;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const float weight = __builtin_amdgcn_exp2f(fmaf(tops[i], a.scale_log2, -base));
                const float4 v = part[i * LANES + lane];
                y = make_float4(y.x + v.x * weight, y.y + v.y * weight, y.z + v.z * weight, y.w + v.w * weight);
                all += sums[i] * weight;
            }
            const float inv = all == 0.f ? 0.f : 1.0f / all;
            const __half h[4] = {__float2half(y.x * inv), __float2half(y.y * inv), __float2half(y.z * inv), __float2half(y.w * inv)};
            *reinterpret_cast<uint2*>(a.out + ((long long)(w.s.start + x.token) * a.heads + x.head) * HD + lane * 4) = *reinterpret_cast<const uint2*>(h);
        }
    }
}

// What a call takes: rows of a unit, workgroups at most, and the cost below which a part is not cut.
struct Plan {
    int rows, workgroups, least;
};

Plan plan_of(int heads, const tl_pages* pages, int64_t most_rows)
{
    (void)heads, (void)pages, (void)most_rows;
    return Plan{64, (int)ceil_div(2 * compute_units(), 8) * 8, 512};
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

template <int HD, bool BYTES>
void launch_attention(const PagedAttn& a, const Plan& p, hipStream_t st)
{
    hipLaunchKernelGGL((tl_paged_rows<HD, 1, BYTES>), dim3((unsigned)p.workgroups), dim3(256), 0, st, a);
    hipLaunchKernelGGL((tl_paged_join<HD, 64>), dim3((unsigned)p.workgroups, 8), dim3(256), 0, st, a);
}

}  // namespace

extern "C" int tl_paged_attention_workspace(int heads, const tl_pages* pages, int64_t most_rows, int64_t* bytes)
{
    if (int rc = check_heads(heads, pages)) return rc;
    if (!bytes || most_rows < 0) return fail(TL_ERR_ARG, "bytes is null or most_rows negative");
    *bytes = workspace_of(plan_of(heads, pages, most_rows), pages->head_dim);
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
    if (!(scale > 0.f) || scale > 3e38f) return fail(TL_ERR_ARG, "scale=%g is not a positive number", (double)scale);
    if (!in_pieces(q, {q_token, q_head}, 2) || !in_pieces(out, {}, 2) || !in_pieces(workspace, {}, 1)) return fail(TL_ERR_ALIGN, "addresses and strides must be whole 16-byte pieces");
    const Plan p = plan_of(heads, pages, most_rows);
    if (workspace_bytes < workspace_of(p, pages->head_dim))
        return fail(TL_ERR_SIZE, "workspace has %lld bytes, %lld needed", (long long)workspace_bytes, (long long)workspace_of(p, pages->head_dim));
    a.q = static_cast<const __half*>(q), a.q_t = q_token, a.q_h = q_head;
    a.out = static_cast<__half*>(out);
    a.heads = heads, a.group = heads / pages->kv_heads;
    a.tile_heads = std::min(a.group, p.rows);
    a.blocks = (int)ceil_div(a.group, a.tile_heads);
    a.tile_tokens = p.rows / a.tile_heads;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.least = p.least;
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
