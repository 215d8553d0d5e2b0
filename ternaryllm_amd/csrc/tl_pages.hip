// Heads of queries and keys normalised and rotated, on their own or on their way into the pages of a cache, and rows read back
// out of the pages (the reference's apply_rotary_pos_emb and Cache.update, ternaryLLM_GPU/TernaryLLM/TernaryAttn.py:91-98, for
// sequences of different lengths).
#include <climits>

#include "tl_paged.h"

using namespace tl;

namespace tl {

int take_pages(const tl_pages* g, const tl_page_batch* c, int64_t tokens, Pages* p, Batch* b)
{
    if (!g || !c || !g->k || !g->v || (c->seqs != 0 && (!c->table || !c->starts || !c->lengths))) return fail(TL_ERR_ARG, "null pointer");
    if (g->dtype != TL_F16 && g->dtype != TL_E4M3) return fail(TL_ERR_DTYPE, "pages of dtype code %d unknown", g->dtype);
    if ((g->dtype == TL_E4M3) != (g->k_exponents && g->v_exponents)) return fail(TL_ERR_ARG, "pages have exponents if and only if they are of 8 bits");
    if (g->page_size < 16 || g->page_size > 1024 || (g->page_size & (g->page_size - 1))) return fail(TL_ERR_SHAPE, "page_size=%d is not a power of two from 16 to 1024", g->page_size);
    if (g->pages <= 0 || g->pages > INT32_MAX || g->kv_heads <= 0 || g->kv_heads > (1 << 16)) return fail(TL_ERR_SHAPE, "pages and kv_heads must be positive");
    if (g->head_dim <= 0 || g->head_dim % 16 || g->head_dim > 512) return fail(TL_ERR_SHAPE, "head_dim=%d is not a multiple of 16 up to 512", g->head_dim);
    if (g->slot_stride < g->head_dim || g->head_stride <= 0 || g->page_stride <= 0 || g->slot_stride > (1 << 30) / g->page_size)
        return fail(TL_ERR_SHAPE, "strides of the pages must be positive, and a head's slots within 2^30 elements");
    if (c->seqs < 0 || c->table_pages < 0 || c->table_stride < c->table_pages || (int64_t)c->table_pages * g->page_size > INT32_MAX)
        return fail(TL_ERR_SHAPE, "the page table has %d x %d pages, rows %lld apart", c->seqs, c->table_pages, (long long)c->table_stride);
    if (tokens < 0 || tokens > (1 << 28)) return fail(TL_ERR_SHAPE, "%lld rows", (long long)tokens);
    const int64_t es = g->dtype == TL_F16 ? 2 : 1;
    if (!in_pieces(g->k, {g->page_stride, g->head_stride, g->slot_stride}, es) || !in_pieces(g->v, {}, es))
        return fail(TL_ERR_ALIGN, "addresses and strides of the pages must be whole 16-byte pieces");
    *p = Pages{g->k, g->v, static_cast<unsigned char*>(g->k_exponents), static_cast<unsigned char*>(g->v_exponents), g->page_stride, g->head_stride,
               g->slot_stride, (unsigned)g->pages, __builtin_ctz((unsigned)g->page_size), g->kv_heads, g->head_dim};
    *b = Batch{c->table, c->starts, c->lengths, c->table_stride, c->table_pages, c->seqs, (int)tokens};
    return TL_OK;
}

}  // namespace tl

namespace {

constexpr int kHalf = 256;                      // pairs of the longest head

struct Rows {
    const void* x;
    long long x_t, x_h;
    void* y;
    long long y_t, y_h;
    const void* w;
    int heads;
};

struct RopeHeads {
    Rows q, k, v;                               // v: without norm and rotation
    const double* freq;
    const long long* positions;
    int hd, pairs, interleaved;
    int first;                                  // row of this launch
    float factor, eps;
    Pages pages;
    Batch batch;
};

enum Where { kRows, kHalfPages, kBytePages };   // where keys and values go

typedef float float2v __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// Eight neighbouring values as they lie, and as fp32.
template <typename T>
struct Raw {
    u32x4 a[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw<T> raw_eight(const T* p)
{
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.a[i] = reinterpret_cast<const u32x4*>(p)[i];
    return r;
}

struct Eight {
    float v[8];
    template <typename T>
    __device__ __forceinline__ void set(const Raw<T>& r)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 2) v[i] = to_f(__builtin_bit_cast(__half, (unsigned short)(r.a[0][i >> 1] >> (i & 1) * 16)));
            else v[i] = __uint_as_float(r.a[i >> 2][i & 3]);
        }
    }
    template <typename U>
    __device__ __forceinline__ void store(U* p) const
    {
        if constexpr (sizeof(U) == 2) {
            u32x4 h;
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v{settled(v[2 * i]), settled(v[2 * i + 1])}), half2v));
            *reinterpret_cast<u32x4*>(p) = h;
        } else {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
};

// f over the 2^bits neighbouring lanes that share a head, on the vector unit: lanes a step apart, then mirrored groups, whose values are alike
// by then.
template <typename F>
__device__ __forceinline__ float over_lanes(float x, int bits, F f)
{
    auto with = [&](auto control) {
        return f(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(control)::value, 0xf, 0xf, true)));
    };
    if (bits > 0) x = with(std::integral_constant<int, 0xb1>{});      // 1, 0, 3, 2
    if (bits > 1) x = with(std::integral_constant<int, 0x4e>{});      // 2, 3, 0, 1
    if (bits > 2) x = with(std::integral_constant<int, 0x141>{});     // eight lanes mirrored
    if (bits > 3) x = with(std::integral_constant<int, 0x140>{});     // sixteen
    if (bits > 4) {
        const auto near = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = f(__uint_as_float(near[0]), __uint_as_float(near[1]));
    }
    if (bits > 5) {
        const auto far = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = f(__uint_as_float(far[0]), __uint_as_float(far[1]));
    }
    return x;
}

// The exponent of a row of 8-bit values: the least e with most <= 448 * 2^e = 1.75 * 2^(e + 8), -32 to 8.
__device__ __forceinline__ int row_exponent(float most)
{
    const uint32_t bits = __float_as_uint(most);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return min(max(e, -32), 8);
}

// Eight codes of x / 2^e.  The conversion rounds to the nearest, ties to even.  Only in rows of the largest exponent can a value be too large
// for it: it is held at the largest code that stands for a finite fp16 number.  What is not a number stays that.
__device__ __forceinline__ uint2 byte_codes(const float* x, int e)
{
    const float scale = __uint_as_float((uint32_t)(127 - e) << 23);
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = x[i] * scale;
    if (e == 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = c[i] != c[i] ? c[i] : fminf(fmaxf(c[i], -240.0f), 240.0f);
    }
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// A workgroup takes a token, 2^bits lanes one of its heads, a lane eight neighbouring values, a wave at a time heads of queries, of keys or of
// values.  The token's cosines and sines are made once, for all its heads: the angle in 64 bits, taken modulo a turn there (at position
// 10^6 an fp32 angle is off by 0.06), its sine and cosine in 32.  A value's partner is another lane's unless pairs are neighbours: rows
// cross in LDS, within their wave.  Everything is fp32 from the load to the one rounding of the result.
// Bound by memory, for few tokens by the trips to it in a row (the first kTurns heads of a group of lanes are asked for before the place and the
// angles are looked for), and nearly by the vector unit: with 280 instructions for eight values, addresses of 64 bits and a kind of head
// to each lane, 8192 tokens of 32 / 8 / 8 heads into pages of 8 bits took 72 us; 53 so (3.5 TB/s), 4096 tokens of 32 / 8 heads 22 (3.8 TB/s).
constexpr int kTurns = 4;

template <typename T, Where W>
__global__ __launch_bounds__(256) void tl_rope_heads_k(RopeHeads a, int bits)
{
    // the cosine and sine of pair i: float4 i / 8 of plane i % 8 / 2; a lane's eight values: half of them in each plane (lanes side by side hit all banks)
    __shared__ float4 turn[4][kHalf / 8];
    __shared__ float4 cross[2][256];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), token = a.first + (int)blockIdx.x;
    const int p = lane & ((1 << bits) - 1), d = p * 8, each = 64 >> bits, sub = lane >> bits;   // each: heads of a wave at a time
    const bool inside = d < a.hd;
    const int gq = (a.q.heads + each - 1) / each, gk = gq + (a.k.heads + each - 1) / each, groups = gk + (a.v.heads + each - 1) / each;
    // group g of heads: its kind, this lane's head and the first value's place behind the token's
    auto kind_of = [&](int g) { return g < gq ? 0 : g < gk ? 1 : 2; };
    auto head_of = [&](int g) { return (g - (g < gq ? 0 : g < gk ? gq : gk)) * each + sub; };
    const T* const from[3] = {static_cast<const T*>(a.q.x) + token * a.q.x_t, static_cast<const T*>(a.k.x) + token * a.k.x_t, static_cast<const T*>(a.v.x) + token * a.v.x_t};
    Raw<T> raw[kTurns];
    auto ask = [&](int first) {
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int g = first + 4 * i;
            if (g >= groups) continue;
            const int h = head_of(g);
            const unsigned at = (unsigned)h * (unsigned)(g < gq ? a.q.x_h : g < gk ? a.k.x_h : a.v.x_h) + (unsigned)d;
            if (inside && h < (g < gq ? a.q.heads : g < gk ? a.k.heads : a.v.heads)) raw[i] = raw_eight((g < gq ? from[0] : g < gk ? from[1] : from[2]) + at);
        }
    };
    ask(wave);
    Raw<T> weight[2];
    if (inside && a.q.w) weight[0] = raw_eight(static_cast<const T*>(a.q.w) + d);
    if (inside && a.k.w) weight[1] = raw_eight(static_cast<const T*>(a.k.w) + d);
    Place at{0, 0, 0};
    Slot slot{-1, 0};
    if constexpr (W != kRows) {
        at = place_of(a.batch, token);
        if (at.seq < 0) return;                                 // (the same for every wave)
        slot = slot_of(a.pages, a.batch, at);
        slot.page = __builtin_amdgcn_readfirstlane(slot.page);
        slot.slot = __builtin_amdgcn_readfirstlane(slot.slot);
    }
    if (a.pairs) {
        const long long position = a.positions ? a.positions[token] : (long long)at.index;
        for (int i = tid; i < a.pairs; i += 256) {
            double turns = (double)position * a.freq[i] * 0.15915494309189535;   // 1 / (2 pi)
            turns -= rint(turns);
            const float most = (float)turns, rest = (float)(turns - (double)most) * 6.2831853f;   // what the rounding to fp32 leaves, as an angle
            float s, c;
            sincospif(2.0f * most, &s, &c);
            const float cosine = fmaf(-s, rest, c), sine = fmaf(c, rest, s);
            reinterpret_cast<float2*>(&turn[(i & 7) >> 1][i >> 3])[i & 1] = make_float2(cosine * a.factor, sine * a.factor);
        }
        __syncthreads();
    }
    const int row = tid - p;                                    // this head's first lane, among all
    const bool whole = (a.pairs & 7) == 0;                      // the halves of a head are whole lanes
    const float part = 1.0f / (float)a.hd;
    for (int first = wave; first < groups; first += 4 * kTurns) {
        if (first > wave) ask(first);
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int g = first + 4 * i;
            if (g >= groups) break;
            const int kind = kind_of(g), h = head_of(g);
            const bool there = inside && h < (kind == 0 ? a.q.heads : kind == 1 ? a.k.heads : a.v.heads);
            Eight x;
            if (there) x.set(raw[i]);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) x.v[j] = 0.f;
            if (kind < 2 && (kind == 0 ? a.q.w : a.k.w)) {
                auto mean_of_squares = [&](float eps) {
                    float squares = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) squares = fmaf(x.v[j], x.v[j], squares);
                    return fmaf(over_lanes(squares, bits, [](float u, float v) { return u + v; }), part, eps);
                };
                float mean = mean_of_squares(a.eps);
                if constexpr (sizeof(T) == 4) {                 // heads whose squares leave the range of fp32: of x times a power of two, which cancels
                    const bool large = !(mean < __builtin_huge_valf()), small = mean < 0x1p-100f;
                    if (__builtin_amdgcn_ballot_w64(large || small) != 0) {
                        const float by = large ? 0x1p-70f : small ? 0x1p100f : 1.0f;
#pragma unroll
                        for (int j = 0; j < 8; ++j) x.v[j] *= by;
                        mean = mean_of_squares(a.eps * by * by);
                    }
                }
                // (a step of Newton's on the instruction's root: an error of all of a head's values alike turns more of its 8-bit codes than any other; of 0 and
                // infinity there is none)
                const float root = rsqrtf(mean);
                const float inv = root > 0.f && root < __builtin_huge_valf() ? fmaf(0.5f * root, fmaf(-mean * root, root, 1.0f), root) : root;
                Eight w;
                w.set(kind == 0 ? weight[0] : weight[1]);
                if (there) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x.v[j] *= inv * w.v[j];
                }
            }
            if (kind < 2 && a.interleaved) {
                if (d < 2 * a.pairs) {
                    const float4 t[2] = {turn[p & 1 ? 2 : 0][p >> 1], turn[p & 1 ? 3 : 1][p >> 1]};
                    const float cs[8] = {t[0].x, t[0].y, t[0].z, t[0].w, t[1].x, t[1].y, t[1].z, t[1].w};
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        if (d + j < 2 * a.pairs) {
                            const float c = cs[j], s = cs[j + 1], lo = x.v[j], hi = x.v[j + 1];
                            x.v[j] = fmaf(lo, c, -(hi * s));
                            x.v[j + 1] = fmaf(hi, c, lo * s);
                        }
                    }
                }
            } else if (kind < 2 && a.pairs) {
                cross[0][tid] = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
                cross[1][tid] = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                if (whole) {
                    if (d < 2 * a.pairs) {
                        const bool low = d < a.pairs;
                        const int other = low ? d + a.pairs : d - a.pairs, chunk = (low ? d : other) >> 3;
                        const float4 y0 = cross[0][row + (other >> 3)], y1 = cross[1][row + (other >> 3)];
                        const float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
                        const uint32_t sign = low ? 0x80000000u : 0u;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float4 t = turn[j][chunk];
                            x.v[2 * j] = fmaf(x.v[2 * j], t.x, __uint_as_float(__float_as_uint(y[2 * j] * t.y) ^ sign));
                            x.v[2 * j + 1] = fmaf(x.v[2 * j + 1], t.z, __uint_as_float(__float_as_uint(y[2 * j + 1] * t.w) ^ sign));
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool low = d + j < a.pairs;
                        const int pair = low ? d + j : d + j - a.pairs;
                        if (pair < a.pairs) {
                            const int other = low ? pair + a.pairs : pair;
                            const float2 t = reinterpret_cast<const float2*>(&turn[(pair & 7) >> 1][pair >> 3])[pair & 1];
                            const float y = reinterpret_cast<const float*>(&cross[(other & 7) >> 2][row + (other >> 3)])[other & 3] * t.y;
                            x.v[j] = fmaf(x.v[j], t.x, low ? -y : y);
                        }
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
            if (W == kRows || kind == 0) {
                T* to = kind == 0 ? static_cast<T*>(a.q.y) + token * a.q.y_t : static_cast<T*>(a.k.y) + token * a.k.y_t;
                if (there) x.store(to + ((unsigned)h * (unsigned)(kind == 0 ? a.q.y_h : a.k.y_h) + (unsigned)d));
            } else if constexpr (W != kRows) {
                const long long page = slot.page * a.pages.page_stride + slot.slot * a.pages.slot_stride;
                void* base = kind == 1 ? a.pages.k : a.pages.v;
                const long long to = page + h * a.pages.head_stride + d;
                if constexpr (W == kHalfPages) {
                    if (there && slot.page >= 0) x.store(static_cast<__half*>(base) + to);
                } else {
                    float most = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x.v[j]));
                    most = over_lanes(most, bits, [](float u, float v) { return fmaxf(u, v); });
                    const int e = row_exponent(most);
                    if (there && slot.page >= 0) {
                        *reinterpret_cast<uint2*>(static_cast<unsigned char*>(base) + to) = byte_codes(x.v, e);
                        if (p == 0) (kind == 1 ? a.pages.k_exp : a.pages.v_exp)[(((long long)slot.page * a.pages.kv_heads + h) << a.pages.shift) + slot.slot] = (unsigned char)(e + 127);
                    }
                }
            }
        }
    }
}

struct ReadPages {
    Pages pages;
    Batch batch;
    void *k_out, *v_out;
    long long out_t, out_h;
    int first;                                  // workgroup of this launch
};

// 2^bits lanes take a row of a token, a lane 16 bytes of it in the pages, a wave kReadTurns times as many rows as it has such lanes, all asked for at
// once; `waves` of them a token.  Bound by memory: while the four waves of a workgroup took a token, one turn each behind the trips to memory that
// find its page, 65536 tokens of 8 heads in 8 bits were 104 us (82 so); a wave for all of a token's 64 rows took 24.4 us for 17 K tokens in fp16 (23.5 so).
constexpr int kReadTurns = 4;

template <typename T, bool BYTES>
__global__ __launch_bounds__(256) void tl_read_pages_k(ReadPages a, int bits, int waves)
{
    constexpr int VALUES = BYTES ? 16 : 8;
    const int lane = (int)threadIdx.x & 63, id = __builtin_amdgcn_readfirstlane((a.first + (int)blockIdx.x) * 4 + ((int)threadIdx.x >> 6));
    const int token = id / waves, per_turn = 64 >> bits, rows = 2 * a.pages.kv_heads;
    if (token >= a.batch.tokens) return;
    const Place at = place_of(a.batch, token);
    if (at.seq < 0) return;
    const Slot slot = slot_of(a.pages, a.batch, at);
    const int d = (lane & ((1 << bits) - 1)) * VALUES, first = (id - token * waves) * kReadTurns * per_turn + (lane >> bits);
    if (d >= a.pages.hd) return;
    u32x4 raw[kReadTurns];
    int e[kReadTurns];
#pragma unroll
    for (int i = 0; i < kReadTurns; ++i) {
        const int row = first + i * per_turn, which = row >= a.pages.kv_heads, h = row - which * a.pages.kv_heads;
        if (row >= rows || slot.page < 0) continue;
        const long long from = slot.page * a.pages.page_stride + h * a.pages.head_stride + slot.slot * a.pages.slot_stride + d;
        raw[i] = *reinterpret_cast<const u32x4*>(static_cast<const char*>(which ? a.pages.v : a.pages.k) + from * (BYTES ? 1 : 2));
        if constexpr (BYTES) e[i] = (which ? a.pages.v_exp : a.pages.k_exp)[(((long long)slot.page * a.pages.kv_heads + h) << a.pages.shift) + slot.slot];
    }
#pragma unroll
    for (int i = 0; i < kReadTurns; ++i) {
        const int row = first + i * per_turn, which = row >= a.pages.kv_heads, h = row - which * a.pages.kv_heads;
        T* out = static_cast<T*>(which ? a.v_out : a.k_out);
        if (row >= rows || !out) continue;
        out += token * a.out_t + h * a.out_h + d;
        Eight x[VALUES / 8];
        if (slot.page < 0) {
#pragma unroll
            for (int j = 0; j < VALUES; ++j) x[j / 8].v[j % 8] = __builtin_nanf("");
        } else if constexpr (BYTES) {
            const float scale = ldexpf(1.0f, e[i] - 127);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[i][j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[i][j], true);
                float* v = x[j / 2].v + j % 2 * 4;
                v[0] = lo[0] * scale, v[1] = lo[1] * scale, v[2] = hi[0] * scale, v[3] = hi[1] * scale;
            }
        } else {
            x[0].set(Raw<__half>{{raw[i]}});
        }
#pragma unroll
        for (int j = 0; j < VALUES / 8; ++j) x[j].store(out + j * 8);
    }
}

// Lanes of a head of which each has `values`, as a power of two.
int lane_bits(int hd, int values)
{
    int bits = 0;
    while (values << bits < hd) ++bits;
    return bits;
}

int take_rows(const tl_head_rows* r, int64_t es, int64_t tokens, bool out, Rows* to)
{
    if (!r || r->heads == 0) {
        *to = Rows{nullptr, 0, 0, nullptr, 0, 0, nullptr, 0};
        return TL_OK;
    }
    if (r->heads < 0 || r->heads > (1 << 16)) return fail(TL_ERR_SHAPE, "%d heads", r->heads);
    if (tokens > 0 && (!r->x || (out && !r->y))) return fail(TL_ERR_ARG, "device pointer is null");
    if (!in_pieces(r->x, {r->x_token, r->x_head}, es) || (out && !in_pieces(r->y, {r->y_token, r->y_head}, es)) || !in_pieces(r->norm_weight, {}, es))
        return fail(TL_ERR_ALIGN, "addresses and strides must be whole 16-byte pieces");
    const int64_t reach = std::max(r->x_head, out ? r->y_head : 0);
    if (r->x_head < 0 || (out && r->y_head < 0) || reach > INT32_MAX / r->heads) return fail(TL_ERR_SHAPE, "a token's heads must lie within 2^31 elements, in order");
    *to = Rows{r->x, r->x_token, r->x_head, r->y, r->y_token, r->y_head, r->norm_weight, r->heads};
    return TL_OK;
}

int take_rotation(const tl_rotation* r, int hd, int64_t tokens, bool batch, RopeHeads* a)
{
    if (!r) return fail(TL_ERR_ARG, "null pointer");
    if (r->pairs < 0 || 2 * r->pairs > hd) return fail(TL_ERR_SHAPE, "%d pairs of values in heads of %d", r->pairs, hd);
    if (r->pairs && tokens > 0 && (!r->frequencies || (!r->positions && !batch))) return fail(TL_ERR_ARG, "device pointer is null");
    a->freq = r->frequencies;
    a->positions = reinterpret_cast<const long long*>(r->positions);
    a->hd = hd;
    a->pairs = r->pairs;
    a->interleaved = r->interleaved != 0;
    a->factor = r->factor;
    a->eps = r->eps;
    return TL_OK;
}

template <typename T>
void launch_rope(RopeHeads a, Where where, int64_t tokens, hipStream_t st)
{
    const dim3 block(256);
    const int bits = lane_bits(a.hd, 8);
    in_launches(tokens, [&](int first, dim3 grid) {
        a.first = first;
        if (where == kRows) hipLaunchKernelGGL((tl_rope_heads_k<T, kRows>), grid, block, 0, st, a, bits);
        else if (where == kHalfPages) hipLaunchKernelGGL((tl_rope_heads_k<T, kHalfPages>), grid, block, 0, st, a, bits);
        else hipLaunchKernelGGL((tl_rope_heads_k<T, kBytePages>), grid, block, 0, st, a, bits);
    });
}

}  // namespace

extern "C" int tl_rope_heads(const tl_head_rows* q, const tl_head_rows* k, int dtype, int64_t tokens, int head_dim, const tl_rotation* rotation, void* stream)
{
    if (int rc = check_dtype(dtype, "q")) return rc;
    if (tokens < 0 || tokens > (1 << 28)) return fail(TL_ERR_SHAPE, "%lld rows", (long long)tokens);
    if (head_dim <= 0 || head_dim % 8 || head_dim > 512) return fail(TL_ERR_UNSUPPORTED, "head_dim=%d (multiples of 8 up to 512 supported)", head_dim);
    const int64_t es = dtype == TL_F16 ? 2 : 4;
    RopeHeads a{};
    if (int rc = take_rows(q, es, tokens, true, &a.q)) return rc;
    if (int rc = take_rows(k, es, tokens, true, &a.k)) return rc;
    if (int rc = take_rotation(rotation, head_dim, tokens, false, &a)) return rc;
    if (tokens == 0 || a.q.heads + a.k.heads == 0) return TL_OK;
    if (dtype == TL_F16) launch_rope<__half>(a, kRows, tokens, static_cast<hipStream_t>(stream));
    else launch_rope<float>(a, kRows, tokens, static_cast<hipStream_t>(stream));
    return finish_launch();
}

extern "C" int tl_rope_to_pages(const tl_head_rows* q, const tl_head_rows* k, const tl_head_rows* v, int dtype, int64_t tokens, const tl_rotation* rotation,
                                const tl_pages* pages, const tl_page_batch* batch, void* stream)
{
    if (int rc = check_dtype(dtype, "k")) return rc;
    RopeHeads a{};
    if (int rc = take_pages(pages, batch, tokens, &a.pages, &a.batch)) return rc;
    const int64_t es = dtype == TL_F16 ? 2 : 4;
    const int hd = a.pages.hd;
    if (int rc = take_rows(q, es, tokens, true, &a.q)) return rc;
    if (int rc = take_rows(k, es, tokens, false, &a.k)) return rc;
    if (int rc = take_rows(v, es, tokens, false, &a.v)) return rc;
    if (a.k.heads != a.pages.kv_heads || a.v.heads != a.pages.kv_heads) return fail(TL_ERR_SHAPE, "k and v have %d and %d heads, the pages %d", a.k.heads, a.v.heads, a.pages.kv_heads);
    if (a.v.w) return fail(TL_ERR_ARG, "values are not normalised");
    if (int rc = take_rotation(rotation, hd, tokens, true, &a)) return rc;
    if (tokens == 0 || a.batch.seqs == 0) return TL_OK;
    const Where where = pages->dtype == TL_E4M3 ? kBytePages : kHalfPages;
    if (dtype == TL_F16) launch_rope<__half>(a, where, tokens, static_cast<hipStream_t>(stream));
    else launch_rope<float>(a, where, tokens, static_cast<hipStream_t>(stream));
    return finish_launch();
}

extern "C" int tl_read_pages(const tl_pages* pages, const tl_page_batch* batch, int64_t tokens, int dtype, void* k_out, void* v_out, int64_t out_token,
                             int64_t out_head, void* stream)
{
    if (int rc = check_dtype(dtype, "out")) return rc;
    ReadPages a{};
    if (int rc = take_pages(pages, batch, tokens, &a.pages, &a.batch)) return rc;
    const int64_t es = dtype == TL_F16 ? 2 : 4;
    if (!in_pieces(k_out, {out_token, out_head}, es) || !in_pieces(v_out, {}, es)) return fail(TL_ERR_ALIGN, "addresses and strides must be whole 16-byte pieces");
    a.k_out = k_out, a.v_out = v_out, a.out_t = out_token, a.out_h = out_head;
    if (tokens == 0 || a.batch.seqs == 0 || (!k_out && !v_out)) return TL_OK;
    const bool bytes = pages->dtype == TL_E4M3;
    const int bits = lane_bits(a.pages.hd, bytes ? 16 : 8), waves = (int)ceil_div(2 * a.pages.kv_heads, kReadTurns * (64 >> bits));
    const int64_t groups = ceil_div(tokens * waves, 4);
    if (groups > INT32_MAX / 4) return fail(TL_ERR_SHAPE, "%lld rows of %d heads are more than one launch takes", (long long)tokens, a.pages.kv_heads);
    hipStream_t st = static_cast<hipStream_t>(stream);
    auto launch = [&](auto kernel) {
        in_launches(groups, [&](int first, dim3 grid) {
            a.first = first;
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a, bits, waves);
        });
    };
    if (dtype == TL_F16) bytes ? launch(tl_read_pages_k<__half, true>) : launch(tl_read_pages_k<__half, false>);
    else bytes ? launch(tl_read_pages_k<float, true>) : launch(tl_read_pages_k<float, false>);
    return finish_launch();
}
