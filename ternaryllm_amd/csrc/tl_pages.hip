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
    if (g->slot_stride < g->head_dim || g->head_stride <= 0 || g->page_stride <= 0 || g->slot_stride * g->page_size > (1 << 30))
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
    float factor, eps;
    Pages pages;
    Batch batch;
};

enum Where { kRows, kHalfPages, kBytePages };   // where keys and values go

template <typename T>
struct EightOf {
    float v[8];
    __device__ __forceinline__ void load(const T* p)
    {
        if constexpr (sizeof(T) == 2) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f(__builtin_bit_cast(__half, (unsigned short)(a[i >> 1] >> (i & 1) * 16)));
        } else {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
    }
    template <typename U>
    __device__ __forceinline__ void store(U* p) const
    {
        if constexpr (sizeof(U) == 2) {
            __half h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = from_f<__half>(settled(v[i]));
            *reinterpret_cast<u32x4*>(p) = *reinterpret_cast<const u32x4*>(h);
        } else {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
};

// f over the 2^bits neighbouring lanes that share a head.
template <typename F>
__device__ __forceinline__ float over_lanes(float x, int bits, F f)
{
    for (int off = 1 << bits >> 1; off > 0; off >>= 1) x = f(x, __shfl_xor(x, off, 64));
    return x;
}

// The exponent of a row of 8-bit values: the least e with most <= 448 * 2^e = 1.75 * 2^(e + 8), -32 to 8.
__device__ __forceinline__ int row_exponent(float most)
{
    const uint32_t bits = __float_as_uint(most);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return min(max(e, -32), 8);
}

// Eight codes of x / 2^e.  The conversion rounds to the nearest, ties to even; what is too large for it is held at the largest
// code that stands for a finite fp16 number, what is not a number stays that.
__device__ __forceinline__ uint2 byte_codes(const float* x, int e)
{
    const float bound = e == 8 ? 240.0f : 448.0f, scale = __uint_as_float((uint32_t)(127 - e) << 23);
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = x[i] * scale;
        c[i] = y != y ? y : fminf(fmaxf(y, -bound), bound);
    }
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// A workgroup takes a token, 2^bits lanes one of its heads, a lane eight neighbouring values.  The token's cosines and sines
// are made once, for all its heads: the angle in 64 bits, taken modulo a turn there (at position 10^6 an fp32 angle is off by
// 0.06), its sine and cosine in 32.  A value's partner is another lane's unless pairs are neighbours: rows cross in LDS, within
// their wave.  Everything is fp32 from the load to the one rounding of the result.
template <typename T, Where W>
__global__ __launch_bounds__(256) void tl_rope_heads_k(RopeHeads a, int bits)
{
    __shared__ float turn[2 * kHalf];
    __shared__ __align__(16) float cross[256 * 8];
    const int tid = (int)threadIdx.x, token = (int)blockIdx.x;
    Place at{0, 0};
    Slot slot{-1, 0};
    if constexpr (W != kRows) {
        at = place_of(a.batch, token);
        if (at.seq < 0) return;                                 // (the same for every wave)
        slot = slot_of(a.pages, a.batch, at);
    }
    if (a.pairs) {
        const long long position = a.positions ? a.positions[token] : (long long)at.index;
        for (int i = tid; i < a.pairs; i += 256) {
            double turns = (double)position * a.freq[i] * 0.15915494309189535;   // 1 / (2 pi)
            turns -= rint(turns);
            float s, c;
            sincospif(2.0f * (float)turns, &s, &c);
            turn[2 * i] = c * a.factor;
            turn[2 * i + 1] = s * a.factor;
        }
        __syncthreads();
    }
    const int p = tid & ((1 << bits) - 1), d = p * 8, per_pass = 256 >> bits;
    const bool inside = d < a.hd;
    const int rows = a.q.heads + a.k.heads + a.v.heads;
    float* own = cross + (tid & ~((1 << bits) - 1)) * 8;        // this head's row
    for (int row = tid >> bits; row < rows; row += per_pass) {
        const int kind = row < a.q.heads ? 0 : row < a.q.heads + a.k.heads ? 1 : 2;
        const Rows& r = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
        const int h = row - (kind > 0 ? a.q.heads : 0) - (kind > 1 ? a.k.heads : 0);
        EightOf<T> x;
        if (inside) x.load(static_cast<const T*>(r.x) + token * r.x_t + h * r.x_h + d);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) x.v[i] = 0.f;
        if (kind < 2) {
            if (r.w) {
                float squares = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) squares = fmaf(x.v[i], x.v[i], squares);
                squares = over_lanes(squares, bits, [](float u, float v) { return u + v; });
                const float inv = 1.0f / sqrtf(squares / (float)a.hd + a.eps);
                EightOf<T> w;
                if (inside) {
                    w.load(static_cast<const T*>(r.w) + d);
#pragma unroll
                    for (int i = 0; i < 8; ++i) x.v[i] = x.v[i] * inv * w.v[i];
                }
            }
            if (a.interleaved) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const int pair = (d + i) >> 1;
                    if (pair < a.pairs) {
                        const float c = turn[2 * pair], s = turn[2 * pair + 1], lo = x.v[i], hi = x.v[i + 1];
                        x.v[i] = lo * c - hi * s;
                        x.v[i + 1] = hi * c + lo * s;
                    }
                }
            } else if (a.pairs) {
                reinterpret_cast<float4*>(own + d)[0] = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
                reinterpret_cast<float4*>(own + d)[1] = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool low = d + i < a.pairs;
                    const int pair = low ? d + i : d + i - a.pairs;
                    if (pair < a.pairs) {
                        const float c = turn[2 * pair], s = turn[2 * pair + 1], other = own[low ? pair + a.pairs : pair];
                        x.v[i] = low ? x.v[i] * c - other * s : x.v[i] * c + other * s;
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        }
        if (W == kRows || kind == 0) {
            if (inside) x.store(static_cast<T*>(r.y) + token * r.y_t + h * r.y_h + d);
        } else if constexpr (W != kRows) {
            const long long to = slot.page * a.pages.page_stride + h * a.pages.head_stride + slot.slot * a.pages.slot_stride + d;
            void* base = kind == 1 ? a.pages.k : a.pages.v;
            if constexpr (W == kHalfPages) {
                if (inside && slot.page >= 0) x.store(static_cast<__half*>(base) + to);
            } else {
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x.v[i]));
                most = over_lanes(most, bits, [](float u, float v) { return fmaxf(u, v); });
                const int e = row_exponent(most);
                if (inside && slot.page >= 0) {
                    *reinterpret_cast<uint2*>(static_cast<unsigned char*>(base) + to) = byte_codes(x.v, e);
                    if (p == 0) (kind == 1 ? a.pages.k_exp : a.pages.v_exp)[(((long long)slot.page * a.pages.kv_heads + h) << a.pages.shift) + slot.slot] = (unsigned char)(e + 127);
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
};

// A workgroup takes a token, 2^bits lanes one of its rows, a lane eight values.  Bound by memory.
template <typename T, bool BYTES>
__global__ __launch_bounds__(256) void tl_read_pages_k(ReadPages a, int bits)
{
    const int tid = (int)threadIdx.x, token = (int)blockIdx.x;
    const Place at = place_of(a.batch, token);
    if (at.seq < 0) return;
    const Slot slot = slot_of(a.pages, a.batch, at);
    const int d = (tid & ((1 << bits) - 1)) * 8;
    if (d >= a.pages.hd) return;
    for (int row = tid >> bits; row < 2 * a.pages.kv_heads; row += 256 >> bits) {
        const int which = row >= a.pages.kv_heads, h = row - which * a.pages.kv_heads;
        T* out = static_cast<T*>(which ? a.v_out : a.k_out);
        if (!out) continue;
        EightOf<__half> x;
        if (slot.page < 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x.v[i] = __builtin_nanf("");
        } else {
            const long long from = slot.page * a.pages.page_stride + h * a.pages.head_stride + slot.slot * a.pages.slot_stride + d;
            const void* base = which ? a.pages.v : a.pages.k;
            if constexpr (BYTES) {
                const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const unsigned char*>(base) + from);
                const int e = (which ? a.pages.v_exp : a.pages.k_exp)[(((long long)slot.page * a.pages.kv_heads + h) << a.pages.shift) + slot.slot];
                const float scale = ldexpf(1.0f, e - 127);
                const auto a0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, false), a1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, true);
                const auto a2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, false), a3 = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, true);
                x.v[0] = a0[0] * scale, x.v[1] = a0[1] * scale, x.v[2] = a1[0] * scale, x.v[3] = a1[1] * scale;
                x.v[4] = a2[0] * scale, x.v[5] = a2[1] * scale, x.v[6] = a3[0] * scale, x.v[7] = a3[1] * scale;
            } else {
                x.load(static_cast<const __half*>(base) + from);
            }
        }
        x.store(out + token * a.out_t + h * a.out_h + d);
    }
}

int lane_bits(int hd)
{
    int bits = 0;
    while (8 << bits < hd) ++bits;
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
void launch_rope(const RopeHeads& a, Where where, int64_t tokens, hipStream_t st)
{
    const dim3 grid((unsigned)tokens), block(256);
    const int bits = lane_bits(a.hd);
    if (where == kRows) hipLaunchKernelGGL((tl_rope_heads_k<T, kRows>), grid, block, 0, st, a, bits);
    else if (where == kHalfPages) hipLaunchKernelGGL((tl_rope_heads_k<T, kHalfPages>), grid, block, 0, st, a, bits);
    else hipLaunchKernelGGL((tl_rope_heads_k<T, kBytePages>), grid, block, 0, st, a, bits);
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
    const dim3 grid((unsigned)tokens), block(256);
    const int bits = lane_bits(a.pages.hd);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool bytes = pages->dtype == TL_E4M3;
    if (dtype == TL_F16) {
        if (bytes) hipLaunchKernelGGL((tl_read_pages_k<__half, true>), grid, block, 0, st, a, bits);
        else hipLaunchKernelGGL((tl_read_pages_k<__half, false>), grid, block, 0, st, a, bits);
    } else {
        if (bytes) hipLaunchKernelGGL((tl_read_pages_k<float, true>), grid, block, 0, st, a, bits);
        else hipLaunchKernelGGL((tl_read_pages_k<float, false>), grid, block, 0, st, a, bits);
    }
    return finish_launch();
}
