// What a ternary head's rows are worth: softmax cross entropy, and the divergence from a teacher whose top logits are known, with their gradients.
//
//   z_v = s_v / T * sum_k x_k W_kv,  lse = log sum_v exp z_v,  loss = T^2 (sum_i t_i log t_i + sum_i t_i (lse - z_i)),
//   dz_v = T (exp(z_v - lse) - t_v) times the gradient of the row's loss,  dx_k = sum_v dz_v s_v W_kv,  ds_v = sum over rows of dz_v * (sum_k x_k W_kv),
//
// t: the teacher's probabilities of the vocabulary's entries that it names, which add up to 1; of cross entropy, one entry of 1 and T = 1.
// The logits are not kept: the backward pass multiplies again.
#include "tl_loss.h"

using namespace tl;

namespace {

constexpr int kFewColumns = 128;                 // of a workgroup of tl_loss_few_grad
constexpr int kRowThreads = 1024, kJoinThreads = 256;   // of a workgroup that takes a row of logits, of what is left of them
constexpr float kNone = -__builtin_huge_valf(), kLn2 = 0.6931471805599453f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_huge_valf(); }

// A maximum and the sum of exponentials against it (E2: of 2), joined with another pair.  (Nothing yet: -inf and 0.)
template <bool E2>
__device__ __forceinline__ void join(float& top, float& sum, float top2, float sum2)
{
    const float now = fmaxf(top, top2), base = now == kNone ? 0.f : now;
    auto power = [](float x) { return E2 ? __builtin_amdgcn_exp2f(x) : __expf(x); };
    sum = sum * power(top - base) + sum2 * power(top2 - base);
    top = now;
}

// The same over a workgroup of WAVES waves; the result in all threads.
template <int WAVES, bool E2>
__device__ __forceinline__ void join_all(float& top, float& sum)
{
    __shared__ float tops[WAVES], sums[WAVES];
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) join<E2>(top, sum, __shfl_xor(top, off, 64), __shfl_xor(sum, off, 64));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top, sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    top = kNone, sum = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) join<E2>(top, sum, tops[i], sums[i]);
    __syncthreads();
}

template <int WAVES, typename F>
__device__ __forceinline__ float fold_all(float v, F f)
{
    __shared__ float parts[WAVES];
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v = f(v, __shfl_xor(v, off, 64));
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = v;
    __syncthreads();
    v = parts[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) v = f(v, parts[i]);
    __syncthreads();
    return v;
}

// The teacher of a row: what a row's ids and logits stand for.  A wave takes a row.  Repeated ids add up, in the place of the first of them; an entry of
// probability 0 and those added elsewhere get id -1.  known: sum t log t; +inf: the row has no teacher; NaN: one of its entries is none.  Bound by latency: 4.3 us
// for 40 rows of 8, 5.4 for 2048 of 32.
__global__ __launch_bounds__(64) void tl_teacher(TeacherArgs a)
{
    __shared__ __align__(16) int ids[kMostTop];
    __shared__ float shares[kMostTop];
    const int lane = (int)threadIdx.x;
    const long long row = blockIdx.x;
    const int64_t* from = a.ids + row * a.ids_ld;
    auto logit = [&](int i) { return (a.f16 ? __half2float(static_cast<const __half*>(a.logits)[row * a.logits_ld + i]) : static_cast<const float*>(a.logits)[row * a.logits_ld + i]) * a.cool; };
    float top = kNone;
    bool wrong = false;
    for (int i = lane; i < a.top; i += 64) {
        const float v = logit(i);
        wrong |= v != v;
        top = fmaxf(top, v);
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    const bool none = top == kNone;
    float sum = 0.f;
    for (int i = lane; i < a.top; i += 64) {
        const float v = logit(i), e = none ? 0.f : expf(v - top);
        const long long id = from[i];
        const bool outside = id < 0 || id >= a.N;
        wrong |= v > kNone && outside;           // (however little its probability)
        ids[i] = e > 0.f && !outside ? (int)id : -1;
        shares[i] = e;
        sum += e;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off, 64);
    wrong = __builtin_amdgcn_ballot_w64(wrong) != 0 || !(fabsf(top) < __builtin_huge_valf() || none);
    for (int i = a.top + lane; i < (a.top + 3) / 4 * 4; i += 64) ids[i] = -2;
    __syncthreads();
    float known = 0.f;
    for (int i = lane; i < a.top; i += 64) {
        int id = ids[i], same = 0;
        // how often it is there, four entries at a time; mostly that is once
#pragma unroll 4
        for (int j = 0; j < (a.top + 3) / 4; ++j) {
            const i32x4 x = reinterpret_cast<const i32x4*>(ids)[j];
#pragma unroll
            for (int e = 0; e < 4; ++e) same += x[e] == id;
        }
        float share = shares[i];
        if (id >= 0 && same > 1) {
            share = 0.f;
            for (int j = 0, of = id; j < a.top; ++j)
                if (ids[j] == of) {
                    if (j < i) id = -1;          // (added where it stands first)
                    share += shares[j];
                }
        }
        share = id < 0 ? 0.f : share / sum;
        a.entry[row * a.top + i] = wrong ? -1 : id;
        a.share[row * a.top + i] = share;
        known += share > 0.f ? share * logf(share) : 0.f;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) known += __shfl_xor(known, off, 64);
    if (lane == 0) a.known[row] = wrong ? __builtin_nanf("") : none ? __builtin_huge_valf() : known;
}

// The logarithm of a row's sum against its maximum, which differences from the maximum are added to: a large maximum would round most of it away.  NaN: no row
// of finite logits has such a maximum.
template <bool E2>
__device__ __forceinline__ float log_of(float top, float sum) { return finite(top) ? E2 ? log2f(sum) : logf(sum) : __builtin_nanf(""); }

// A row's divergence from sum t (lse - z), by one thread; lse: as it is kept.
__device__ __forceinline__ void put_divergence(const LossArgs& a, int row, float lse, float gap)
{
    const float known = a.known[row];
    const bool none = known == __builtin_huge_valf();
    a.loss[row] = none ? 0.f : a.heat * a.heat * (known + gap);
    a.lse[row] = none ? kNone : known == known ? lse : __builtin_nanf("");
}

// A row's loss from its maximum, its sum and its entries' logits (z(entry), each asked for by one thread of the workgroup; E2: all as exponents of 2), and what
// the backward pass wants of it: lse, NaN where the loss is, -inf for a row that counts for nothing.
template <int WAVES, bool E2, typename Z>
__device__ __forceinline__ void put_loss(const LossArgs& a, int row, float top, float sum, Z z)
{
    const int tid = (int)threadIdx.x;
    const float above = log_of<E2>(top, sum), lse = top + above;
    if (a.targets) {
        if (tid != 0) return;
        const long long target = a.targets[row];
        const bool counts = target != a.ignore, there = target >= 0 && target < a.N;
        const float loss = !counts ? 0.f : there ? (top - z((int)target, 0) + above) * (E2 ? kLn2 : 1.f) : __builtin_nanf("");
        a.loss[row] = loss;
        a.lse[row] = !counts ? kNone : there ? lse : __builtin_nanf("");
        return;
    }
    float gap = 0.f;
    for (int i = tid; i < a.top; i += WAVES * 64) {
        const int id = a.entry[(long long)row * a.top + i];
        if (id >= 0) gap = fmaf(a.share[(long long)row * a.top + i], top - z(id, i) + above, gap);
    }
    gap = fold_all<WAVES>(gap, [](float x, float y) { return x + y; });
    if (tid == 0) put_divergence(a, row, lse, gap * (E2 ? kLn2 : 1.f));
}

// f(the scales of four columns from 4 i on, and of a column), for scales of the call's kind.  (Loads that each ask for the kind are on their way one after the
// other, and those of a value each are many: 32000 of one workgroup's took 30 us, and 7.)
template <typename F>
__device__ __forceinline__ void with_scales(const LossArgs& a, F f)
{
    auto both = [&](auto type) {
        using T = decltype(type);
        typedef T four __attribute__((ext_vector_type(4)));
        const T* p = static_cast<const T*>(a.scale);
        auto one = [=](int n) { return (float)p[n]; };
        if (reinterpret_cast<uintptr_t>(p) % sizeof(four) == 0) f([=](int i) { return __builtin_convertvector(reinterpret_cast<const four*>(p)[i], f32x4); }, one);
        else f([=](int i) { return f32x4{one(4 * i), one(4 * i + 1), one(4 * i + 2), one(4 * i + 3)}; }, one);
    };
    if (!a.scale) f([](int) { return f32x4{1.f, 1.f, 1.f, 1.f}; }, [](int) { return 1.f; });
    else if (a.scale_f16) both(_Float16{});
    else both(float{});
}

// A logit from its product, as it is rounded in both passes.
__device__ __forceinline__ float logit_of(const LossArgs& a, float raw, float scale) { return rounded_product(rounded_product(raw, scale), a.cool); }

// The largest column scale, by one workgroup, where lse ends: what the gradients' fp16 probabilities are raised by goes by it.
template <int WAVES>
__device__ __forceinline__ void put_largest_scale(const LossArgs& a)
{
    constexpr int U = 8, THREADS = WAVES * 64;
    float most = a.scale ? 0.f : 1.f;
    bool wrong = false;
    auto look = [&](float s) { wrong |= !finite(s), most = fmaxf(most, fabsf(s)); };
    with_scales(a, [&](auto four, auto one) {
        const int whole = a.N / 4;
        for (int first = (int)threadIdx.x; first < whole; first += THREADS * U) {
            f32x4 s[U];
#pragma unroll
            for (int u = 0; u < U; ++u) s[u] = four(min(first + u * THREADS, whole - 1));
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) look(s[u][e]);
        }
        if ((int)threadIdx.x < a.N - 4 * whole) look(one(4 * whole + (int)threadIdx.x));
    });
    most = fold_all<WAVES>(wrong ? __builtin_huge_valf() : most, [](float x, float y) { return fmaxf(x, y); });
    if (threadIdx.x == 0) a.lse[a.M] = most;
}

// Few rows: their logits are in the workspace, without scales.  A workgroup takes a row, one more the scales.  Bound by latency: 6.4 us for
// a row of 32000, 7 for 16, as the scales' largest takes alone.
__global__ __launch_bounds__(kRowThreads) void tl_loss_few(LossArgs a)
{
    constexpr int WAVES = kRowThreads / 64, U = 4;
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x;
    if (row == a.M) {
        put_largest_scale<WAVES>(a);
        return;
    }
    const float* raw = a.raw + (long long)blockIdx.x * a.raw_ld;
    auto z = [&](int n) { return logit_of(a, raw[n], load_scale(a.scale, a.scale_f16, n)); };
    float top = kNone, sum = 0.f;
    bool wrong = false;
    with_scales(a, [&](auto four, auto one) {
        const int whole = a.N / 4;
        for (int first = tid; first < whole; first += kRowThreads * U) {
            f32x4 v[U], s[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = min(first + u * kRowThreads, whole - 1);
                v[u] = reinterpret_cast<const f32x4*>(raw)[i], s[u] = four(i);
            }
            float most = kNone, part = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[u][e] = first + u * kRowThreads < whole ? logit_of(a, v[u][e], s[u][e]) : kNone;
                    most = fmaxf(most, v[u][e]), wrong |= v[u][e] != v[u][e];
                }
            const float base = most == kNone ? 0.f : most;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) part += __expf(v[u][e] - base);
            join<false>(top, sum, most, part);
        }
        if (tid < a.N - 4 * whole) {
            const float v = logit_of(a, raw[4 * whole + tid], one(4 * whole + tid));
            wrong |= v != v;
            join<false>(top, sum, v, 1.f);
        }
    });
    // (a maximum passes over what is not a number; +inf does not count as a maximum either)
    if (wrong) top = __builtin_huge_valf();
    join_all<WAVES, false>(top, sum);
    put_loss<WAVES, false>(a, row, top, sum, [&](int n, int) { return z(n); });
}

// Many rows: a product has left maxima and sums of parts of their columns, and the logits that are wanted, all as exponents of 2.  A workgroup takes a row, one
// more the scales.
// 5 us for 40 rows of 500 parts, 12 for 4096 (16 MB).
__global__ __launch_bounds__(kJoinThreads) void tl_loss_join(LossArgs a, const float2* parts, const float* gaps, const float* picks, int count)
{
    const int row = a.first + (int)blockIdx.x;
    if (row == a.M) {
        put_largest_scale<kJoinThreads / 64>(a);
        return;
    }
    const float2* own = parts + (long long)blockIdx.x * count;
    float top = kNone, sum = 0.f;
    for (int i = (int)threadIdx.x; i < count; i += 256) join<true>(top, sum, own[i].x, own[i].y);
    join_all<4, true>(top, sum);
    if (a.targets) {
        put_loss<4, true>(a, row, top, sum, [&](int, int) { return picks[blockIdx.x]; });
        return;
    }
    float gap = 0.f;
    for (int i = (int)threadIdx.x; i < count; i += 256) gap += gaps[(long long)blockIdx.x * count + i];
    gap = fold_all<4>(gap, [](float x, float y) { return x + y; });
    const float above = log_of<true>(top, sum);
    if (threadIdx.x == 0) put_divergence(a, row, top + above, (top - gap + above) * kLn2);
}

// ds from its parts, rows one after the other, and from what rows of the call before have left; 64 columns to a workgroup of four waves, which share the parts
// out.
__device__ __forceinline__ void put_ds(const ScaleGradient& d, int group)
{
    __shared__ float sums[4][64];
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, n = group * 64 + lane;
    constexpr int U = 8;
    float sum = 0.f;
    for (int first = wave; first < d.count; first += 4 * U) {
        float v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = first + 4 * u < d.count && n < d.N ? d.parts[(first + 4 * u) * d.ld + n] : 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) sum += v[u];
    }
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || n >= d.N) return;
    sum = (sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane]) * d.heat;
    store_out(d.out, d.f16, n, d.before ? d.before[n] + sum : sum);
}

__global__ __launch_bounds__(256) void tl_loss_ds(ScaleGradient d) { put_ds(d, (int)blockIdx.x); }

// Few rows, backward: P = dz s 2^e of up to 48 rows, and ds.  A thread takes a column, all rows one after
// the other.  Bound by latency: 8.6 us for 40 rows of 5003 columns, 10 for 48 fp32 ones of 8000.
template <typename T>
__global__ __launch_bounds__(kFewColumns) void tl_loss_few_grad(LossArgs a)
{
    const int rows = a.M;
    __shared__ float wanted[kSmallMaxM][kFewColumns];
    const int tid = (int)threadIdx.x, first = (int)blockIdx.x * kFewColumns, n = first + tid;
    for (int m = 0; m < rows; ++m) wanted[m][tid] = 0.f;
    __syncthreads();
    if (a.targets) {
        if (tid < rows) {
            const long long target = a.targets[tid] - first;
            if (target >= 0 && target < kFewColumns) wanted[tid][target] = 1.f;
        }
    } else {
        for (int i = tid; i < rows * a.top; i += kFewColumns) {
            const int entry = a.entry[i];
            const unsigned c = (unsigned)(entry - first);
            if (entry >= 0 && c < kFewColumns) wanted[i / a.top][c] = a.share[i];   // (an entry stands once in a row)
        }
    }
    __syncthreads();
    if (n >= a.raw_ld) return;
    const bool there = n < a.N;
    const float s = there ? load_scale(a.scale, a.scale_f16, n) : 0.f, up = raise_of(a.lse[a.M], sizeof(T) == 2);
    float ds = 0.f;
    constexpr int U = 8;
    for (int m0 = 0; m0 < rows; m0 += U) {
        float raw[U], lse[U], grad[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int m = min(m0 + u, rows - 1);
            raw[u] = there ? a.raw[(long long)m * a.raw_ld + n] : 0.f;
            lse[u] = a.lse[m];
            grad[u] = a.grad[m];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (m0 + u >= rows) break;
            const bool counts = finite(lse[u]);
            const float dz = counts && there ? __expf(logit_of(a, raw[u], s) - lse[u]) - wanted[m0 + u][tid] : 0.f;
            static_cast<T*>(a.P)[(long long)(m0 + u) * a.raw_ld + n] = (T)settled(dz * (s * up));
            ds += counts ? dz * raw[u] * grad[u] : lse[u] == kNone ? 0.f : __builtin_nanf("");
        }
    }
    if (a.ds && there) store_out(a.ds, a.scale_f16, n, ds * a.heat);
}

// dx = what a row is multiplied by times the product of P, the sum of `parts` of them; a thread takes four values of a row.  The first d_groups workgroups take
// the gradient of the scales beside it.  4.3 us for 40 rows of 2048 in eight parts, 5.6 for 1024 of 1024.
template <typename T>
__global__ __launch_bounds__(256) void tl_loss_out(LossArgs a, const float* from, int rows, int parts, ScaleGradient d, unsigned d_groups)
{
    if (blockIdx.x < d_groups) {
        put_ds(d, (int)blockIdx.x);
        return;
    }
    const long long at = (long long)(blockIdx.x - d_groups) * 256 + threadIdx.x;
    const int pieces = (a.K + 3) / 4, m = (int)(at / pieces), k = (int)(at % pieces) * 4;
    if (m >= rows) return;
    const int row = a.first + m;
    const float factor = row_factor(a.lse[row], a.grad[row], a.heat, raise_of(a.lse[a.M], sizeof(T) == 2));
    const bool counts = lse_counts(a.lse[row]);
    float sum[4] = {};
    T* to = static_cast<T*>(a.dx) + row * a.dx_ld + k;
    if (a.K % 4 == 0) {
        for (int i = 0; i < parts; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(from + ((long long)i * rows + m) * a.K + k);
            sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
        }
    } else {
        for (int i = 0; i < parts; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += k + e < a.K ? from[((long long)i * rows + m) * a.K + k + e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (k + e < a.K) to[e] = (T)settled(counts ? sum[e] * factor : factor);
}

// The codes of a weight [K][N], transposed: those of a weight of N rows and K columns.  Once for a weight; a thread makes a dword (16 weights) from 16
// others: 90 us for 4096 x 32000.
__global__ __launch_bounds__(256) void tl_back_codes(const uint32_t* codes, int K, int N, int planes, uint32_t* out, long long dwords)
{
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    if (at >= dwords) return;
    const int units_in = (K + TL_CODE_UNIT_ROWS - 1) / TL_CODE_UNIT_ROWS, units = (N + TL_CODE_UNIT_ROWS - 1) / TL_CODE_UNIT_ROWS;
    const int d = (int)(at & 3), lane = (int)(at >> 2 & 63);
    const long long unit = at >> 8;
    const int u = (int)(unit % units), plane = (int)(unit / units % planes), block = (int)(unit / units / planes);
    const int k = block * 16 + (lane & 15);
    uint32_t word = 0;
    if (k < K) {
        const int r = k % TL_CODE_UNIT_ROWS;
        const int shift = 14 - 2 * (4 * (r >> 5 & 1) + (r >> 1 & 3)) + 16 * (r & 1);
        for (int i = 0; i < 16; ++i) {
            const int h = i >> 3, p = i >> 1 & 3, j = i & 1;
            const int v = u * TL_CODE_UNIT_ROWS + 64 * d + 32 * h + 8 * (lane >> 4) + 2 * p + j;
            if (v >= N) continue;
            const long long from = (((long long)(v / 16) * planes + plane) * units_in + k / TL_CODE_UNIT_ROWS) * (TL_CODE_UNIT_BYTES / 4) +
                                   ((r >> 3 & 3) * 16 + v % 16) * 4 + (r >> 6);
            word |= (codes[from] >> shift & 3u) << (14 - 2 * (4 * h + p) + 16 * j);
        }
    }
    out[at] = word;
}

// ---------------------------------------------------------------------------
// Host.
// ---------------------------------------------------------------------------
int64_t back_units(const tl_layout_header* h) { return ceil_div(h->columns, TL_CODE_UNIT_ROWS) * ceil_div(h->inners, 16) * h->code_planes; }

int check_weight(const tl_layout_header* h, const void* blob)
{
    if (int rc = check_header(h)) return rc;
    if (!blob || reinterpret_cast<uintptr_t>(blob) % 256) return fail(TL_ERR_ALIGN, "the blob must be on the device, 256-byte aligned");
    if (!h->off_codes) return fail(TL_ERR_UNSUPPORTED, "a weight without codes has no loss: pack it anew");
    return TL_OK;
}

// (Its square and its reciprocal are factors of results, and the reciprocal of logits: all of them fp32 numbers of full precision.)
int check_temperature(float t)
{
    return t >= 1e-6f && t <= 1e6f ? TL_OK : fail(TL_ERR_ARG, "temperature=%g is no number from 1e-6 to 1e6", (double)t);
}

int check_target(const tl_loss_target* t)
{
    if (!t) return fail(TL_ERR_ARG, "null pointer");
    if (int rc = check_temperature(t->temperature)) return rc;
    if ((t->targets != nullptr) == (t->entries != nullptr)) return fail(TL_ERR_ARG, "either targets or a teacher's entries");
    if (t->targets && t->temperature != 1.f) return fail(TL_ERR_ARG, "cross entropy has no temperature");
    if (t->entries && (t->top < 1 || t->top > kMostTop)) return fail(TL_ERR_ARG, "%d entries of a teacher (1 to %d)", t->top, kMostTop);
    if (t->entries && (!t->shares || !t->known)) return fail(TL_ERR_ARG, "entries, shares and known come together");
    return TL_OK;
}

int check_rows(const void* x, int x_dtype, int64_t ldx, int64_t M, const tl_layout_header* h, const void* scale, int scale_dtype)
{
    if (int rc = check_dtype(x_dtype, "x")) return rc;
    if (int rc = check_dtype(scale_dtype, "scale")) return rc;
    if (M < 0 || M > (1 << 24)) return fail(TL_ERR_SHAPE, "%lld rows (0 to 2^24)", (long long)M);
    if (M == 0) return TL_OK;
    if (!x) return fail(TL_ERR_ARG, "device pointer is null");
    if (ldx < (int64_t)h->inners || ldx > (1 << 24)) return fail(TL_ERR_SHAPE, "ldx=%lld is none for rows of %u", (long long)ldx, h->inners);
    if (reinterpret_cast<uintptr_t>(x) % (x_dtype == TL_F16 ? 2 : 4) || reinterpret_cast<uintptr_t>(scale) % (scale_dtype == TL_F16 ? 2 : 4))
        return fail(TL_ERR_ALIGN, "x and scale must be aligned to their type");
    return TL_OK;
}

LossArgs loss_args(const tl_layout_header* h, int64_t M, const void* scale, int scale_dtype, const tl_loss_target* t)
{
    LossArgs a{};
    a.M = (int)M, a.N = (int)h->columns, a.K = (int)h->inners;
    a.scale = scale, a.scale_f16 = scale_dtype == TL_F16;
    a.targets = t->targets, a.ignore = t->ignore;
    a.entry = t->entries, a.share = t->shares, a.known = t->known, a.top = t->entries ? t->top : 1;
    a.heat = t->temperature, a.cool = 1.0f / t->temperature;
    return a;
}

// The parts of a workspace, each a whole number of 256 bytes.
struct Parts {
    char* base;
    int64_t used = 0;
    void* take(int64_t bytes)
    {
        void* p = base ? base + used : nullptr;
        used += round_up(bytes, 256);
        return p;
    }
};

struct FewParts {
    float* raw;          // [rows][ld]
    void* product;       // workspace of the product of the logits
    void* P;             // backward: [rows][ld]
    float* sums;         // [rows][K]
};

FewParts few_parts(Parts& p, const tl_layout_header* h, int64_t M, int x_dtype, bool backward, int64_t product_bytes)
{
    const int64_t rows = M, ld = round_up(h->columns, 64);
    FewParts f{};
    f.raw = static_cast<float*>(p.take(rows * ld * 4));
    f.product = p.take(product_bytes);
    if (backward) {
        f.P = p.take(rows * ld * (x_dtype == TL_F16 ? 2 : 4));
        f.sums = static_cast<float*>(p.take(rows * h->inners * 4));
    }
    return f;
}

int product_workspace(const tl_layout_header* h, int64_t M, int x_dtype, int64_t* bytes)
{
    *bytes = 0;
    return M ? tl_spmm_workspace(h, M, x_dtype, TL_X_ROW_MAJOR, bytes) : TL_OK;
}

void rows_out(const LossArgs& a, int x_dtype, const float* sums, int rows, int parts, const ScaleGradient* d, hipStream_t st)
{
    const ScaleGradient none{};
    const unsigned groups = d ? (unsigned)ceil_div(d->N, 64) : 0;
    const dim3 grid(groups + (unsigned)ceil_div((int64_t)ceil_div(a.K, 4) * rows, 256));
    if (x_dtype == TL_F16) hipLaunchKernelGGL(tl_loss_out<_Float16>, grid, dim3(256), 0, st, a, sums, rows, parts, d ? *d : none, groups);
    else hipLaunchKernelGGL(tl_loss_out<float>, grid, dim3(256), 0, st, a, sums, rows, parts, d ? *d : none, groups);
}

// The product of few rows of P with the transposed weight.
int back_product(const tl_layout_header* h, const void* back, const LossArgs& a, int x_dtype, float* sums, hipStream_t st)
{
    KernelArgs k;
    std::memset(&k, 0, sizeof(k));
    k.X = a.P, k.ldx = a.raw_ld;
    k.Y = sums, k.ldy = a.K;
    k.M = a.M, k.N = a.K, k.NB = (int)ceil_div(a.K, 16);
    k.K = (int)round_up(a.N, 8);                 // (P is padded with zeros, the codes too)
    k.planes = (int)h->code_planes, k.units = (int)ceil_div(a.N, TL_CODE_UNIT_ROWS);
    k.c0 = Codes{static_cast<const unsigned char*>(back), k.planes};
    k.x_f16 = x_dtype == TL_F16, k.one = 1.0f;
    k.tile_rows = 1;                             // (T = 0: there is no index stream to walk; P's sums are finite, or what they are multiplied by is NaN)
    return launch_matrix_few(k, x_dtype, false, st);
}

// Many rows: so many at a time, and what the workspace holds for them.
constexpr int64_t kForwardRows = 16384;
constexpr int64_t kGradientBytes = 128 << 20;    // of P, and of its image

// Rows and columns of P at a time.  All columns where all rows of them fit; else pieces of the vocabulary, and as many rows as fit of those.  (Of a weight whose
// rows repeat all columns in any case: its planes of codes are walked one after the other.)
struct PieceOfP {
    int64_t rows, columns;
};

PieceOfP piece_of_p(const tl_layout_header* h, int64_t M, int x_dtype)
{
    const int64_t each = x_dtype == TL_F16 ? 2 : 6, all = round_up(h->columns, 64);
    const bool whole = h->code_planes > 1 || all <= kPieceColumns || std::min(M, kForwardRows) * all * each <= kGradientBytes;
    const int64_t columns = whole ? all : kPieceColumns;
    return PieceOfP{std::min(M, std::min(kForwardRows, std::max<int64_t>(kGradientBytes / (columns * each) / 128 * 128, 128))), columns};
}

// Rows whose logits are not kept.  (us few / many, fp16: 24 rows of 4096 over 32000 rated 26.7 / 27.1, a step 82 / 83; 33 41.7 / 32.2, 121 / 90; of 1024 24 17.3 / 15.1,
// 60 / 58; but 33 of 2048 over 5003, whose tiles leave most of the chip idle, 15.6 / 20.7, 43 / 55.  fp32 24 of 4096 over 32000 53 / 57, 179 / 165.)
bool takes_many(const tl_layout_header* h, int64_t M)
{
    return M > kFewRows || (M > kFewRows / 2 && (int64_t)h->columns > 64ll * compute_units());
}

struct ManyParts {
    int64_t rows;
    void* image;         // of the rows of x
    float2* parts;       // forward: [rows][columns / 64 or 32]
    float *gaps, *picks;
    int64_t columns;     // backward: of P
    int splits;          // workgroups that share out the columns of P for an output of their product
    void* P;             // [rows][columns]; of fp32 rows in three bf16 parts
    float *sums;         // [pieces * splits][rows][K], or, of one split, [rows][K]; null: neither
    float *ds_parts, *ds;
};

KernelArgs back_args(const tl_layout_header* h, int x_dtype, int rows)
{
    KernelArgs b;
    std::memset(&b, 0, sizeof(b));
    b.M = b.call_rows = rows, b.N = (int)h->inners, b.NB = (int)ceil_div(h->inners, 16);
    b.planes = (int)h->code_planes, b.units = (int)ceil_div(h->columns, TL_CODE_UNIT_ROWS);
    b.x_f16 = x_dtype == TL_F16, b.one = 1.0f, b.tile_rows = 1;
    return b;
}


ManyParts many_parts(Parts& p, const tl_layout_header* h, int64_t M, int x_dtype, bool backward)
{
    const int64_t N = h->columns, K = h->inners;
    const PieceOfP piece = piece_of_p(h, M, x_dtype);
    ManyParts f{};
    f.rows = backward ? piece.rows : std::min(M, kForwardRows);
    f.image = p.take(loss_image_bytes(K, f.rows, x_dtype));
    if (!backward) {
        const int64_t count = f.rows * ceil_div(N, x_dtype == TL_F16 ? 64 : 32);
        f.parts = static_cast<float2*>(p.take(count * 8));
        f.gaps = static_cast<float*>(p.take(count * 4));
        f.picks = static_cast<float*>(p.take(f.rows * 4));
        return f;
    }
    f.columns = piece.columns;
    f.splits = loss_splits(back_args(h, x_dtype, (int)f.rows), x_dtype, (int)ceil_div(std::min(f.columns, N), TL_CODE_UNIT_ROWS));
    const int64_t pieces = ceil_div(N, f.columns);
    f.P = p.take(f.rows * f.columns * (x_dtype == TL_F16 ? 2 : 6));
    f.sums = pieces * f.splits > 1 ? static_cast<float*>(p.take((f.splits > 1 ? pieces * f.splits : 1) * f.rows * K * 4)) : nullptr;
    f.ds_parts = static_cast<float*>(p.take(ceil_div(f.rows, 32) * f.columns * 4));
    f.ds = static_cast<float*>(p.take(N * 4));
    return f;
}

KernelArgs rows_product(const tl_layout_header* h, const void* blob, const void* x, int x_dtype, int64_t ldx, int64_t first, int rows, const LossArgs& a)
{
    KernelArgs k;
    std::memset(&k, 0, sizeof(k));
    k.w0 = weight_ptrs(h, blob, a.scale);
    k.X = static_cast<const char*>(x) + first * ldx * (x_dtype == TL_F16 ? 2 : 4);
    k.ldx = ldx;
    k.M = k.call_rows = rows, k.N = a.N, k.K = a.K, k.T = (int)h->n_tiles, k.tile_rows = (int)h->tile_rows;
    k.NB = (int)h->n_blocks, k.c0 = weight_codes(h, blob), k.units = (int)h->code_units, k.planes = k.c0.planes;
    k.x_f16 = x_dtype == TL_F16, k.scale_f16 = a.scale_f16;
    k.one = 1.0f;
    LossRows& l = k.loss;
    l.targets = a.targets ? a.targets + first : nullptr;
    l.entry = a.entry ? a.entry + first * a.top : nullptr;
    l.share = a.share ? a.share + first * a.top : nullptr;
    l.top = a.top;
    l.top_magic = a.top > 1 ? (unsigned)((((uint64_t)1 << 32) + a.top - 1) / a.top) : 0;
    l.cool = a.cool, l.heat = a.heat;
    return k;
}

int many_forward(const tl_layout_header* h, const void* blob, const void* x, int x_dtype, int64_t ldx, LossArgs a, const ManyParts& f, hipStream_t st)
{
    for (int64_t m = 0; m < a.M; m += f.rows) {
        const int rows = (int)std::min<int64_t>(a.M - m, f.rows);
        KernelArgs k = rows_product(h, blob, x, x_dtype, ldx, m, rows, a);
        if (int rc = make_loss_image(&k, x_dtype, f.image, st)) return rc;
        k.loss.parts = f.parts, k.loss.gaps = f.gaps, k.loss.picks = f.picks;
        if (int rc = launch_loss(k, x_dtype, kLossLogits, st)) return rc;
        a.first = (int)m;
        hipLaunchKernelGGL(tl_loss_join, dim3((unsigned)(rows + (m + rows == a.M))), dim3(kJoinThreads), 0, st, a, f.parts, f.gaps, f.picks,
                           (int)ceil_div(a.N, loss_part(k, x_dtype, kLossLogits)));
    }
    return TL_OK;
}

int many_backward(const tl_layout_header* h, const void* blob, const void* back, const void* x, int x_dtype, int64_t ldx, const LossArgs& a, const ManyParts& f,
                  hipStream_t st)
{
    const int es = x_dtype == TL_F16 ? 2 : 4, planes = (int)h->code_planes, pieces = (int)ceil_div(a.N, f.columns);
    for (int64_t m = 0; m < a.M; m += f.rows) {
        const int rows = (int)std::min<int64_t>(a.M - m, f.rows);
        KernelArgs k = rows_product(h, blob, x, x_dtype, ldx, m, rows, a);
        if (int rc = make_loss_image(&k, x_dtype, f.image, st)) return rc;
        k.loss.lse = a.lse + m, k.loss.grad = a.grad + m, k.loss.largest = a.lse + a.M;
        KernelArgs b = back_args(h, x_dtype, rows);
        b.c0 = Codes{static_cast<const unsigned char*>(back), planes};
        b.loss = k.loss;
        b.loss.splits = f.splits;
        ScaleGradient d{};
        bool beside = false;                     // the rows' gradient, in one launch with it
        for (int piece = 0; piece < pieces; ++piece) {
            const int64_t n = piece * f.columns, wide = std::min<int64_t>(a.N - n, f.columns), padded = round_up(wide, 8);
            KernelArgs some = k;
            some.N = (int)wide, some.NB = (int)ceil_div(wide, 16);
            some.c0.base += n / 16 * planes * k.units * TL_CODE_UNIT_BYTES;
            if (a.scale) some.w0.scale = static_cast<const char*>(a.scale) + n * (a.scale_f16 ? 2 : 4);
            some.Y = f.P, some.y_f16 = 1, some.ldy = f.columns;
            some.loss.first = (int)n, some.loss.padded = (int)padded, some.loss.plane = f.rows * f.columns;
            some.loss.ds = a.ds ? f.ds_parts : nullptr, some.loss.ds_ld = f.columns;
            if (int rc = launch_loss(some, x_dtype, kLossGradients, st)) return rc;
            // (sums of rows in several parts are kept in fp32 until the last)
            const bool end = m + rows == a.M;
            d = ScaleGradient{f.ds_parts, (int)ceil_div(rows, loss_part(some, x_dtype, kLossGradients)), some.loss.ds_ld, (int)wide, a.heat, m > 0 ? f.ds + n : nullptr,
                              end ? static_cast<char*>(a.ds) + n * (a.scale_f16 ? 2 : 4) : reinterpret_cast<char*>(f.ds + n), end && a.scale_f16};
            beside = a.ds && a.dx && f.splits > 1 && pieces == 1;
            if (a.ds && !beside) hipLaunchKernelGGL(tl_loss_ds, dim3((unsigned)ceil_div(wide, 64)), dim3(256), 0, st, d);
            if (!a.dx) continue;
            // (rows of P begin with column n, a whole unit, those of the transposed weight with column 0)
            b.K = (int)(n + padded);
            b.image = f.P, b.image_ld = f.columns, b.image_plane = some.loss.plane;
            b.loss.unit0 = (int)(n / TL_CODE_UNIT_ROWS), b.loss.units = planes > 1 ? planes * b.units : (int)ceil_div(wide, TL_CODE_UNIT_ROWS);
            const bool last = f.splits == 1 && piece + 1 == pieces;
            b.loss.sums = f.splits == 1 && piece > 0 ? f.sums : nullptr, b.loss.last = last;
            b.Y = last ? static_cast<char*>(a.dx) + m * a.dx_ld * es : reinterpret_cast<char*>(f.sums + (int64_t)(f.splits == 1 ? 0 : piece * f.splits) * rows * a.K);
            b.y_f16 = last && k.x_f16, b.ldy = last ? a.dx_ld : a.K;
            if (int rc = launch_loss(b, x_dtype, kLossBack, st)) return rc;
        }
        if (a.dx && f.splits > 1) {
            LossArgs some = a;
            some.first = (int)m;
            rows_out(some, x_dtype, f.sums, rows, pieces * f.splits, beside ? &d : nullptr, st);
        }
    }
    return TL_OK;
}

}  // namespace

extern "C" int tl_teacher_entries(const int64_t* ids, int64_t ids_ld, const void* logits, int dtype, int64_t logits_ld, int64_t M, int top, int columns,
                                  float temperature, int32_t* entries, float* shares, float* known, void* stream)
{
    if (int rc = check_dtype(dtype, "logits")) return rc;
    if (M < 0 || M > (1 << 24) || columns < 1) return fail(TL_ERR_SHAPE, "%lld rows over %d columns", (long long)M, columns);
    if (top < 1 || top > kMostTop) return fail(TL_ERR_ARG, "%d entries of a teacher (1 to %d)", top, kMostTop);
    if (int rc = check_temperature(temperature)) return rc;
    if (M == 0) return TL_OK;
    if (!ids || !logits || !entries || !shares || !known) return fail(TL_ERR_ARG, "device pointer is null");
    if (ids_ld < top || logits_ld < top) return fail(TL_ERR_SHAPE, "rows of ids or logits are shorter than %d", top);
    TeacherArgs a{ids, logits, ids_ld, logits_ld, dtype == TL_F16, top, columns, 1.0f / temperature, entries, shares, known};
    hipLaunchKernelGGL(tl_teacher, dim3((unsigned)M), dim3(64), 0, static_cast<hipStream_t>(stream), a);
    return finish_launch();
}

extern "C" int tl_back_codes_size(const tl_layout_header* header, int64_t* bytes)
{
    if (int rc = check_header(header)) return rc;
    if (!bytes) return fail(TL_ERR_ARG, "null pointer");
    if (!header->off_codes) return fail(TL_ERR_UNSUPPORTED, "a weight without codes cannot be transposed: pack it anew");
    *bytes = back_units(header) * TL_CODE_UNIT_BYTES;
    return TL_OK;
}

extern "C" int tl_back_codes_make(const tl_layout_header* header, const void* blob_dev, void* back, void* stream)
{
    if (int rc = check_weight(header, blob_dev)) return rc;
    if (!back || reinterpret_cast<uintptr_t>(back) % 16) return fail(TL_ERR_ALIGN, "the transposed codes must be on the device, 16-byte aligned");
    const int64_t dwords = back_units(header) * (TL_CODE_UNIT_BYTES / 4);
    if (dwords > (int64_t)INT32_MAX * 256) return fail(TL_ERR_SHAPE, "a weight of %u x %u is too large", header->inners, header->columns);
    hipLaunchKernelGGL(tl_back_codes, dim3((unsigned)ceil_div(dwords, 256)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       reinterpret_cast<const uint32_t*>(static_cast<const char*>(blob_dev) + header->off_codes), (int)header->inners, (int)header->columns,
                       (int)header->code_planes, static_cast<uint32_t*>(back), (long long)dwords);
    return finish_launch();
}

extern "C" int tl_head_loss_workspace(const tl_layout_header* header, int64_t M, int x_dtype, const tl_loss_target* target, int backward, int64_t* bytes)
{
    if (int rc = check_header(header)) return rc;
    if (int rc = check_dtype(x_dtype, "x")) return rc;
    if (int rc = check_target(target)) return rc;
    if (!bytes || M < 0 || M > (1 << 24)) return fail(TL_ERR_ARG, "a pointer is null, or %lld rows (0 to 2^24)", (long long)M);
    Parts p{nullptr};
    if (takes_many(header, M)) {
        many_parts(p, header, M, x_dtype, backward != 0);
    } else {
        int64_t product = 0;
        if (int rc = product_workspace(header, M, x_dtype, &product)) return rc;
        few_parts(p, header, M, x_dtype, backward != 0, product);
    }
    *bytes = p.used;
    return TL_OK;
}

namespace {

int check_call(const tl_layout_header* header, const void* blob_dev, const void* x, int x_dtype, int64_t ldx, int64_t M, const void* scale, int scale_dtype,
               const tl_loss_target* target, bool backward, const void* workspace, int64_t workspace_bytes)
{
    if (int rc = check_weight(header, blob_dev)) return rc;
    if (int rc = check_target(target)) return rc;
    if (int rc = check_rows(x, x_dtype, ldx, M, header, scale, scale_dtype)) return rc;
    int64_t need = 0;
    if (int rc = tl_head_loss_workspace(header, M, x_dtype, target, backward, &need)) return rc;
    if (M > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256)) return fail(TL_ERR_ALIGN, "the workspace must be on the device, 256-byte aligned");
    if (workspace_bytes < need) return fail(TL_ERR_SIZE, "workspace has %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    return TL_OK;
}

// The logits of few rows, without scales.
int raw_product(const tl_layout_header* header, const void* blob_dev, const void* x, int x_dtype, int64_t ldx, const LossArgs& a, const FewParts& f,
                int64_t product_bytes, void* stream)
{
    return tl_spmm(header, blob_dev, x, x_dtype, TL_X_ROW_MAJOR, ldx, a.M, f.raw, TL_F32, a.raw_ld, nullptr, TL_F32, product_bytes ? f.product : nullptr,
                   product_bytes, stream);
}

}  // namespace

extern "C" int tl_head_loss(const tl_layout_header* header, const void* blob_dev, const void* x, int x_dtype, int64_t ldx, int64_t M, const void* scale,
                            int scale_dtype, const tl_loss_target* target, float* loss, float* lse, void* workspace, int64_t workspace_bytes, void* stream)
{
    if (int rc = check_call(header, blob_dev, x, x_dtype, ldx, M, scale, scale_dtype, target, false, workspace, workspace_bytes)) return rc;
    if (M == 0) return TL_OK;
    if (!loss || !lse) return fail(TL_ERR_ARG, "device pointer is null");
    hipStream_t st = static_cast<hipStream_t>(stream);
    LossArgs a = loss_args(header, M, scale, scale_dtype, target);
    a.loss = loss, a.lse = lse;
    Parts p{static_cast<char*>(workspace)};
    if (takes_many(header, M)) {
        if (int rc = many_forward(header, blob_dev, x, x_dtype, ldx, a, many_parts(p, header, M, x_dtype, false), st)) return rc;
        return finish_launch();
    }
    int64_t product = 0;
    if (int rc = product_workspace(header, M, x_dtype, &product)) return rc;
    const FewParts f = few_parts(p, header, M, x_dtype, false, product);
    a.raw = f.raw, a.raw_ld = round_up(header->columns, 64);
    if (int rc = raw_product(header, blob_dev, x, x_dtype, ldx, a, f, product, stream)) return rc;
    hipLaunchKernelGGL(tl_loss_few, dim3((unsigned)M + 1), dim3(kRowThreads), 0, st, a);
    return finish_launch();
}

extern "C" int tl_head_loss_backward(const tl_layout_header* header, const void* blob_dev, const void* back, const void* x, int x_dtype, int64_t ldx, int64_t M,
                                     const void* scale, int scale_dtype, const tl_loss_target* target, const float* lse, const float* grad, void* dx,
                                     int64_t dx_ld, void* dscale, void* workspace, int64_t workspace_bytes, void* stream)
{
    if (int rc = check_call(header, blob_dev, x, x_dtype, ldx, M, scale, scale_dtype, target, true, workspace, workspace_bytes)) return rc;
    if (dx && (!back || reinterpret_cast<uintptr_t>(back) % 16)) return fail(TL_ERR_ALIGN, "the transposed codes must be on the device, 16-byte aligned");
    if (dx && dx_ld < (int64_t)header->inners) return fail(TL_ERR_SHAPE, "dx_ld=%lld is none for rows of %u", (long long)dx_ld, header->inners);
    if (dscale && !scale) return fail(TL_ERR_ARG, "a gradient of scales that there are none of");
    if (M == 0) return TL_OK;
    if (!lse || !grad) return fail(TL_ERR_ARG, "device pointer is null");
    hipStream_t st = static_cast<hipStream_t>(stream);
    LossArgs a = loss_args(header, M, scale, scale_dtype, target);
    a.lse = const_cast<float*>(lse), a.grad = grad;
    a.dx = dx, a.dx_ld = dx_ld;
    Parts p{static_cast<char*>(workspace)};
    a.ds = dscale;
    if (takes_many(header, M)) {
        if (int rc = many_backward(header, blob_dev, back, x, x_dtype, ldx, a, many_parts(p, header, M, x_dtype, true), st)) return rc;
    } else {
        int64_t product = 0;
        if (int rc = product_workspace(header, M, x_dtype, &product)) return rc;
        const FewParts f = few_parts(p, header, M, x_dtype, true, product);
        a.raw = f.raw, a.raw_ld = round_up(header->columns, 64);
        a.P = f.P;
        const dim3 groups((unsigned)ceil_div(a.raw_ld, kFewColumns));
        if (int rc = raw_product(header, blob_dev, x, x_dtype, ldx, a, f, product, stream)) return rc;
        if (x_dtype == TL_F16) hipLaunchKernelGGL(tl_loss_few_grad<_Float16>, groups, dim3(kFewColumns), 0, st, a);
        else hipLaunchKernelGGL(tl_loss_few_grad<float>, groups, dim3(kFewColumns), 0, st, a);
        if (dx) {
            if (int rc = back_product(header, back, a, x_dtype, f.sums, st)) return rc;
            rows_out(a, x_dtype, f.sums, a.M, 1, nullptr, st);
        }
    }
    return finish_launch();
}
