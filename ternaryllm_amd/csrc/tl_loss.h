// What the kernels of a head's losses share: their arguments, and what a row's gradient is multiplied by.
#pragma once
#include "tl_device.h"

namespace tl {

constexpr int kPieceColumns = 16384;  // columns of P at a time, of many rows (whole units of the transposed codes)
constexpr int kFewRows = 48;          // whose logits are kept for as long as a call takes
constexpr int kMostTop = 1024;        // entries of a teacher's row

struct TeacherArgs {
    const int64_t* ids;               // [M][ids_ld]
    const void* logits;               // [M][logits_ld]
    long long ids_ld, logits_ld;
    int f16, top, N;
    float cool;                       // 1 / temperature
    int* entry;                       // [M][top]
    float *share, *known;             // [M][top], [M]
};

struct LossArgs {
    const void* scale;                // [N] or null
    int scale_f16;
    int M, N, K, top;
    int first;                        // row of the call that the launch begins with
    float heat, cool;                 // the temperature, and 1 / it
    const int64_t* targets;           // [M], or null: the teacher's entries
    long long ignore;
    const int* entry;                 // [M][top], -1: none
    const float *share, *known;
    float *loss, *lse;                // [M], [M + 1]: what the backward pass keeps (of many rows as an exponent of 2, as their product takes it), and the largest
                                      // column scale
    const float* raw;                 // [rows][raw_ld]: products without scales
    long long raw_ld;
    const float* grad;                // [M], of the losses
    void* P;                          // [rows][raw_ld], x's type
    void* ds;                         // [N] of the scales' type, or null
    void* dx;                         // [M][dx_ld], x's type
    long long dx_ld;
};

// The gradient of the scales from its parts.
struct ScaleGradient {
    const float* parts;               // [count][ld]
    int count;
    long long ld;
    int N;
    float heat;
    const float* before;              // null, or [N]: of the rows before
    void* out;
    int f16;
};

// The power of two that probabilities are raised by, times their columns' scales.  fp16: so that the largest is 2^15 at most and those that are lost, below
// 2^-25, are 2^-40 of it: without it, and with the scales of a head of 4096 rows, all probabilities below 2^-19 would lose bits.  fp32, which are multiplied in
// scaled bf16 parts that end at 2^112 (tl_few.hip): so that the largest is 2^101 at most; nothing is lost there but of scales 2^-200 of the largest.
// NaN where a scale is not finite: so are all gradients of rows then.
__device__ __forceinline__ float raise_of(float largest_scale, bool f16)
{
    if (!(largest_scale < __builtin_huge_valf())) return __builtin_nanf("");
    if (!(largest_scale > 0.f)) return 1.f;
    const int e = ilogbf(largest_scale);
    return ldexpf(1.f, f16 ? min(max(14 - e, -126), 126) : min(100 - e, 0));
}

// A product that is rounded before anything is taken off it.  (A large logit less one that the same was made of is 0, and its exponential 1; as one
// instruction with the subtraction it would be what the rounding had dropped, from 2^24 on whole numbers, and its exponential 0 or infinite.)
__device__ __forceinline__ float rounded_product(float x, float y)
{
#pragma clang fp contract(off)
    return x * y;
}

// Whether a row has a gradient of its own: not, it counts for nothing (-inf), or its loss is NaN.
__device__ __forceinline__ bool lse_counts(float lse) { return fabsf(lse) < __builtin_huge_valf(); }

// What the product of a row's P is multiplied by: 0 for a row that counts for nothing, NaN where its loss is.
__device__ __forceinline__ float row_factor(float lse, float grad, float heat, float raised)
{
    if (lse == -__builtin_huge_valf()) return 0.f;
    if (lse != lse) return lse;
    return grad * heat / raised;
}

}  // namespace tl
