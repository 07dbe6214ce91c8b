// Rows held in 8 bits: what the kernels of vl_quant*.cu share.
//
// A row x is held as whole numbers c in [-127, 127] and one fp32 scale s: s = max|x| / 127 rounded to fp32, c = x / s
// rounded to the nearest whole number, ties to even, of the exact quotient.  Codes are int8 [n, ld], ld a multiple of
// 16 with zeros behind `dim`; beside them stands sum c^2 as int32.  A row with an infinity or a NaN gets the scale NaN
// and the codes 0, so everything made of it is NaN.  Products of codes are summed in 32-bit integers, exactly: the order
// of a sum, the padding and the kernel that makes it do not show in a result.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "vl_common.cuh"

struct VlQuantRows {
    const int8_t* codes;       // [n, ld]
    const float* scales;       // [n]
    const int32_t* norms;      // [n]: sum of squared codes
};

template <typename T> __device__ __forceinline__ float vl_to_float(T x);
template <> __device__ __forceinline__ float vl_to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float vl_to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float vl_to_float<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T vl_from_float(float x);
template <> __device__ __forceinline__ float vl_from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 vl_from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half vl_from_float<__half>(float x) { return __float2half_rn(x); }

// The scale of a row whose largest magnitude is `largest` (an infinity or a NaN when the row holds one).
__device__ __forceinline__ float vl_quant_scale(float largest)
{
    return largest <= 3.402823466e38f ? __fdiv_rn(largest, 127.0f) : __int_as_float(0x7fc00000);       // NaN compares false
}

// The code of x is the nearest whole number to the exact x / s.  Made with the inverse of s, x / s is off by less than 2^-16 of
// a step, so its rounding can only be wrong next to a half; the remainder x - q s tells, and an FMA makes it exactly
// there (it is a multiple of the smaller of both last places and at most about s/2; where the rounding of a larger one
// matters, it still compares right).  Scales whose inverse may overflow or whose half may not be a number (`tiny`) take a
// division in 64 bits.
__device__ __forceinline__ bool vl_quant_tiny(float s) { return !(s >= 1e-30f); }     // zero and NaN too

template <typename T> __device__ __forceinline__ float2 vl_to_float2(uint32_t two);
template <> __device__ __forceinline__ float2 vl_to_float2<__nv_bfloat16>(uint32_t two)
{
    return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 vl_to_float2<__half>(uint32_t two)
{
    return __half22float2(*reinterpret_cast<const __half2*>(&two));
}

// Four consecutive elements of a row, starting at e: one load where VEC says that groups of four are aligned, zeros behind dim.
// They are kept as they come and widened where they are used.
template <typename T> struct VlFour { uint2 raw; };
template <> struct VlFour<float> { float4 raw; };
template <typename T>
__device__ __forceinline__ float4 vl_widen(const VlFour<T>& v)
{
    if constexpr (sizeof(T) == 4) {
        return v.raw;
    } else {
        const float2 a = vl_to_float2<T>(v.raw.x), b = vl_to_float2<T>(v.raw.y);
        return make_float4(a.x, a.y, b.x, b.y);
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ VlFour<T> vl_load4(const T* __restrict__ x, int e, int dim)
{
    VlFour<T> v;
    if constexpr (sizeof(T) == 4) {
        if (VEC && e + 4 <= dim) v.raw = __ldg(reinterpret_cast<const float4*>(x + e));
        else v.raw = make_float4(e < dim ? x[e] : 0.0f, e + 1 < dim ? x[e + 1] : 0.0f, e + 2 < dim ? x[e + 2] : 0.0f, e + 3 < dim ? x[e + 3] : 0.0f);
    } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(x);
        if (VEC && e + 4 <= dim) v.raw = __ldg(reinterpret_cast<const uint2*>(h + e));
        else v.raw = make_uint2((e < dim ? h[e] : 0u) | (uint32_t)(e + 1 < dim ? h[e + 1] : 0u) << 16,
                                (e + 2 < dim ? h[e + 2] : 0u) | (uint32_t)(e + 3 < dim ? h[e + 3] : 0u) << 16);
    }
    return v;
}
// Running largest magnitude; a NaN stays.
__device__ __forceinline__ float vl_magnitude(float m, float4 v)
{
    float a, b;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(a) : "f"(v.x), "f"(v.y), "f"(m));
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(b) : "f"(v.z), "f"(v.w), "f"(a));
    return b;
}
// ... of a warp: the bits of numbers that are not negative order like the numbers, and put infinities and NaN last
__device__ __forceinline__ float vl_warp_magnitude(float m) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m))); }
struct VlQuantScale {
    float s, inv;
    bool tiny;
};
__device__ __forceinline__ VlQuantScale vl_quant_scale_of(float largest)
{
    const float s = vl_quant_scale(largest);
    return {s, __fdiv_rn(1.0f, s), vl_quant_tiny(s)};
}
__device__ __forceinline__ uint32_t vl_quant_word(int a, int b, int c, int d)
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Four codes in a word, for scales that are not tiny: x / s + 1.5 * 2^23 has the nearest whole number in its low bits.  Where
// that may be wrong, next to a half, the remainders decide (in bf16 rows the half of the largest element, 63.5 steps, is
// common: one in 768 random ones).
__device__ __forceinline__ int vl_quant_beside_half(float t, float rest, float half)
{
    const int q = __float_as_int(t);
    return fabsf(rest) > half || (fabsf(rest) == half && (q & 1)) ? q + (rest < 0.0f ? -1 : 1) : q;
}
__device__ __forceinline__ uint32_t vl_quant_codes(float4 v, const VlQuantScale& q)
{
    constexpr float kMagic = 12582912.0f;
    const float tx = __fmaf_rn(v.x, q.inv, kMagic), ty = __fmaf_rn(v.y, q.inv, kMagic);
    const float tz = __fmaf_rn(v.z, q.inv, kMagic), tw = __fmaf_rn(v.w, q.inv, kMagic);
    const float rx = __fmaf_rn(-__fsub_rn(tx, kMagic), q.s, v.x), ry = __fmaf_rn(-__fsub_rn(ty, kMagic), q.s, v.y);
    const float rz = __fmaf_rn(-__fsub_rn(tz, kMagic), q.s, v.z), rw = __fmaf_rn(-__fsub_rn(tw, kMagic), q.s, v.w);
    const float half = 0.5f * q.s;
    float rest;
    asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(rest) : "f"(rx), "f"(ry), "f"(rz));
    if (fmaxf(rest, fabsf(rw)) < half)
        return vl_quant_word(__float_as_int(tx), __float_as_int(ty), __float_as_int(tz), __float_as_int(tw));
    return vl_quant_word(vl_quant_beside_half(tx, rx, half), vl_quant_beside_half(ty, ry, half), vl_quant_beside_half(tz, rz, half),
                         vl_quant_beside_half(tw, rw, half));
}
// The same for tiny scales, in 64 bits.
__device__ __forceinline__ int vl_quant_code_tiny(float x, float s)
{
    if (!(s > 0.0f)) return 0;
    const double q = rint((double)x / (double)s);
    return (int)(q > 127.0 ? 127.0 : (q < -127.0 ? -127.0 : q));
}
__device__ __forceinline__ uint32_t vl_quant_codes_tiny(float4 v, float s)
{
    return vl_quant_word(vl_quant_code_tiny(v.x, s), vl_quant_code_tiny(v.y, s), vl_quant_code_tiny(v.z, s), vl_quant_code_tiny(v.w, s));
}

// a[i] of an array in registers
template <typename A, int R>
__device__ __forceinline__ A vl_pick(const A (&a)[R], int i)
{
    A x = a[0];
#pragma unroll
    for (int k = 1; k < R; ++k) x = i == k ? a[k] : x;
    return x;
}

// R rows by one warp: `put(r, e, word)` takes the codes of elements e .. e + 3 of row r, for every such group below code_ld.
// A null row is skipped.  The first 128 HELD elements stay in registers between the search for the largest one and the
// rounding, the rest are read again.  What has to be done once per row (two divisions) is done for all R at once, in R
// lanes.  All lanes get the scales and the sums of squared codes.
template <typename T, bool VEC, int HELD, int R, typename Put>
__device__ __forceinline__ void vl_quant_rows(const T* const (&x)[R], int dim, int code_ld, int lane, float (&scale)[R], int (&norm)[R], Put put)
{
    VlFour<T> v[R][HELD];
    float mine = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < HELD; ++j) v[r][j] = vl_load4<T, VEC>(x[r], (j * 32 + lane) * 4, x[r] ? dim : 0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float largest = 0.0f;
#pragma unroll
        for (int j = 0; j < HELD; ++j) largest = vl_magnitude(largest, vl_widen<T>(v[r][j]));
        if (x[r])
            for (int e = (HELD * 32 + lane) * 4; e < dim; e += 128) largest = vl_magnitude(largest, vl_widen<T>(vl_load4<T, VEC>(x[r], e, dim)));
        largest = vl_warp_magnitude(largest);
        if (lane == r || R == 1) mine = largest;
    }
    const VlQuantScale own = vl_quant_scale_of(mine);
    float inv[R];
    int sum[R];
    int rows_again = 0;                  // rows whose scale is tiny: all their words are made below
#pragma unroll
    for (int r = 0; r < R; ++r) {
        scale[r] = R == 1 ? own.s : __shfl_sync(0xffffffffu, own.s, r);
        inv[r] = R == 1 ? own.inv : __shfl_sync(0xffffffffu, own.inv, r);
        sum[r] = 0;
        if (vl_quant_tiny(scale[r])) {
            rows_again |= 1 << r;
        } else {
#pragma unroll
            for (int j = 0; j < HELD; ++j) {
                const int e = (j * 32 + lane) * 4;
                const uint32_t word = vl_quant_codes(vl_widen<T>(v[r][j]), {scale[r], inv[r], false});
                if (x[r] && e < code_ld) {
                    put(r, e, word);
                    sum[r] = __dp4a((int)word, (int)word, sum[r]);
                }
            }
        }
    }
    // what is left, in one copy of the code: rows with tiny scales, and the words behind 128 HELD elements
    if (rows_again || HELD * 128 < code_ld) {
#pragma unroll 1
        for (int r = 0; r < R; ++r) {
            const T* p = vl_pick(x, r);
            if (!p) continue;
            const bool tiny = rows_again >> r & 1;
            const VlQuantScale q = {vl_pick(scale, r), vl_pick(inv, r), tiny};
            int more = 0;
#pragma unroll 1
            for (int e = (tiny ? lane : HELD * 32 + lane) * 4; e < code_ld; e += 128) {
                const float4 four = vl_widen<T>(vl_load4<T, VEC>(p, e, dim));
                const uint32_t word = tiny ? vl_quant_codes_tiny(four, q.s) : vl_quant_codes(four, q);
                put(r, e, word);
                more = __dp4a((int)word, (int)word, more);
            }
#pragma unroll
            for (int k = 0; k < R; ++k) sum[k] += k == r ? more : 0;
        }
        __syncwarp();
    }
#pragma unroll
    for (int k = 0; k < R; ++k) norm[k] = __reduce_add_sync(0xffffffffu, sum[k]);
}

// Results of a whole-number product `dot` of two rows with scales qs, cs and squared sums qn, cn.  Every kernel comes
// here, so the same pair has the same bits wherever it is computed.
//
// Ordinary rows (vl_quant_ordinary) are finished in fp32.  Dots are exact there (a dot is no larger than the larger squared
// sum, and that is at most 2^24), and the scales' product is kept as an exact pair sh + sl where 1 - t or a + b - 2 t
// may be small against its terms:
//   product  sh f + sl f: the second product's rounding does not count, so one rounding.  Results of 16 bits (NARROW) are made of
//            sh f alone, two roundings of 32 bits before that of 16, which is 2^13 times as large and more (500,000 x 96 x 1,000
//            queries, bf16: 287 us, with the second product 309; 60,007 x 1536 x 4,000, fp32: 497 and 495)
//   cosine   1/2 - sh f, rounded once by an FMA, and that - sl f: two roundings of the result itself
//   l2       squared lengths a, b are pairs hi - over as well, hi of 20 bits, so that of rows of like length their sum is exact
//            (otherwise its error is made exactly and summed with the rest).  2 sh f is taken from it in one FMA, and the rest
//            (below 2^-18 (a + b), summed apart) is added: two roundings of the result itself, and 5 * 2^-43 (a + b).  In results
//            below 2^-16 (a + b) that would show, and near rows are made from the differences of their codes and scales
//            instead: vl_quant_pair64.  (200,000 x 768 x 2,500 queries: 664 us; with one rounding, by a third exact difference in
//            fp32 838, by sums in 64 bits without conversions 785.  A store all of whose rows are near each other, 200,000 x 768
//            x 1,000, takes 850 us instead of 222; one whose lengths vary 10,000 times 273 instead of 238.)
// Scales within 2^+-40 keep every term a normal number and the pairs exact.  Other rows take 64-bit arithmetic too, whose
// conversions run at 4 a clock and SM.
struct VlQuantSide {
    float s, hi, over;       // scale; squared length (squared l2 only): hi - over
    int n;
    bool ordinary;
};
__device__ __forceinline__ bool vl_quant_ordinary(float s, int n)
{
    return ((s >= 9.094947e-13f && s <= 1.0995116e12f) || s == 0.0f) && n <= (1 << 24);
}
template <int METRIC>
__device__ __forceinline__ VlQuantSide vl_quant_side(float s, int n)
{
    VlQuantSide r = {s, 0.0f, 0.0f, n, vl_quant_ordinary(s, n)};
    if (METRIC == VL_METRIC_SQL2) {
        const float sh = __fmul_rn(s, s), sl = __fmaf_rn(s, s, -sh), f = (float)n;
        const float length = __fmul_rn(sh, f);
        r.hi = __uint_as_float(__float_as_uint(length) & ~15u);
        r.over = __fadd_rn(__fsub_rn(r.hi, length), __fmaf_rn(-sl, f, __fmaf_rn(-sh, f, length)));
    }
    return r;
}
// The part of a + b below which a squared distance is that of near rows.
constexpr float kQuantNear = 1.0f / (1 << 16);

// In 64 bits, for any rows.  Products of scales are exact here.  l2 with D = codes_q - codes_r is
//   |qs c_q - cs c_r|^2 = (qs - cs)^2 dot + qs^2 <c_q, D> - cs^2 <c_r, D>,   <c_q, D> = qn - dot, <c_r, D> = dot - cn,
// whole numbers that are small for near rows, as is the difference of their scales: nothing large cancels, and equal rows are
// exactly 0 apart.
template <int METRIC>
__device__ __forceinline__ float vl_quant_pair64(int dot, float qs, int qn, float cs, int cn)
{
    const double q = qs, c = cs, f = dot;
    if (METRIC == VL_METRIC_SQL2) {
        const double apart = __dsub_rn(q, c);
        const double a = __dmul_rn(__dmul_rn(q, q), __dsub_rn((double)qn, f)), b = __dmul_rn(__dmul_rn(c, c), __dsub_rn((double)cn, f));
        const float d = (float)__fma_rn(__dmul_rn(apart, apart), f, __dadd_rn(a, b));
        return d <= 0.0f ? 0.0f : d;                        // a NaN stays
    }
    const double t = __dmul_rn(__dmul_rn(q, c), f);
    if (METRIC == VL_QUANT_PRODUCT) return (float)t;
    const float d = (float)__dmul_rn(__dsub_rn(1.0, t), 0.5);
    return d <= 0.0f ? 0.0f : (d > 1.0f ? 1.0f : d);
}
template <int METRIC>
static __device__ __noinline__ float vl_quant_pair64_apart(int dot, float qs, int qn, float cs, int cn)
{
    return vl_quant_pair64<METRIC>(dot, qs, qn, cs, cn);
}
// APART: what is rarely taken stands apart, and leaves the caller its registers (30,000 lists of 64 ids, 1M x 768, l2: 262 us, and
// 274 with it inside).
template <int METRIC, bool APART, bool NARROW>
__device__ __forceinline__ float vl_quant_pair(int dot, const VlQuantSide& q, const VlQuantSide& r)
{
    if (q.ordinary && r.ordinary) {
        const float f = (float)dot;
        const float cs = METRIC == VL_QUANT_PRODUCT ? r.s : (METRIC == VL_METRIC_COSINE ? 0.5f * r.s : 2.0f * r.s);
        const float sh = __fmul_rn(q.s, cs), sl = __fmaf_rn(q.s, cs, -sh);
        if (METRIC == VL_QUANT_PRODUCT) return NARROW ? __fmul_rn(sh, f) : __fmaf_rn(sh, f, __fmul_rn(sl, f));
        if (METRIC == VL_METRIC_COSINE) return __saturatef(__fmaf_rn(-sl, f, __fmaf_rn(-sh, f, 0.5f)));
        const float ab = __fadd_rn(q.hi, r.hi), of_r = __fsub_rn(ab, q.hi);
        const float more = __fadd_rn(__fsub_rn(__fsub_rn(ab, of_r), q.hi), __fsub_rn(of_r, r.hi));           // ab - a - b, exactly
        const float d = __fsub_rn(__fmaf_rn(-sh, f, ab), __fmaf_rn(sl, f, __fadd_rn(__fadd_rn(q.over, r.over), more)));
        if (d > __fmul_rn(kQuantNear, ab)) return d;
    }
    return APART ? vl_quant_pair64_apart<METRIC>(dot, q.s, q.n, r.s, r.n) : vl_quant_pair64<METRIC>(dot, q.s, q.n, r.s, r.n);
}

// Whether 24 bits hold the sum of any two numbers of 20 bits from `less` to `more`: leading digits three places apart, a carry, and 20.
__device__ __forceinline__ bool vl_quant_alike(float less, float more)
{
    return (int)(__float_as_uint(more) >> 23) - (int)(__float_as_uint(less) >> 23) <= 3;
}

// Two results at once of ordinary rows, by the operations of vl_quant_pair on packed numbers: `s`, `hi`, `over` of two
// queries, and of the held row its scale (for cosine half of it, for l2 twice), the negative of that, and its squared length.
// ALIKE: a + b is exact, and all are at most 16 times the shortest one.  `least` takes the smallest squared distance, or the smallest
// excess over that of near rows where lengths vary: where it is not above that of near rows, or not above 0, vl_quant_pair has to look at them.
template <int METRIC, bool NARROW, bool ALIKE>
__device__ __forceinline__ void vl_quant_pair2(int dot0, int dot1, vl_f2 s, vl_f2 hi, vl_f2 over, vl_f2 cs, vl_f2 ncs, vl_f2 rhi, vl_f2 rover,
                                               float& r0, float& r1, float& least)
{
    const vl_f2 f = vl_f2_pack((float)dot0, (float)dot1);
    const vl_f2 sh = vl_f2_mul(s, cs), nsh = vl_f2_mul(s, ncs);
    if (METRIC == VL_QUANT_PRODUCT) {
        vl_f2_unpack(NARROW ? vl_f2_mul(sh, f) : vl_f2_fma(sh, f, vl_f2_mul(vl_f2_fma(s, cs, nsh), f)), r0, r1);
    } else if (METRIC == VL_METRIC_COSINE) {
        const vl_f2 h = vl_f2_fma(nsh, f, vl_f2_pack(0.5f, 0.5f)), nsl = vl_f2_fma(s, ncs, sh);
        float f0, f1, h0, h1, l0, l1;
        vl_f2_unpack(f, f0, f1);
        vl_f2_unpack(h, h0, h1);
        vl_f2_unpack(nsl, l0, l1);
        r0 = __saturatef(__fmaf_rn(l0, f0, h0));
        r1 = __saturatef(__fmaf_rn(l1, f1, h1));
    } else {
        const vl_f2 ab = vl_f2_add(hi, rhi), sl = vl_f2_fma(s, cs, nsh);
        vl_f2 rest = vl_f2_add(over, rover);
        if (!ALIKE) {
            const vl_f2 of_r = vl_f2_sub(ab, hi);
            rest = vl_f2_add(rest, vl_f2_add(vl_f2_sub(vl_f2_sub(ab, of_r), hi), vl_f2_sub(of_r, rhi)));
        }
        const vl_f2 d = vl_f2_sub(vl_f2_fma(nsh, f, ab), vl_f2_fma(sl, f, rest));
        vl_f2_unpack(d, r0, r1);
        float l0, l1;
        vl_f2_unpack(ALIKE ? d : vl_f2_fma(vl_f2_pack(-kQuantNear, -kQuantNear), ab, d), l0, l1);
        asm("min.f32 %0, %1, %2, %3;" : "=f"(least) : "f"(l0), "f"(l1), "f"(least));
    }
}

// Up to so many queries of so many columns are held in 8 bits by the scan itself.
#define VL_QUANT_FEW_QUERIES 16
#define VL_QUANT_FEW_COLUMNS 4096

// Scores of every query against the rows [row_lo, row_hi) (vl_quant_scan.cu); codes of both are 16-byte aligned.  `queries`:
// few floating-point rows that the scan holds in 8 bits itself, or null: `q` has them.  `wait_us`: the longest wait inside, 0 for two seconds.
int vl_quant_scan(const void* queries, int q_type, int64_t q_ld, const VlQuantRows& q, int64_t nq, const VlQuantRows& rows, int64_t n,
                  int dim, int code_ld, int64_t row_lo, int64_t row_hi, void* out, int type, int64_t out_ld, int metric, int wait_us, int* status,
                  cudaStream_t stream);
