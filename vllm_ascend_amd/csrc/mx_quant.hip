// Rows of hidden states to MXFP4 and back, and the residual addition + RMS norm that hands its rows on quantised.
#include "mx_common.h"

#include <type_traits>

namespace moe355 {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMostThreads = 0xffffffff;  // of a launch

// HBM bound: 2 (4) bytes in and 17/32 out a value; 65536 rows of 7168 in 198 us, 6.0 TB/s.  (8192 rows, 149 MB, in 28 us; 23 on the same
// buffers again, which the 256 MiB of the last cache hold.)
template <int DT>
__global__ __launch_bounds__(kThreads) void mx_quant_kernel(const char* __restrict__ x, int64_t pieces,
                                                           uint32_t* __restrict__ codes, uint8_t* __restrict__ scale)
{
    mx_quant_piece<DT>(x, (int64_t)blockIdx.x * kThreads + threadIdx.x, pieces, codes, scale);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void mx_dequant_kernel(const uint32_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scale, int64_t pieces,
                                                             char* __restrict__ out)
{
    constexpr int kSize = DT == MOE355_DT_F32 ? 4 : 2;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= pieces) return;
    const uint32_t c = codes[i], b = scale[i >> 2];
    // 2^(b - 127); 2^-127 is subnormal, 255 stands for NaN
    const float s = __uint_as_float(b == 255 ? 0x7fc00000u : b == 0 ? 0x00400000u : b << 23);
    float v[8];
    const v2f p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    const v2f p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
    v[0] = p0[0] * s, v[1] = p0[1] * s, v[2] = p1[0] * s, v[3] = p1[1] * s;
    v[4] = p2[0] * s, v[5] = p2[1] * s, v[6] = p3[0] * s, v[7] = p3[1] * s;
    if constexpr (DT == MOE355_DT_F32) {
        v4f* to = (v4f*)(out + i * 8 * kSize);
        to[0] = (v4f){v[0], v[1], v[2], v[3]};
        to[1] = (v4f){v[4], v[5], v[6], v[7]};
    } else {
        v8u16 h;
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = f32_to_half<DT>(v[j]);
        *(v8u16*)(out + i * 8 * kSize) = h;
    }
}

// ------------------------------------------------------------------------------------------------ norm
// x = r16(x1 + x2); y = r16(f32(x / sqrt(mean x^2 + eps) * gamma + beta)); then y to int8 with a scale a row, by the sequence
// of dynamic_quant, or to MXFP4, or as it is.
//
// Squares, their sum and the norm itself are in 64 bits: a square of a 16-bit value is exact there, so the sum does not depend
// on how the row is spread over lanes to any bit that reaches y, and y is what the formula gives, rounded to 32 and to 16 bits.
// The launch is HBM bound all the same, 9 bytes a value to int8: 65536 rows of 7168 in 840 us, 5.0 TB/s (to MXFP4 690 us, 5.8 TB/s; a
// large copy reaches 5.0).  4096 rows, 264 MB, take 59 us (50); 49 (41) on the same buffers again, part of which the last cache
// holds.  A row of 7168 alone 5 us.
//
// y is rounded to 16 bits before it is quantised because that is what the next operators of the model see: the router's gate
// and a shared expert read y, and quantising y later gives the same codes.
struct NormArgs {
    const void *x1, *x2, *gamma, *beta;
    int64_t cols;
    double per_cols, eps;  // 1 / cols
    void *x, *y, *q, *scale;
};

// eight weights as they are held in memory
template <int GDT>
struct Weights8 {
    v8u16 h;
    __device__ __forceinline__ void fetch(const void* p, int64_t i) { h = ((const v8u16*)p)[i]; }
    __device__ __forceinline__ float at(int j) const { return half_to_f32<GDT>(h[j]); }
};
template <>
struct Weights8<MOE355_DT_F32> {
    v4f v[2];
    __device__ __forceinline__ void fetch(const void* p, int64_t i) { v[0] = ((const v4f*)p)[2 * i], v[1] = ((const v4f*)p)[2 * i + 1]; }
    __device__ __forceinline__ float at(int j) const { return v[j / 4][j % 4]; }
};

// 1 / sqrt(v): the hardware's estimate and two steps of Newton's method; what those cannot do (0, infinity, NaN, far ends) divides
__device__ __forceinline__ double reciprocal_root(double v)
{
    if (!(v > 0x1p-500 && v < 0x1p500)) return 1.0 / __builtin_sqrt(v);
    double r = __builtin_amdgcn_rsq(v);
#pragma unroll
    for (int i = 0; i < 2; ++i) r = r * __builtin_fma(-0.5 * v * r, r, 1.5);
    return r;
}

__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// One workgroup a row, NV pieces of eight values a thread (held in registers between the passes).  NV = 0: rows of any length,
// read again by every pass.
template <int DT, int GDT, int KIND, int NV>
__global__ __launch_bounds__(1024) void norm_quant_kernel(NormArgs a)
{
    __shared__ double sums[16];
    __shared__ float maxima[16];
    const int tid = threadIdx.x, wave = tid >> 6, nwaves = (int)(blockDim.x + 63) >> 6, threads = blockDim.x;
    const int64_t cols = a.cols, row = blockIdx.x, nv = cols >> 3;
    const v8u16* x1 = (const v8u16*)a.x1 + row * nv;
    const v8u16* x2 = a.x2 ? (const v8u16*)a.x2 + row * nv : nullptr;
    v8u16* xo = a.x ? (v8u16*)a.x + row * nv : nullptr;
    v8u16* yo = a.y ? (v8u16*)a.y + row * nv : nullptr;
    constexpr int HELD = NV > 0 ? NV : 1;
    const v8u16 zero = {0, 0, 0, 0, 0, 0, 0, 0};
    v8u16 held[HELD];

    auto sum_of = [&](int64_t i) {
        v8u16 v = x1[i];
        if (x2) {
            const v8u16 r = x2[i];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = f32_to_half<DT>(half_to_f32<DT>(v[j]) + half_to_f32<DT>(r[j]));
        }
        return v;
    };
    auto square = [&](v8u16 v) {
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double d = (double)half_to_f32<DT>(v[j]);
            s = __builtin_fma(d, d, s);
        }
        return s;
    };

    // the weights of the held pieces are asked for with them
    Weights8<GDT> gamma[HELD], beta[HELD];
    auto weights = [&](int64_t i, Weights8<GDT>& g, Weights8<GDT>& b) {
        g.fetch(a.gamma, i);
        if (a.beta) b.fetch(a.beta, i);
    };
    // non-temporal: 4096 rows of 7168 to int8 60 -> 55 us, to MXFP4 50 -> 43, 777 of 2048 5.3 -> 5.1, on the same buffers again (of
    // q as well: no difference)
    auto put = [&](v8u16* to, v8u16 v) { __builtin_nontemporal_store(v, to); };
    double sum = 0.0;
    if constexpr (NV > 0) {
#pragma unroll
        for (int n = 0; n < HELD; ++n) {
            const int64_t i = tid + (int64_t)n * threads;
            held[n] = i < nv ? sum_of(i) : zero;
            if (i < nv) weights(i, gamma[n], beta[n]);
        }
#pragma unroll
        for (int n = 0; n < HELD; ++n) {
            const int64_t i = tid + (int64_t)n * threads;
            if (xo && i < nv) put(xo + i, held[n]);
            sum += square(held[n]);
        }
    } else {
        for (int64_t i = tid; i < nv; i += threads) {
            const v8u16 v = sum_of(i);
            sum += square(v);
        }
    }
    sum = wave_sum_f64(sum);
    if ((tid & 63) == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < nwaves; ++w) sum += sums[w];
    const double by = reciprocal_root(sum * a.per_cols + a.eps);

    auto norm = [&](v8u16 v, const Weights8<GDT>& g, const Weights8<GDT>& b) {
        v8u16 y;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            double t = (double)half_to_f32<DT>(v[j]) * by * (double)g.at(j);
            if (a.beta) t += (double)b.at(j);
            y[j] = f32_to_half<DT>((float)t);
        }
        return y;
    };
    float largest = 0.0f;
    auto look = [&](v8u16 y) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = __builtin_fabsf(half_to_f32<DT>(y[j]));
            largest = f > largest ? f : largest;  // passes over NaN
        }
    };
    auto to_mx = [&](v8u16 y, int64_t i) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = half_to_f32<DT>(y[j]);
        const MxScale s = mx_scale(mx_largest_of_quad(v));
        ((uint32_t*)a.q)[row * nv + i] = mx_quantise8(v, s);
        if ((tid & 3) == 0) ((uint8_t*)a.scale)[(row * nv + i) >> 2] = (uint8_t)s.byte;
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int n = 0; n < HELD; ++n) {
            const int64_t i = tid + (int64_t)n * threads;
            if (i < nv) {
                held[n] = norm(held[n], gamma[n], beta[n]);
                if (yo) put(yo + i, held[n]);
                if constexpr (KIND == MOE355_NORM_INT8) look(held[n]);
                if constexpr (KIND == MOE355_NORM_MXFP4) to_mx(held[n], i);
            }
        }
    } else {
        for (int64_t i = tid; i < nv; i += threads) {
            weights(i, gamma[0], beta[0]);
            const v8u16 v = sum_of(i), y = norm(v, gamma[0], beta[0]);
            if constexpr (KIND == MOE355_NORM_INT8) look(y);
            else {
                if (xo) put(xo + i, v);
                if (yo) put(yo + i, y);
                if constexpr (KIND == MOE355_NORM_MXFP4) to_mx(y, i);
            }
        }
    }
    if constexpr (KIND == MOE355_NORM_INT8) {
        largest = wave_max(largest);
        if ((tid & 63) == 0) maxima[wave] = largest;
        __syncthreads();
        largest = 0.0f;
        for (int w = 0; w < nwaves; ++w) largest = maxima[w] > largest ? maxima[w] : largest;
        const float s = largest / 127.0f;
        const RowDivisor d = row_divisor(s);
        if (tid == 0) ((float*)a.scale)[row] = largest == 0.0f ? 0.0f : s;
        uint2* q = (uint2*)a.q + row * nv;
        auto emit = [&](auto fast) {
            constexpr bool F = decltype(fast)::value;
            if constexpr (NV > 0) {
#pragma unroll
                for (int n = 0; n < HELD; ++n) {
                    const int64_t i = tid + (int64_t)n * threads;
                    if (i < nv) q[i] = quantise_by_row<F, DT>(held[n], d);
                }
            } else {
                // the sums are written by this pass, the last one to read the inputs: they may be the same buffer
                for (int64_t i = tid; i < nv; i += threads) {
                    weights(i, gamma[0], beta[0]);
                    const v8u16 v = sum_of(i), y = norm(v, gamma[0], beta[0]);
                    if (xo) put(xo + i, v);
                    if (yo) put(yo + i, y);
                    q[i] = quantise_by_row<F, DT>(y, d);
                }
            }
        };
        if (d.fast) emit(std::true_type{});
        else emit(std::false_type{});
    }
}

// Pieces of eight values a thread (0: as many as it takes) and threads a row
struct NormShape {
    int per_thread;
    unsigned threads;
};
NormShape norm_shape(int64_t cols)
{
    const int64_t nv = cols >> 3;
    const unsigned waves = (unsigned)((nv + 63) / 64);
    // Two pieces a thread from 512 on: 4096 rows of 7168 to int8 74.1 -> 65.9 us, to MXFP4 59.6 -> 56.6 (four 65.7, 56.5, but a row
    // alone 7.7 instead of 6.3); 8192 rows of 2048 33.4 with one, 35.8 with two (the same buffers again).
    if (nv <= 512) return {1, 64 * waves};
    if (nv <= 2048) return {2, 64 * ((waves + 1) / 2)};
    return {0, 1024};
}

template <int DT, int GDT, int KIND>
void launch_norm(const NormArgs& a, int64_t rows, hipStream_t st)
{
    const NormShape s = norm_shape(a.cols);
    const dim3 grid((unsigned)rows), threads(s.threads);
    if (s.per_thread == 1) hipLaunchKernelGGL((norm_quant_kernel<DT, GDT, KIND, 1>), grid, threads, 0, st, a);
    else if (s.per_thread == 2) hipLaunchKernelGGL((norm_quant_kernel<DT, GDT, KIND, 2>), grid, threads, 0, st, a);
    else hipLaunchKernelGGL((norm_quant_kernel<DT, GDT, KIND, 0>), grid, threads, 0, st, a);
}

bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace
}  // namespace moe355

using namespace moe355;

extern "C" int moe355_dynamic_mx_quant(const void* x, int x_dtype, int64_t rows, int64_t cols, uint8_t* codes, uint8_t* scale,
                                       void* stream)
{
    if (rows < 0 || cols <= 0 || x_dtype < MOE355_DT_F32 || x_dtype > MOE355_DT_F16) return MOE355_E_ARG;
    if (cols % 32 || rows > (int64_t)1 << 40 || cols > (int64_t)1 << 20) return MOE355_E_SHAPE;
    if (rows == 0) return MOE355_OK;
    if (!x || !codes || !scale) return MOE355_E_ARG;
    if (!aligned(x, 16) || !aligned(codes, 4)) return MOE355_E_SHAPE;
    const int64_t pieces = rows * (cols / 8), groups = (pieces + kThreads - 1) / kThreads;
    if (groups > kMostThreads / kThreads) return MOE355_E_SHAPE;
#define MOE355_MXQ(D_)                                                                                                   \
    hipLaunchKernelGGL(mx_quant_kernel<D_>, dim3((unsigned)groups), dim3(kThreads), 0, (hipStream_t)stream, (const char*)x, \
                       pieces, (uint32_t*)codes, scale)
    if (x_dtype == MOE355_DT_BF16) MOE355_MXQ(MOE355_DT_BF16);
    else if (x_dtype == MOE355_DT_F16) MOE355_MXQ(MOE355_DT_F16);
    else MOE355_MXQ(MOE355_DT_F32);
#undef MOE355_MXQ
    return launch_status();
}

extern "C" int moe355_mx_dequant(const uint8_t* codes, const uint8_t* scale, int64_t rows, int64_t cols, void* out,
                                 int out_dtype, void* stream)
{
    if (rows < 0 || cols <= 0 || out_dtype < MOE355_DT_F32 || out_dtype > MOE355_DT_F16) return MOE355_E_ARG;
    if (cols % 32 || rows > (int64_t)1 << 40 || cols > (int64_t)1 << 20) return MOE355_E_SHAPE;
    if (rows == 0) return MOE355_OK;
    if (!codes || !scale || !out) return MOE355_E_ARG;
    if (!aligned(out, 16) || !aligned(codes, 4)) return MOE355_E_SHAPE;
    const int64_t pieces = rows * (cols / 8), groups = (pieces + kThreads - 1) / kThreads;
    if (groups > kMostThreads / kThreads) return MOE355_E_SHAPE;
#define MOE355_MXD(D_)                                                                                            \
    hipLaunchKernelGGL(mx_dequant_kernel<D_>, dim3((unsigned)groups), dim3(kThreads), 0, (hipStream_t)stream,        \
                       (const uint32_t*)codes, scale, pieces, (char*)out)
    if (out_dtype == MOE355_DT_BF16) MOE355_MXD(MOE355_DT_BF16);
    else if (out_dtype == MOE355_DT_F16) MOE355_MXD(MOE355_DT_F16);
    else MOE355_MXD(MOE355_DT_F32);
#undef MOE355_MXD
    return launch_status();
}

extern "C" int moe355_add_rms_norm_quant(const void* x1, const void* x2, const void* gamma, const void* beta, int x_dtype,
                                         int weight_dtype, int64_t rows, int64_t cols, double epsilon, int kind, void* x,
                                         void* y, void* q, void* scale, void* stream)
{
    if (rows < 0 || cols <= 0 || (x_dtype != MOE355_DT_BF16 && x_dtype != MOE355_DT_F16)) return MOE355_E_ARG;
    if (weight_dtype != x_dtype && weight_dtype != MOE355_DT_F32) return MOE355_E_ARG;
    if (kind < MOE355_NORM_PLAIN || kind > MOE355_NORM_MXFP4 || !(epsilon >= 0.0)) return MOE355_E_ARG;
    if (cols > (int64_t)1 << 20 || rows > kMostThreads / norm_shape(cols).threads || cols % (kind == MOE355_NORM_MXFP4 ? 32 : 8)) return MOE355_E_SHAPE;
    if (rows == 0) return MOE355_OK;
    if (!x1 || !gamma || (kind != MOE355_NORM_PLAIN ? !q || !scale : !y)) return MOE355_E_ARG;
    if (!aligned(x1, 16) || !aligned(x2, 16) || !aligned(x, 16) || !aligned(y, 16) || !aligned(q, 8) || !aligned(gamma, 16) ||
        !aligned(beta, 16))
        return MOE355_E_SHAPE;
    const NormArgs a = {x1, x2, gamma, beta, cols, 1.0 / (double)cols, epsilon, x, y, q, scale};
#define MOE355_NQ(D_, G_)                                                                                    \
    (kind == MOE355_NORM_INT8    ? launch_norm<D_, G_, MOE355_NORM_INT8>(a, rows, (hipStream_t)stream)       \
     : kind == MOE355_NORM_MXFP4 ? launch_norm<D_, G_, MOE355_NORM_MXFP4>(a, rows, (hipStream_t)stream)      \
                                 : launch_norm<D_, G_, MOE355_NORM_PLAIN>(a, rows, (hipStream_t)stream))
    if (x_dtype == MOE355_DT_BF16) {
        if (weight_dtype == MOE355_DT_F32) MOE355_NQ(MOE355_DT_BF16, MOE355_DT_F32);
        else MOE355_NQ(MOE355_DT_BF16, MOE355_DT_BF16);
    } else {
        if (weight_dtype == MOE355_DT_F32) MOE355_NQ(MOE355_DT_F16, MOE355_DT_F32);
        else MOE355_NQ(MOE355_DT_F16, MOE355_DT_F16);
    }
#undef MOE355_NQ
    return launch_status();
}
