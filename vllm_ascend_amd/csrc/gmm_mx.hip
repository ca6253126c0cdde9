// Products of MXFP4 rows with their experts' MXFP4 weights: to 16 bits, or through SwiGLU back to MXFP4.
#include "gmm_mx.h"

namespace moe355 {
namespace {

// [E, N, K / 2] codes and [E, N, K / 32] scales to the order of gmm_mx.h, 16 bytes a thread
__global__ __launch_bounds__(256) void mx_format_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scale,
                                                       int64_t channels, int64_t K, uint8_t* __restrict__ to,
                                                       uint8_t* __restrict__ to_scale)
{
    const int64_t steps = K / 64, windows = (K + 255) / 256, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int64_t unit = i >> 6, tile = unit / steps, step = unit % steps;
    if (tile >= channels / 32) return;
    const int64_t row = tile * 32 + (lane & 31), window = step >> 2, left = steps - 4 * window, nb = left < 4 ? left : 4;
    const int64_t block = window * 8 + half * nb + (step & 3);
    ((v4i*)to)[i] = *(const v4i*)(codes + row * (K / 2) + block * 16);
    to_scale[(tile * windows + window) * 256 + lane * 4 + (step & 3)] = scale[row * (K / 32) + block];
    if (step == steps - 1)
        for (int64_t j = nb; j < 4; ++j) to_scale[(tile * windows + window) * 256 + lane * 4 + j] = 0;
}

constexpr int kWaves = 4;

// Weights streamed: a workgroup has 64 channels of an expert (32 gate and their 32 up channels for SwiGLU) and its rows, 32 at
// a time; its wavefronts have every fourth window of K and add their sums through LDS.
template <int EPI, int DT>
__global__ __launch_bounds__(64 * kWaves) void gmm_mx_stream_kernel(MxArgs a)
{
    __shared__ float part[kWaves - 1][2][16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, e = blockIdx.y;
    const int64_t tiles = a.N / 32, steps = a.K / 64, windows = (a.K + 255) / 256;
    const int64_t t0 = EPI == MX_SWIGLU ? blockIdx.x : 2 * (int64_t)blockIdx.x;
    const bool two = EPI == MX_SWIGLU || t0 + 1 < tiles;
    const int64_t t1 = EPI == MX_SWIGLU ? t0 + tiles / 2 : two ? t0 + 1 : t0;
    int64_t row0, row1;
    mx_expert_rows(a, e, lane, row0, row1);
    const uint8_t* w0 = a.w + (e * tiles + t0) * steps * 1024 + lane * 16;
    const uint8_t* w1 = a.w + (e * tiles + t1) * steps * 1024 + lane * 16;
    const uint8_t* s0 = a.w_scale + (e * tiles + t0) * windows * 256 + lane * 4;
    const uint8_t* s1 = a.w_scale + (e * tiles + t1) * windows * 256 + lane * 4;
    for (int64_t r = row0; r < row1; r += 32) {
        const int64_t row = r + (lane & 31);
        int64_t token = row < row1 ? (a.row_token ? a.row_token[row] : row) : -1;
        const bool there = token >= 0 && token < a.x_rows;
        if (!there) token = 0;
        const uint8_t* x = a.x + token * (a.K / 2);
        const uint8_t* xs = a.x_scale + token * (a.K / 32);
        v16f acc0 = {}, acc1 = {};
        for (int64_t w = wave; w < windows; w += kWaves) {
            const int nb = steps - 4 * w < 4 ? (int)(steps - 4 * w) : 4;
            const int sa0 = *(const int*)(s0 + w * 256), sa1 = *(const int*)(s1 + w * 256);
            int sb = 0;
            if (there)
                for (int j = 0; j < nb; ++j) sb |= (int)xs[w * 8 + half * nb + j] << (8 * j);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j >= nb) break;
                const v4i a0 = *(const v4i*)(w0 + (4 * w + j) * 1024), a1 = *(const v4i*)(w1 + (4 * w + j) * 1024);
                v4i b = {0, 0, 0, 0};
                if (there) b = *(const v4i*)(x + w * 128 + half * nb * 16 + j * 16);
                acc0 = mfma_mx(a0, b, acc0, sa0, sb, j);
                acc1 = mfma_mx(a1, b, acc1, sa1, sb, j);
            }
        }
        if (wave > 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                part[wave - 1][0][i][lane] = acc0[i];
                part[wave - 1][1][i][lane] = acc1[i];
            }
        }
        __syncthreads();
        if (wave == 0) {
            for (int v = 0; v < kWaves - 1; ++v)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    acc0[i] += part[v][0][i][lane];
                    acc1[i] += part[v][1][i][lane];
                }
            const bool store = row < row1;
            if constexpr (EPI == MX_SWIGLU) {
                mx_swiglu_store(acc0, acc1, a.limit, half, store, (uint8_t*)a.out + row * (a.N / 4) + t0 * 16,
                                a.out_scale + row * (a.N / 64) + t0);
            } else {
                uint16_t* to = (uint16_t*)a.out + row * a.N;
                mx_store_half<DT>(acc0, half, store, to + t0 * 32);
                mx_store_half<DT>(acc1, half, store && two, to + t1 * 32);
            }
        }
        __syncthreads();
    }
}

bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

int check(const MxArgs& a, bool swiglu)
{
    if (a.rows < 0 || a.x_rows < 0 || a.K <= 0 || a.N <= 0 || a.E <= 0) return MOE355_E_ARG;
    if (a.gl_type != MOE355_GL_CUMSUM && a.gl_type != MOE355_GL_COUNT) return MOE355_E_ARG;
    if (a.K % 64 || a.N % (swiglu ? 64 : 32) || a.K > (int64_t)1 << 20 || a.N > (int64_t)1 << 20 || a.E > 32768)
        return MOE355_E_SHAPE;
    if (a.rows > 0x7fffffff || a.x_rows > 0x7fffffff) return MOE355_E_SHAPE;
    return MOE355_OK;
}

int run(const MxArgs& a, bool swiglu, int out_dtype, void* workspace, size_t workspace_bytes, hipStream_t st)
{
    if (const int rc = check(a, swiglu)) return rc;
    if (a.rows == 0) return MOE355_OK;
    if (!a.x || !a.x_scale || !a.w || !a.w_scale || (!a.group_list && a.E > 1) || !a.out || (swiglu && !a.out_scale)) return MOE355_E_ARG;
    if (!aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.w_scale, 4) || !aligned(a.out, 16)) return MOE355_E_SHAPE;
    if (a.rows >= 48 * (int64_t)a.E && mx_tiled_takes(a)) return launch_mx_tiled(a, swiglu, out_dtype, workspace, workspace_bytes, st);
    const dim3 grid((unsigned)((a.N / 32 + 1) / 2), (unsigned)a.E);
    if (swiglu) hipLaunchKernelGGL((gmm_mx_stream_kernel<MX_SWIGLU, MOE355_DT_BF16>), grid, dim3(64 * kWaves), 0, st, a);
    else if (out_dtype == MOE355_DT_BF16)
        hipLaunchKernelGGL((gmm_mx_stream_kernel<MX_HALF, MOE355_DT_BF16>), grid, dim3(64 * kWaves), 0, st, a);
    else hipLaunchKernelGGL((gmm_mx_stream_kernel<MX_HALF, MOE355_DT_F16>), grid, dim3(64 * kWaves), 0, st, a);
    return launch_status();
}

}  // namespace
}  // namespace moe355

using namespace moe355;

extern "C" int moe355_format_cast_mx(const uint8_t* codes, const uint8_t* scale, int64_t num_experts, int64_t n, int64_t k,
                                     uint8_t* codes_out, uint8_t* scale_out, void* stream)
{
    if (num_experts <= 0 || n <= 0 || k <= 0) return MOE355_E_ARG;
    if (n % 32 || k % 64 || n > (int64_t)1 << 20 || k > (int64_t)1 << 20 || num_experts > 32768) return MOE355_E_SHAPE;
    if (!codes || !scale || !codes_out || !scale_out) return MOE355_E_ARG;
    if (!aligned(codes, 16) || !aligned(codes_out, 16)) return MOE355_E_SHAPE;
    const int64_t channels = num_experts * n, groups = (channels / 32 * (k / 64) * 64 + 255) / 256;
    if (groups > 0x7fffffff) return MOE355_E_SHAPE;
    hipLaunchKernelGGL(mx_format_kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, codes, scale, channels, k,
                       codes_out, scale_out);
    return launch_status();
}

extern "C" size_t moe355_gmm_mx_workspace(int64_t rows, int64_t n, int64_t k, int num_experts)
{
    (void)n, (void)k;
    return rows > 0 && num_experts > 0 ? mx_tiled_workspace(rows, num_experts) : 256;
}

extern "C" int moe355_gmm_mx(const uint8_t* x, const uint8_t* x_scale, const int32_t* row_token, int64_t x_rows,
                             const uint8_t* w, const uint8_t* w_scale, const int64_t* group_list, int group_list_type,
                             int64_t rows, int64_t k, int64_t n, int num_experts, void* out, int out_dtype, void* workspace,
                             size_t workspace_bytes, void* stream)
{
    if (out_dtype != MOE355_DT_BF16 && out_dtype != MOE355_DT_F16) return MOE355_E_ARG;
    const MxArgs a = {x, x_scale, row_token, w, w_scale, group_list, group_list_type, rows, x_rows, k, n, num_experts, 0.0f,
                      out, nullptr};
    return run(a, false, out_dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int moe355_gmm_mx_swiglu_quant(const uint8_t* x, const uint8_t* x_scale, const int32_t* row_token, int64_t x_rows,
                                          const uint8_t* w, const uint8_t* w_scale, const int64_t* group_list,
                                          int group_list_type, int64_t rows, int64_t k, int64_t n, int num_experts,
                                          float swiglu_limit, uint8_t* out, uint8_t* out_scale, void* workspace,
                                          size_t workspace_bytes, void* stream)
{
    const MxArgs a = {x, x_scale, row_token, w, w_scale, group_list, group_list_type, rows, x_rows, k, n, num_experts,
                      swiglu_limit, out, out_scale};
    return run(a, true, MOE355_DT_BF16, workspace, workspace_bytes, (hipStream_t)stream);
}
