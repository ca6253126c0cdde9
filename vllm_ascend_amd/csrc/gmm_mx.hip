// Products of MXFP4 rows with their experts' MXFP4 weights: to 16 bits, or through SwiGLU back to MXFP4.
#include "gmm_mx_stream.h"
#include <stdlib.h>

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

// Few rows an expert: a workgroup has 64 channels of an expert and all its rows, 32 at a time; its wavefronts have a part of K each
// and add their sums through LDS.  Three workgroups' wavefronts a SIMD (168 registers), which is why the form of 64 rows is not
// here.
template <int EPI, int DT>
__global__ __launch_bounds__(512, 3) void gmm_mx_stream_kernel(MxArgs a)
{
    extern __shared__ __attribute__((aligned(16))) float mx_parts[];
    const int e = blockIdx.y, lane = threadIdx.x & 63;
    // an expert without rows: seen before anything else is read
    if (a.group_list) {
        const int64_t n = a.group_list[e];
        if (n <= (a.gl_type == MOE355_GL_CUMSUM && e > 0 ? a.group_list[e - 1] : 0)) return;
    }
    int64_t row0, row1;
    mx_expert_rows(a, e, lane, row0, row1);
    if (row0 >= row1) return;
    const int tiles = (int)(a.N / 32), windows = (int)((a.K + 255) / 256);
    MxStream<EPI, DT> s = {a, mx_parts, lane, lane >> 5};
    s.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    s.waves = blockDim.x >> 6;
    const int part = (windows + s.waves - 1) / s.waves;
    s.w_begin = s.wave * part < windows ? s.wave * part : windows;
    s.w_end = s.w_begin + part < windows ? s.w_begin + part : windows;
    s.t0 = EPI == MX_SWIGLU ? blockIdx.x : 2 * blockIdx.x;
    s.store0 = true;
    s.store1 = EPI == MX_SWIGLU || s.t0 + 1 < tiles;
    s.t1 = EPI == MX_SWIGLU ? s.t0 + tiles / 2 : s.store1 ? s.t0 + 1 : s.t0;
    s.operands(e);
    if (row1 - row0 <= 32) return s.template rows<1, true>(row0, row1);
    for (int64_t r = row0; r < row1; r += 32) s.template rows<1, false>(r, row1);
}

template <int EPI, int DT>
void launch_stream(const MxArgs& a, hipStream_t st)
{
    const int64_t pairs = (a.N / 32 + 1) / 2, windows = (a.K + 255) / 256, experts = a.rows < a.E ? a.rows : a.E;
    int waves = 1;
    while (waves < 8 && pairs * experts * waves < 256 * 12 && 2 * waves <= windows) waves *= 2;
    if (const char* s = getenv("MXW")) waves = atoi(s);
    hipLaunchKernelGGL((gmm_mx_stream_kernel<EPI, DT>), dim3((unsigned)pairs, (unsigned)a.E), dim3(64 * waves),
                       (waves - 1) * 32 * 64 * 4, st, a);
}

bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

int check(const MxArgs& a, bool swiglu)
{
    if (a.rows < 0 || a.x_rows < 0 || a.K <= 0 || a.N <= 0 || a.E <= 0) return MOE355_E_ARG;
    if (a.gl_type != MOE355_GL_CUMSUM && a.gl_type != MOE355_GL_COUNT) return MOE355_E_ARG;
    if (a.K % 64 || a.N % (swiglu ? 64 : 32) || a.K > (int64_t)1 << 20 || a.N > (int64_t)1 << 20 || a.E > 32768)
        return MOE355_E_SHAPE;
    // rows of x are reached by offsets of 32 bits
    if (a.rows > 0x7fffffff || a.x_rows > 0x7fffffff || a.x_rows * (a.K / 2) > 0xfff00000) return MOE355_E_SHAPE;
    return MOE355_OK;
}

int run(const MxArgs& a, bool swiglu, int out_dtype, void* workspace, size_t workspace_bytes, hipStream_t st)
{
    if (const int rc = check(a, swiglu)) return rc;
    if (a.rows == 0) return MOE355_OK;
    if (a.x_rows == 0 || !a.x || !a.x_scale || !a.w || !a.w_scale || (!a.group_list && a.E > 1) || !a.out || (swiglu && !a.out_scale)) return MOE355_E_ARG;
    if (!aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.w_scale, 4) || !aligned(a.out, 16)) return MOE355_E_SHAPE;
    if (a.rows >= (getenv("MXT") ? atoi(getenv("MXT")) : 48) * (int64_t)a.E) return launch_mx_tiled(a, swiglu, out_dtype, workspace, workspace_bytes, st);
    if (swiglu) launch_stream<MX_SWIGLU, MOE355_DT_BF16>(a, st);
    else if (out_dtype == MOE355_DT_BF16) launch_stream<MX_HALF, MOE355_DT_BF16>(a, st);
    else launch_stream<MX_HALF, MOE355_DT_F16>(a, st);
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
