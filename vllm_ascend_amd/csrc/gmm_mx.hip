// Products of MXFP4 rows with their experts' MXFP4 weights: to 16 bits, or through SwiGLU back to MXFP4.
#include "gmm_mx_stream.h"

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

// Few rows an expert: a workgroup has 64 channels of an expert and its rows, 32 at a time (every gridDim.z-th 32).  With fewer rows
// than experts it looks for its expert among those that have some, so that nothing is launched for the others (one token, 8 of 128
// experts of 2048 -> 2 x 768: 10.3 -> 5.6 us, of 256 of 7168 -> 2 x 2048: 34.8 -> 21.7).  Its wavefronts
// have a part of K each and add their sums through LDS.  Three wavefronts a SIMD (168 registers), which is why the form of 64 rows
// is not here.
template <int EPI, int DT>
__global__ __launch_bounds__(256, 3) void gmm_mx_stream_kernel(MxArgs a)
{
    extern __shared__ __attribute__((aligned(16))) float mx_parts[];
    const int lane = threadIdx.x & 63;
    int e = blockIdx.y;
    int64_t row0, row1;
    if (a.group_list && a.rows < a.E) {
        if (!mx_find_expert(a, blockIdx.y, lane, e, row0, row1)) return;
    } else {
        // an expert without rows: seen before anything else is read
        if (a.group_list) {
            const int64_t n = a.group_list[e];
            if (n <= (a.gl_type == MOE355_GL_CUMSUM && e > 0 ? a.group_list[e - 1] : 0)) return;
        }
        mx_expert_rows(a, e, lane, row0, row1);
    }
    if (row0 + 32 * (int64_t)blockIdx.z >= row1) return;
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
    for (int64_t r = row0 + 32 * blockIdx.z; r < row1; r += 32 * gridDim.z) s.template rows<1, false>(r, row1);
}

template <int EPI, int DT>
void launch_stream(const MxArgs& a, hipStream_t st)
{
    const int64_t pairs = (a.N / 32 + 1) / 2, windows = (a.K + 255) / 256, experts = a.rows < a.E ? a.rows : a.E;
    // chunks of 32 rows side by side, twice as many as an expert has on average
    const int64_t chunks = (2 * a.rows + 32 * a.E - 1) / (32 * a.E), most = (a.rows + 31) / 32, z = chunks < most ? chunks : most;
    // Wavefronts that share a K: two or four from 14 and 28 windows on, where a workgroup's start is less of it, and as long as there
    // are no more wavefronts than compute units; more than four are slower (fewer workgroups fit a compute unit).  us with
    // 1 / 2 / 4 / 8: 64 tokens, 256 experts of 7168 -> 2 x 2048 (28 windows) 497 / 493 / 487 / -, of 2048 -> 7168 (8 windows)
    // 258 / 255 / 276 / -; 4 tokens, 128 experts of 2048 -> 2 x 768 10.3 / 10.9 / 11.9 / 17.8, one token (192 workgroups) 5.7 / 5.6 /
    // 5.9 / 7.2; a row of 7168 -> 4096 (64 workgroups) 7.9 / 6.6 / 6.2 / 6.9, 32 rows 12.5 / 10.3 / 9.4 / 11.9.
    int waves = windows >= 28 ? 4 : windows >= 14 ? 2 : 1;
    while (waves < 4 && pairs * experts * z * waves <= 256 && 2 * waves <= windows) waves *= 2;
    hipLaunchKernelGGL((gmm_mx_stream_kernel<EPI, DT>), dim3((unsigned)pairs, (unsigned)experts, (unsigned)z), dim3(64 * waves),
                       (waves - 1) * 32 * 64 * 4, st, a);
}

bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace

int mx_check(const MxArgs& a, bool swiglu)
{
    if (a.rows < 0 || a.x_rows < 0 || a.K <= 0 || a.N <= 0 || a.E <= 0) return MOE355_E_ARG;
    if (a.gl_type != MOE355_GL_CUMSUM && a.gl_type != MOE355_GL_COUNT) return MOE355_E_ARG;
    if (a.K % 64 || a.N % (swiglu ? 64 : 32) || a.K > (int64_t)1 << 20 || a.N > (int64_t)1 << 20 || a.E > 32768)
        return MOE355_E_SHAPE;
    // rows of x are reached by offsets of 32 bits
    if (a.rows > 0x7fffffff || a.x_rows > 0x7fffffff || a.x_rows * (a.K / 2) > kMxNowhere) return MOE355_E_SHAPE;
    if (!mx_launches(a.rows, a.N, a.E, swiglu)) return MOE355_E_SHAPE;
    if (a.rows == 0) return MOE355_OK;
    if (a.x_rows == 0 || !a.x || !a.x_scale || !a.w || !a.w_scale || (!a.group_list && a.E > 1) || !a.out || (swiglu && !a.out_scale))
        return MOE355_E_ARG;
    if (!aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.w_scale, 4) || !aligned(a.out, 16)) return MOE355_E_SHAPE;
    return MOE355_OK;
}

MxForm mx_form(int64_t rows, int64_t n, int num_experts, bool swiglu, bool grouped)
{
    // Streaming has no list to make and splits K, so it is for calls that tiles would not fill the chip with: up to 512 workgroups
    // of 32 rows x 64 channels, and for fewer than 4 rows an expert.  us streamed / tiles, on the same buffers again: 8 experts of 1024
    // -> 2 x 1408, 64 / 128 / 256 tokens of 2 slots 6.5 / 7.7 / 9.8 against 8.1 / 10.9 / 12.9 (352, 352, 704 workgroups), of 1408 ->
    // 1024 64 / 256 tokens 5.2 / 5.3 against 7.0 / 9.8; one expert of 7168 -> 4096, 128 / 256 / 512 / 1024 rows 9.8 / 16.6 / 30.4 / 56
    // against 23.8 / 26.4 / 27.2 / 28.1 (256 to 2048 workgroups; between 512 and 1024 either may be ahead).  128 experts of 2048 -> 2 x
    // 768, 4 / 16 / 64 / 256 tokens of 8 slots 10.3 / 27.9 / 36.0 / 41.1 against 16.3 / 28.8 / 37.5 / 39.7.  Skewed (Zipf(1.1)) the same
    // with 64 / 256 tokens 25.9 / 65.8 against 28.8 / 39.9, 256 experts of 7168 -> 2 x 2048 with 64 / 127 / 128 tokens 157 / 223 / 218
    // against 171 / 217 / 193 and of 2048 -> 7168 with 64 / 127 77 / 111 against 86 / 108: a hot expert's many rows go through its few
    // workgroups, which pays for tiles from 4 rows an expert on.  (The call that this rule serves worst has one slot a token and all
    // tokens at one expert: 1000 of them at one of 256, 274 against 55.  Workgroups for more chunks of every expert's rows are no
    // remedy: six instead of one, 64 tokens of 256 experts 523 -> 630 uniform, 157 -> 193 skewed.)
    const int64_t pairs = swiglu ? n / 64 : (n / 32 + 1) / 2, chunks = (rows + 32 * (int64_t)num_experts - 1) / (32 * (int64_t)num_experts);
    if (rows < 4 * (int64_t)num_experts || pairs * num_experts * chunks <= 512) return MX_STREAM;
    // Finding the tiles in the product costs a workgroup for every tile that an expert might have, most of which end at once; a
    // list takes a launch of 5 us in front.  Found / listed, us, at 3 / 6 / 12 / 25 / 33 thousand of them: 35.8 / 37.3 / 39.4
    // / 52.0 / 38.0 against 38.3 / 40.7 / 43.3 / 53.0 / 33.2, the last two skewed 45.8 / 35.4 against 42.0 / 27.0.
    const int64_t columns = swiglu ? (n / 64 + 3) / 4 : (n / 32 + 7) / 8, tiles = (rows + kMxTileRows - 1) / kMxTileRows;
    return grouped && columns * num_experts * tiles > 16384 ? MX_LISTED : MX_TILES;
}

int mx_launch(const MxArgs& a, bool swiglu, int out_dtype, MxForm form, const MxMap& map, hipStream_t st)
{
    if (form != MX_STREAM) return launch_mx_tiled(a, swiglu, out_dtype, form, map, st);
    if (swiglu) launch_stream<MX_SWIGLU, MOE355_DT_BF16>(a, st);
    else if (out_dtype == MOE355_DT_BF16) launch_stream<MX_HALF, MOE355_DT_BF16>(a, st);
    else launch_stream<MX_HALF, MOE355_DT_F16>(a, st);
    return launch_status();
}

namespace {

int run(const MxArgs& a, bool swiglu, int out_dtype, void* workspace, size_t workspace_bytes, hipStream_t st)
{
    if (const int rc = mx_check(a, swiglu)) return rc;
    if (a.rows == 0) return MOE355_OK;
    const MxForm form = mx_form(a.rows, a.N, a.E, swiglu, a.group_list != nullptr);
    MxMap map = {};
    if (form == MX_LISTED) {
        if (!workspace || !aligned(workspace, 256) || workspace_bytes < mx_map_bytes(a.rows, a.E)) return MOE355_E_WORKSPACE;
        map = mx_map_in(workspace, a.rows, a.E);
        mx_build_map(a, map, st);
    }
    return mx_launch(a, swiglu, out_dtype, form, map, st);
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
    if (groups > 0xffffffff / 256) return MOE355_E_SHAPE;  // a launch has at most 2^32 - 1 threads
    hipLaunchKernelGGL(mx_format_kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, codes, scale, channels, k,
                       codes_out, scale_out);
    return launch_status();
}

extern "C" size_t moe355_gmm_mx_workspace(int64_t rows, int64_t n, int num_experts, int swiglu)
{
    if (rows <= 0 || n <= 0 || num_experts <= 0) return 0;
    return mx_form(rows, n, num_experts, swiglu != 0, true) == MX_LISTED ? mx_map_bytes(rows, num_experts) : 0;
}

extern "C" int moe355_gmm_mx(const uint8_t* x, const uint8_t* x_scale, const int32_t* row_token, int64_t x_rows,
                             const uint8_t* w, const uint8_t* w_scale, const int64_t* group_list, int group_list_type,
                             int64_t rows, int64_t k, int64_t n, int num_experts, void* out, int out_dtype, void* workspace,
                             size_t workspace_bytes, void* stream)
{
    if (out_dtype != MOE355_DT_BF16 && out_dtype != MOE355_DT_F16) return MOE355_E_ARG;
    const MxArgs a = {x, x_scale, row_token, w, w_scale, group_list, group_list_type, rows, x_rows, k, n, num_experts, 0.0f,
                      out, nullptr, mx_far(rows, n)};
    return run(a, false, out_dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int moe355_gmm_mx_swiglu_quant(const uint8_t* x, const uint8_t* x_scale, const int32_t* row_token, int64_t x_rows,
                                          const uint8_t* w, const uint8_t* w_scale, const int64_t* group_list,
                                          int group_list_type, int64_t rows, int64_t k, int64_t n, int num_experts,
                                          float swiglu_limit, uint8_t* out, uint8_t* out_scale, void* workspace,
                                          size_t workspace_bytes, void* stream)
{
    const MxArgs a = {x, x_scale, row_token, w, w_scale, group_list, group_list_type, rows, x_rows, k, n, num_experts,
                      swiglu_limit, out, out_scale, false};
    return run(a, true, MOE355_DT_BF16, workspace, workspace_bytes, (hipStream_t)stream);
}
