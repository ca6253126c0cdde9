// Products of MXFP4 rows with their experts' MXFP4 weights: to 16 bits, or through SwiGLU back to MXFP4.
#include "gmm_mx.h"
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

// Weights streamed, for few rows an expert.  A workgroup has 64 channels of an expert (32 gate channels and their 32 up
// channels for SwiGLU) and all its rows, 64 or, where no more are left, 32 at a time; its wavefronts have a part of K each and
// add their sums through LDS.  Every wavefront keeps the loads of two windows of 256 K on their way, 8 KiB of weights each,
// and nothing else waits for memory in between: HBM bound.
//
// How many wavefronts share a K: enough of them for the chip, no more (launch_stream).
template <int EPI, int DT>
struct MxStream {
    const MxArgs& a;
    float* lds;  // [wavefronts - 1][2][16][64]
    int lane, half, wave, waves, tiles, steps, windows, full, tail, w_begin, w_end, t0, t1;
    bool two;
    __amdgpu_buffer_rsrc_t w0, w1, ws0, ws1, xb, xsb;
    uint32_t scale_end;

    struct Weights {
        v4i a[2][4];
        int s[2];
    };
    template <int MT>
    struct Tokens {
        v4i b[MT][4];
        int s[MT];
    };

    template <bool ONCE>
    __device__ __forceinline__ void fetch_weights(int w, Weights& to) const
    {
        // past the end of this wavefront's part: nothing is read
        const int at = w < w_end ? w * 4096 + lane * 16 : 0x7ffff000, scale_at = w * 256 + lane * 4;
        constexpr int kHint = ONCE ? 2 : 0;  // the only reader: non-temporal
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            to.a[0][j] = __builtin_amdgcn_raw_buffer_load_b128(w0, at + j * 1024, 0, kHint);
            to.a[1][j] = __builtin_amdgcn_raw_buffer_load_b128(w1, at + j * 1024, 0, kHint);
        }
        to.s[0] = __builtin_amdgcn_raw_buffer_load_b32(ws0, scale_at, 0, 0);
        to.s[1] = __builtin_amdgcn_raw_buffer_load_b32(ws1, scale_at, 0, 0);
    }

    template <int MT>
    __device__ __forceinline__ void fetch_tokens(int w, const uint32_t (&x)[MT], const uint32_t (&xs)[MT], Tokens<MT>& to) const
    {
        w = w < w_end ? w : w_end - 1;
        const int nb = w < full ? 4 : tail;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            // (a shorter window's last pieces are the next row's, and not used)
            const uint32_t at = x[t] + w * 128 + half * nb * 16;
#pragma unroll
            for (int j = 0; j < 4; ++j) to.b[t][j] = __builtin_amdgcn_raw_buffer_load_b128(xb, at + j * 16, 0, 0);
            to.s[t] = mx_row_scales(xsb, xs[t] + w * 8 + half * nb, scale_end);
        }
    }

    template <int MT, bool WHOLE>
    __device__ __forceinline__ void multiply(const Weights& w, const Tokens<MT>& x, int nb, v16f (&acc)[2][MT]) const
    {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (WHOLE || j < nb) {
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    acc[0][t] = mfma_mx(w.a[0][j], x.b[t][j], acc[0][t], w.s[0], x.s[t], j);
                    acc[1][t] = mfma_mx(w.a[1][j], x.b[t][j], acc[1][t], w.s[1], x.s[t], j);
                }
            }
    }

    // rows r .. r + 32 MT - 1 of those up to row1
    template <int MT, bool ONCE>
    __device__ __forceinline__ void rows(int64_t r, int64_t row1)
    {
        Weights held[2];
        fetch_weights<ONCE>(w_begin, held[0]);
        uint32_t x[MT], xs[MT];
        bool there[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            int64_t row = r + t * 32 + (lane & 31);
            row = row < row1 ? row : row1 - 1;  // not stored
            int64_t token = a.row_token ? a.row_token[row] : row;
            there[t] = token >= 0 && token < a.x_rows;
            if (!there[t]) token = 0;
            x[t] = (uint32_t)token * (uint32_t)(a.K / 2);
            xs[t] = (uint32_t)token * (uint32_t)(a.K / 32);
        }
        v16f acc[2][MT] = {};
        if (w_begin < w_end) {
            Tokens<MT> tokens[2];
            fetch_tokens<MT>(w_begin, x, xs, tokens[0]);
            int w = w_begin;
            const int whole = w_end < full ? w_end : full;
            for (; w + 1 < whole; w += 2) {
                fetch_weights<ONCE>(w + 1, held[1]);
                fetch_tokens<MT>(w + 1, x, xs, tokens[1]);
                __builtin_amdgcn_sched_barrier(0);
                multiply<MT, true>(held[0], tokens[0], 4, acc);
                __builtin_amdgcn_sched_barrier(0);
                fetch_weights<ONCE>(w + 2, held[0]);
                fetch_tokens<MT>(w + 2, x, xs, tokens[0]);
                __builtin_amdgcn_sched_barrier(0);
                multiply<MT, true>(held[1], tokens[1], 4, acc);
                __builtin_amdgcn_sched_barrier(0);
            }
            for (; w < w_end; ++w) {  // at most two more, of which the last one may be short
                fetch_weights<ONCE>(w + 1, held[1]);
                fetch_tokens<MT>(w + 1, x, xs, tokens[1]);
                multiply<MT, false>(held[0], tokens[0], w < full ? 4 : tail, acc);
                held[0] = held[1];
                tokens[0] = tokens[1];
            }
        }
        // block t's sums meet in wavefront t % waves
        if (waves > 1) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int to = t % waves;
                if (wave != to) {
                    float* p = lds + ((wave > to ? wave - 1 : wave) * 32) * 64 + lane;
#pragma unroll
                    for (int i = 0; i < 16; ++i) p[i * 64] = acc[0][t][i], p[(16 + i) * 64] = acc[1][t][i];
                }
                __syncthreads();
                if (wave == to) {
                    for (int v = 0; v < waves - 1; ++v) {
                        const float* p = lds + v * 32 * 64 + lane;
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[0][t][i] += p[i * 64], acc[1][t][i] += p[(16 + i) * 64];
                    }
                }
                __syncthreads();
            }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if (t % waves != wave) continue;
            const int64_t row = r + t * 32 + (lane & 31);
            const bool store = row < row1;
            if (__any(!there[t])) {  // a row that is not there counts as zeros
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    acc[0][t][i] = there[t] ? acc[0][t][i] : 0.0f;
                    acc[1][t][i] = there[t] ? acc[1][t][i] : 0.0f;
                }
            }
            if constexpr (EPI == MX_SWIGLU) {
                mx_swiglu_store(acc[0][t], acc[1][t], a.limit, half, store, (uint8_t*)a.out + row * (a.N / 4) + t0 * 16,
                                a.out_scale + row * (a.N / 64) + t0);
            } else {
                uint16_t* to = (uint16_t*)a.out + row * a.N;
                mx_store_half<DT>(acc[0][t], half, store, to + t0 * 32);
                mx_store_half<DT>(acc[1][t], half, store && two, to + t1 * 32);
            }
        }
    }
};

template <int EPI, int DT>
__global__ __launch_bounds__(512) void gmm_mx_stream_kernel(MxArgs a)
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
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int tiles = (int)(a.N / 32), steps = (int)(a.K / 64), windows = (steps + 3) / 4, part = (windows + waves - 1) / waves;
    const int t0 = EPI == MX_SWIGLU ? blockIdx.x : 2 * blockIdx.x;
    const bool two = EPI == MX_SWIGLU || t0 + 1 < tiles;
    const int t1 = EPI == MX_SWIGLU ? t0 + tiles / 2 : two ? t0 + 1 : t0;
    const int64_t b0 = (int64_t)e * tiles + t0, b1 = (int64_t)e * tiles + t1;
    const int begin = wave * part < windows ? wave * part : windows, end = begin + part < windows ? begin + part : windows;
    MxStream<EPI, DT> s = {a, mx_parts, lane, lane >> 5, wave, waves, tiles, steps, windows, steps >> 2, steps & 3, begin, end, t0, t1,
                           two, mx_buffer(a.w + b0 * steps * 1024, steps * 1024), mx_buffer(a.w + b1 * steps * 1024, steps * 1024),
                           mx_buffer(a.w_scale + b0 * windows * 256, windows * 256),
                           mx_buffer(a.w_scale + b1 * windows * 256, windows * 256), mx_buffer(a.x, (uint32_t)(a.x_rows * (a.K / 2))),
                           mx_buffer(a.x_scale, mx_scale_bytes(a)), mx_scale_bytes(a) - 4};
    if (row1 - row0 <= 32) return s.template rows<1, true>(row0, row1);
    if (row1 - row0 <= 64) return s.template rows<2, true>(row0, row1);
    for (int64_t r = row0; r < row1; r += 64) s.template rows<2, false>(r, row1);
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
    if (a.rows >= 48 * (int64_t)a.E) return launch_mx_tiled(a, swiglu, out_dtype, workspace, workspace_bytes, st);
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
