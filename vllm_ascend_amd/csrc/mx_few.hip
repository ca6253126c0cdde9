// The MXFP4 experts of a few tokens: what one token costs is not the weight stream but launches, 2 to 4 us each on the GPU and 3.6 on
// the host.  There are two here, and nothing is sorted: every (token, slot) pair has workgroups of its own.
//
//   few_up_kernel    a workgroup has a pair and 32 gate channels with their 32 up channels.  It quantises the pair's token itself,
//                    into LDS, while its first weights are on their way, and its wavefronts share K.
//   few_down_kernel  a workgroup has 64 channels of a token and all its slots, a wavefront or more each, so that the token's rows
//                    meet in LDS and leave as one: the combine, and the counts of the experts by one more row of workgroups.
//
// The 32 columns of a product all have the pair's row; lanes 0 and 32 hold what is wanted.  An expert that several tokens chose is
// read for each of them, which is what ends the use (mx_few_takes).
#include "gmm_mx_stream.h"
#include "mx_few.h"

namespace moe355 {
namespace {

constexpr int kFewWaves = 8;

// 64 channels (two blocks) of this wavefront's windows; fetch(w) asks for a window's row, b(w, j) and scale(w) hand it over
template <class Stream, class Row>
__device__ __forceinline__ void few_stream(const Stream& s, typename Stream::Weights (&held)[2], const Row& row, v16f (&acc)[2])
{
    auto multiply = [&](const typename Stream::Weights& w, int at, int nb) {
        const int scale = row.scale(at);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < nb) {
                const v4i b = row.codes(at, nb, j);
                acc[0] = mfma_mx(w.a[0][j], b, acc[0], w.s[0], scale, j);
                acc[1] = mfma_mx(w.a[1][j], b, acc[1], w.s[1], scale, j);
            }
    };
    int w = s.w_begin;
    for (; w + 1 < s.w_end; w += 2) {
        s.template fetch_weights<false>(w + 1, held[1]);
        __builtin_amdgcn_sched_barrier(0);
        multiply(held[0], w, 4);  // (the last window, the only one that may be short, comes below or second)
        __builtin_amdgcn_sched_barrier(0);
        s.template fetch_weights<false>(w + 2, held[0]);
        __builtin_amdgcn_sched_barrier(0);
        multiply(held[1], w + 1, w + 1 < s.full ? 4 : s.tail);
        __builtin_amdgcn_sched_barrier(0);
    }
    if (w < s.w_end) multiply(held[0], w, w < s.full ? 4 : s.tail);
}

// A row in LDS: codes as they are, four scales a window and half of the lanes
struct FewRow {
    const uint8_t* row;
    const int* scales;
    int half;
    __device__ __forceinline__ v4i codes(int w, int nb, int j) const { return *(const v4i*)(row + (w * 8 + half * nb + j) * 16); }
    __device__ __forceinline__ int scale(int w) const { return scales[w * 2 + half]; }
    // where block b of a row of `blocks` blocks has its scale, in bytes
    static __device__ __forceinline__ int place(int b, int blocks)
    {
        const int w = b >> 3, left = blocks - 8 * w, nb = left < 8 ? left / 2 : 4, in = b & 7, h = in >= nb;
        return (w * 2 + h) * 4 + in - h * nb;
    }
};

template <int DT>
__global__ __launch_bounds__(256) void few_up_kernel(MxArgs a, MxFew f)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
    const int lane = threadIdx.x & 63, half = lane >> 5, pair = blockIdx.y, tiles = (int)(a.N / 32);
    const int windows = (int)((a.K + 255) / 256), blocks = (int)(a.K / 32);
    const int e = f.ids[pair];
    if (e < 0 || e >= a.E) return;
    int* const scales = (int*)few_lds;                         // [windows][2]
    float* const sums = (float*)few_lds + (2 * windows + 3) / 4 * 4;  // [waves - 1][2][32]
    MxStream<MX_SWIGLU, DT> s = {a, nullptr, lane, half};
    s.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    s.waves = blockDim.x >> 6;
    uint8_t* const row = (uint8_t*)(sums + (s.waves - 1) * 64);  // [K / 2], and a window's reach past it
    const int part = (windows + s.waves - 1) / s.waves;
    s.w_begin = s.wave * part < windows ? s.wave * part : windows;
    s.w_end = s.w_begin + part < windows ? s.w_begin + part : windows;
    s.t0 = blockIdx.x;
    s.t1 = s.t0 + tiles / 2;
    s.operands(e);
    typename MxStream<MX_SWIGLU, DT>::Weights held[2];
    s.template fetch_weights<false>(s.w_begin, held[0]);
    __builtin_amdgcn_sched_barrier(0);

    const int64_t token = pair / f.top_k;
    if (f.quantised) {
        for (int i = threadIdx.x; i < blocks; i += blockDim.x) {
            ((v4i*)row)[i] = *((const v4i*)((const uint8_t*)f.x + token * (a.K / 2)) + i);
            ((uint8_t*)scales)[FewRow::place(i, blocks)] = f.x_scale[token * blocks + i];
        }
    } else {
        for (int i = threadIdx.x; i < 4 * blocks; i += blockDim.x) {  // as mx_quant_piece does
            float v[8];
            load8<DT>((const uint16_t*)f.x + token * a.K + i * 8, v);
            const MxScale q = mx_scale(mx_largest_of_quad(v));
            ((uint32_t*)row)[i] = mx_quantise8(v, q);
            if ((lane & 3) == 0) ((uint8_t*)scales)[FewRow::place(i >> 2, blocks)] = (uint8_t)q.byte;
        }
    }
    __syncthreads();
    v16f acc[2] = {};
    few_stream(s, held, FewRow{row, scales, half}, acc);
    if (s.waves > 1) {
        if (s.wave > 0 && (lane & 31) == 0) {
            float* p = sums + (s.wave - 1) * 64 + half * 32;
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = acc[0][i], p[16 + i] = acc[1][i];
        }
        __syncthreads();
        if (s.wave > 0) return;
        for (int v = 0; v < s.waves - 1; ++v) {
            const float* p = sums + v * 64 + half * 32;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[0][i] += p[i], acc[1][i] += p[16 + i];
        }
    }
    const MxBlock b = mx_swiglu(acc[0], acc[1], a.limit, true);
    if ((lane & 31) == 0) {
        *(uint2*)((uint8_t*)a.out + pair * (a.N / 4) + s.t0 * 16 + 8 * half) = b.codes;
        if (half == 0) a.out_scale[pair * (a.N / 64) + s.t0] = (uint8_t)b.scale;
    }
}

// A row in memory, read where it is used
template <int EPI, int DT>
struct FewHidden {
    const MxStream<EPI, DT>& s;
    uint32_t x, xs;
    __device__ __forceinline__ v4i codes(int w, int nb, int j) const
    {
        return __builtin_amdgcn_raw_buffer_load_b128(s.xb, x + (w * 8 + s.half * nb + j) * 16, 0, 0);
    }
    __device__ __forceinline__ int scale(int w) const
    {
        MxRowScales r;
        r.fetch(s.xsb, xs + w * 8 + s.half * (w < s.full ? 4 : s.tail), s.scale_end);
        return r.get();
    }
};

template <int DT>
__global__ __launch_bounds__(64 * kFewWaves) void few_down_kernel(MxArgs a, MxFew f, int parts)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
    float* const sums = (float*)few_lds;  // [slots][parts][64]
    const int tokens = gridDim.y - 1, k = f.top_k;
    if ((int)blockIdx.y == tokens) {
        if (blockIdx.x > 0) return;
        for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
            int n = 0;
            for (int p = 0; p < tokens * k; ++p) n += f.ids[p] == e;
            f.expert_tokens[e] = n;
        }
        return;
    }
    const int lane = threadIdx.x & 63, half = lane >> 5, tiles = (int)(a.N / 32), windows = (int)((a.K + 255) / 256);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slot = wave / parts;
    const int pair = blockIdx.y * k + slot, e = f.ids[pair];
    if (e >= 0 && e < a.E) {
        MxStream<MX_HALF, DT> s = {a, nullptr, lane, half};
        const int part = (windows + parts - 1) / parts, mine = wave - slot * parts;
        s.w_begin = mine * part < windows ? mine * part : windows;
        s.w_end = s.w_begin + part < windows ? s.w_begin + part : windows;
        s.t0 = 2 * blockIdx.x;
        s.t1 = s.t0 + 1 < tiles ? s.t0 + 1 : s.t0;
        s.operands(e);
        typename MxStream<MX_HALF, DT>::Weights held[2];
        s.template fetch_weights<false>(s.w_begin, held[0]);
        v16f acc[2] = {};
        few_stream(s, held, FewHidden<MX_HALF, DT>{s, (uint32_t)pair * (uint32_t)(a.K / 2), (uint32_t)pair * (uint32_t)(a.K / 32)}, acc);
        if ((lane & 31) == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float* p = sums + wave * 64 + 8 * (i / 4) + 4 * half + i % 4;
                p[0] = acc[0][i];
                p[32] = acc[1][i];
            }
        }
    }
    __syncthreads();
    // the sequence of the combine: 16-bit rows times their weights, slot by slot in 32 bits, the residual last
    const int64_t channel = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x >= 64 || channel >= a.N) return;
    float out = 0.0f;
    for (int i = 0; i < k; ++i) {
        const int id = f.ids[blockIdx.y * k + i];
        if (id < 0 || id >= a.E) continue;
        float v = sums[i * parts * 64 + threadIdx.x];
        for (int p = 1; p < parts; ++p) v += sums[(i * parts + p) * 64 + threadIdx.x];
        const float product = half_to_f32<DT>(f.probs[blockIdx.y * k + i]) * half_to_f32<DT>(f32_to_half<DT>(v));
        out = out + product;
    }
    const int64_t at = (int64_t)blockIdx.y * a.N + channel;
    if (f.residual) out = out + half_to_f32<DT>(f.residual[at]);
    ((uint16_t*)a.out)[at] = f32_to_half<DT>(out);
}

}  // namespace

bool mx_few_takes(int64_t tokens, int top_k, int64_t hidden, int64_t intermediate)
{
    // A wavefront for every slot of a token, a row of x in LDS; and no more than what an expert that is read for each of its pairs
    // costs less than the launches do.  us on the GPU, here / sorted, and the pairs' products H I in millions: 128 experts of
    // 2048 x 768, 1 / 4 / 8 / 16 tokens of 8 slots 13.5 / 22 / 31 / 53 against 17 / 25 / 35 / 46 (12 / 50 / 100 / 201); 8 of 1024 x
    // 1408, 1 / 8 / 16 / 32 tokens of 2 slots 10.5 / 11.5 / 13.5 / 21.4 against 16 / 17.6 / 17.9 / 18.1 (3 / 23 / 46 / 92); 64 of
    // 2048 x 1408, 4 / 8 tokens of 6 slots 29.5 / 42 against 29 / 40 (69 / 138); 256 of 7168 x 2048, 1 / 2 tokens of 8 slots 39.7 / 77
    // against 41 / 71 (117 / 235); 8 of 4096 x 1024 that 4 tokens have all 24 against 21 (134); 16 tokens of 8 slots of 1024 x 512, 128
    // pairs of 128 experts 25.4 against 24.5 (67).  The host gains 6 us of 23 in all of them.
    return tokens <= 16 && top_k <= kFewWaves && tokens * top_k <= 64 && hidden <= 65536 &&
           tokens * top_k * hidden * intermediate <= 125000000;
}

int mx_few(const MxArgs& up, const MxArgs& down, const MxFew& f, int dtype, int64_t tokens, hipStream_t st)
{
    const int64_t pairs = tokens * f.top_k, windows = (up.K + 255) / 256, windows2 = (down.K + 255) / 256;
    int waves = windows >= 28 ? 4 : windows >= 14 ? 2 : 1;
    while (waves < 4 && up.N / 64 * pairs * waves <= 256 && 2 * waves <= windows) waves *= 2;
    int parts = 1;
    while (2 * parts * f.top_k <= kFewWaves && 2 * parts <= windows2) parts *= 2;
    const size_t lds = (size_t)((2 * windows + 3) / 4 * 4) * 4 + (waves - 1) * 64 * 4 + windows * 128;
    const dim3 up_grid((unsigned)(up.N / 64), (unsigned)pairs), down_grid((unsigned)((down.N / 32 + 1) / 2), (unsigned)tokens + 1);
    const size_t down_lds = (size_t)f.top_k * parts * 64 * 4;
    if (dtype == MOE355_DT_BF16) {
        hipLaunchKernelGGL(few_up_kernel<MOE355_DT_BF16>, up_grid, dim3(64 * waves), lds, st, up, f);
        hipLaunchKernelGGL(few_down_kernel<MOE355_DT_BF16>, down_grid, dim3(64 * f.top_k * parts), down_lds, st, down, f, parts);
    } else {
        hipLaunchKernelGGL(few_up_kernel<MOE355_DT_F16>, up_grid, dim3(64 * waves), lds, st, up, f);
        hipLaunchKernelGGL(few_down_kernel<MOE355_DT_F16>, down_grid, dim3(64 * f.top_k * parts), down_lds, st, down, f, parts);
    }
    return launch_status();
}

}  // namespace moe355
