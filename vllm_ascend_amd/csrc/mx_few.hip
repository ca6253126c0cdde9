// The MXFP4 experts of a few tokens: what one token costs is not the weight stream but launches, 2 to 4 us each on the GPU and 3.6 on
// the host.  There are two here, and nothing is sorted: every (token, slot) pair has workgroups of its own.
//
//   mx_up_few_kernel    a workgroup has a pair and 32 gate channels with their 32 up channels.  It quantises the pair's token itself,
//                       into LDS, while its first weights are on their way, and its wavefronts share K.
//   mx_down_few_kernel  a workgroup has 32 channels of a token and all its slots, a wavefront or more each, so that the token's rows
//                       meet in LDS and leave as one: the combine, and the counts of the experts by one more row of workgroups.
//
// The 32 columns of a product all have the pair's row; lanes 0 and 32 hold what is wanted.  An expert that several tokens chose is
// read for each of them, which is what ends the use (mx_few_takes).  One token through 8 of 128 experts of 2048 x 768 takes 16.6 us on
// the GPU, 11.4 with the weights of the call before (20 MB: 4 us; the two launches by themselves 9.6 and 6.5, or 7.0 and 5.9).
#include "mx_few.h"

namespace moe355 {
namespace {

constexpr int kFewWaves = 8;

// NB blocks of 32 channels of an expert, the windows [begin, end) of their K
template <int NB>
struct FewBlocks {
    __amdgpu_buffer_rsrc_t w[NB], ws[NB];
    int lane, half, full, tail, begin, end;  // whole windows of the row, steps of a last, shorter one

    struct Weights {
        v4i a[NB][4];
        int s[NB];
    };
    // the `part`-th of `parts` parts
    __device__ __forceinline__ FewBlocks(const MxArgs& a, int e, const int (&block)[NB], int part, int parts)
    {
        const int64_t tiles = a.N / 32, steps = a.K / 64;
        const int windows = (int)((steps + 3) / 4), share = (windows + parts - 1) / parts;
        lane = threadIdx.x & 63;
        half = lane >> 5;
        full = (int)(steps >> 2);
        tail = (int)(steps & 3);
        begin = part * share < windows ? part * share : windows;
        end = begin + share < windows ? begin + share : windows;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int64_t at = e * tiles + block[i];
            w[i] = mx_buffer(a.w + at * steps * 1024, (uint32_t)steps * 1024);
            ws[i] = mx_buffer(a.w_scale + at * windows * 256, (uint32_t)windows * 256);
        }
    }
    __device__ __forceinline__ int steps_of(int at) const { return at < full ? 4 : tail; }
    __device__ __forceinline__ void fetch(int at, Weights& to) const
    {
        const int from = at < end ? at * 4096 + lane * 16 : 0x7ffff000;  // past the end: nothing is read
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) to.a[i][j] = __builtin_amdgcn_raw_buffer_load_b128(w[i], from + j * 1024, 0, 0);
            to.s[i] = __builtin_amdgcn_raw_buffer_load_b32(ws[i], at * 256 + lane * 4, 0, 0);
        }
    }
    // `held`: the first window, asked for
    template <class Row>
    __device__ __forceinline__ void products(Weights (&held)[2], const Row& row, v16f (&acc)[NB]) const
    {
        typename Row::Held x[2];
        row.fetch(begin, steps_of(begin), x[0]);
        auto multiply = [&](const Weights& v, const typename Row::Held& r, int nb) {
            const int scale = row.scale(r);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < nb) {
                    const v4i c = row.codes(r, nb, j);
#pragma unroll
                    for (int i = 0; i < NB; ++i) acc[i] = mfma_mx(v.a[i][j], c, acc[i], v.s[i], scale, j);
                }
        };
        auto ask = [&](int at, int slot) {
            fetch(at, held[slot]);
            const int last = at < end ? at : end - 1;
            row.fetch(last, steps_of(last), x[slot]);
            __builtin_amdgcn_sched_barrier(0);
        };
        int at = begin;
        for (; at + 1 < end; at += 2) {
            ask(at + 1, 1);
            multiply(held[0], x[0], 4);  // (the last window, the only one that may be short, is the second one or comes below)
            __builtin_amdgcn_sched_barrier(0);
            ask(at + 2, 0);
            multiply(held[1], x[1], steps_of(at + 1));
            __builtin_amdgcn_sched_barrier(0);
        }
        if (at < end) multiply(held[0], x[0], steps_of(at));
    }
};

// A row in LDS: codes as they are, four scales a window and half of the lanes
struct FewRow {
    const uint8_t* row;
    const int* scales;
    int half;
    struct Held {
        int at;
    };
    __device__ __forceinline__ void fetch(int at, int, Held& to) const { to.at = at; }
    __device__ __forceinline__ v4i codes(const Held& h, int nb, int j) const { return *(const v4i*)(row + (h.at * 8 + half * nb + j) * 16); }
    __device__ __forceinline__ int scale(const Held& h) const { return scales[h.at * 2 + half]; }
    // where block b of a row of `blocks` blocks has its scale, in bytes
    static __device__ __forceinline__ int place(int b, int blocks)
    {
        const int w = b >> 3, left = blocks - 8 * w, nb = left < 8 ? left / 2 : 4, in = b & 7, h = in >= nb;
        return (w * 2 + h) * 4 + in - h * nb;
    }
};

// A row in memory, asked for with the weights
struct FewHidden {
    __amdgpu_buffer_rsrc_t x, xs;
    uint32_t from, scale_from, scale_end;
    int half;
    struct Held {
        v4i b[4];
        MxRowScales s;
    };
    __device__ __forceinline__ FewHidden(const MxArgs& a, int row, int half_) : half(half_)
    {
        scale_end = mx_scale_bytes(a) - 4;
        x = mx_buffer(a.x, (uint32_t)(a.x_rows * (a.K / 2)));
        xs = mx_buffer(a.x_scale, scale_end + 4);
        from = (uint32_t)row * (uint32_t)(a.K / 2);
        scale_from = (uint32_t)row * (uint32_t)(a.K / 32);
    }
    __device__ __forceinline__ void fetch(int at, int nb, Held& to) const
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) to.b[j] = __builtin_amdgcn_raw_buffer_load_b128(x, from + (at * 8 + half * nb + j) * 16, 0, 0);
        to.s.fetch(xs, scale_from + at * 8 + half * nb, scale_end);
    }
    __device__ __forceinline__ v4i codes(const Held& h, int, int j) const { return h.b[j]; }
    __device__ __forceinline__ int scale(const Held& h) const { return h.s.get(); }
};

template <int DT>
__global__ __launch_bounds__(256) void mx_up_few_kernel(MxArgs a, MxFew f)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
    const int lane = threadIdx.x & 63, half = lane >> 5, pair = blockIdx.y, tiles = (int)(a.N / 32);
    const int windows = (int)((a.K + 255) / 256), blocks = (int)(a.K / 32);
    const int e = f.ids[pair];
    if (e < 0 || e >= a.E) return;
    int* const scales = (int*)few_lds;                         // [windows][2]
    float* const sums = (float*)few_lds + (2 * windows + 3) / 4 * 4;  // [waves - 1][2][32]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    uint8_t* const row = (uint8_t*)(sums + (waves - 1) * 64);  // [windows][128]
    const FewBlocks<2> s(a, e, {(int)blockIdx.x, (int)blockIdx.x + tiles / 2}, wave, waves);
    FewBlocks<2>::Weights held[2];
    s.fetch(s.begin, held[0]);
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
    s.products(held, FewRow{row, scales, half}, acc);
    if (waves > 1) {
        if (wave > 0 && (lane & 31) == 0) {
            float* p = sums + (wave - 1) * 64 + half * 32;
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = acc[0][i], p[16 + i] = acc[1][i];
        }
        __syncthreads();
        if (wave > 0) return;
        for (int v = 0; v < waves - 1; ++v) {
            const float* p = sums + v * 64 + half * 32;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[0][i] += p[i], acc[1][i] += p[16 + i];
        }
    }
    const MxBlock b = mx_swiglu(acc[0], acc[1], a.limit, true);
    if ((lane & 31) == 0) {
        *(uint2*)((uint8_t*)a.out + pair * (a.N / 4) + blockIdx.x * 16 + 8 * half) = b.codes;
        if (half == 0) a.out_scale[pair * (a.N / 64) + blockIdx.x] = (uint8_t)b.scale;
    }
}

template <int DT>
__global__ __launch_bounds__(64 * kFewWaves) void mx_down_few_kernel(MxArgs a, MxFew f, int parts)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
    float* const sums = (float*)few_lds;  // [slots][parts][32]
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
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slot = wave / parts;
    const int pair = blockIdx.y * k + slot, e = f.ids[pair];
    if (e >= 0 && e < a.E) {
        const FewBlocks<1> s(a, e, {(int)blockIdx.x}, wave - slot * parts, parts);
        FewBlocks<1>::Weights held[2];
        s.fetch(s.begin, held[0]);
        v16f acc[1] = {};
        if (s.begin < s.end) s.products(held, FewHidden(a, pair, half), acc);
        if ((lane & 31) == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[wave * 32 + 8 * (i / 4) + 4 * half + i % 4] = acc[0][i];
        }
    }
    __syncthreads();
    // the sequence of the combine: 16-bit rows times their weights, slot by slot in 32 bits, the residual last
    const int64_t channel = (int64_t)blockIdx.x * 32 + threadIdx.x;
    if (threadIdx.x >= 32) return;
    float out = 0.0f;
    for (int i = 0; i < k; ++i) {
        const int id = f.ids[blockIdx.y * k + i];
        if (id < 0 || id >= a.E) continue;
        float v = sums[i * parts * 32 + threadIdx.x];
        for (int p = 1; p < parts; ++p) v += sums[(i * parts + p) * 32 + threadIdx.x];
        const float product = half_to_f32<DT>(f.probs[blockIdx.y * k + i]) * half_to_f32<DT>(f32_to_half<DT>(v));
        out = out + product;
    }
    const int64_t at = (int64_t)blockIdx.y * a.N + channel;
    if (f.residual) out = out + half_to_f32<DT>(f.residual[at]);
    ((uint16_t*)a.out)[at] = f32_to_half<DT>(out);
}

}  // namespace

bool mx_few_takes(int64_t tokens, int top_k, int64_t hidden, int64_t intermediate, int num_experts)
{
    // A wavefront for every slot of a token, a row of x in LDS; and the launches that it saves are worth some 125 million weights of
    // each projection in all, 50 million of them read again because several pairs have the same expert.  us on the GPU (same buffers), here /
    // sorted (the host gains 6 of 23 in all of them), and those two numbers: 128 experts of 2048 x 768, 1 / 4 / 8 / 16 tokens of 8
    // slots 12 / 20.7 / 29.8 / 48.2 against 17 / 25 / 34.5 / 46.3 (13, 50, 100, 201; 0); 8 of 1024 x 1408, 1 / 8 / 16 / 32 tokens of 2
    // slots 9.5 / 10.5 / 13.5 / 21.2 against 16 / 17.8 / 18 / 18.2 (3, 23, 46, 92; 0, 12, 35, 81); 64 of 2048 x 1408, 4 / 8 tokens of 6
    // slots 26.4 / 40.5 against 28.3 / 38 (69, 138; 0); 256 of 7168 x 2048, 1 / 2 tokens of 8 slots 36.3 / 76 against 41 / 71.6 (117, 235;
    // 0); 8 of 4096 x 1024 that 4 tokens have all 24.2 against 22.4 (134; 101); 128 of 1024 x 512, 16 tokens of 8 slots 22.7 against
    // 25.2 (67; 0); 16 of 512 x 256, 32 tokens of 4 slots 11.8 against 15.6 (17; 15).
    if (tokens > 32 || top_k > kFewWaves || tokens * top_k > 128 || hidden > 65536) return false;
    const int64_t pairs = tokens * top_k, again = pairs > num_experts ? pairs - num_experts : 0;
    return pairs * hidden * intermediate <= 125000000 && again * hidden * intermediate <= 50000000;
}

int mx_few(const MxArgs& up, const MxArgs& down, const MxFew& f, int dtype, int64_t tokens, hipStream_t st)
{
    const int64_t pairs = tokens * f.top_k, windows = (up.K + 255) / 256, windows2 = (down.K + 255) / 256;
    int waves = windows >= 28 ? 4 : windows >= 14 ? 2 : 1;
    while (waves < 4 && up.N / 64 * pairs * waves <= 256 && 2 * waves <= windows) waves *= 2;
    int parts = 1;
    while (2 * parts * f.top_k <= kFewWaves && 2 * parts <= windows2) parts *= 2;
    const size_t lds = (size_t)((2 * windows + 3) / 4 * 4) * 4 + (waves - 1) * 64 * 4 + windows * 128;
    const dim3 up_grid((unsigned)(up.N / 64), (unsigned)pairs), up_threads(64 * waves), down_threads(64 * f.top_k * parts);
    const dim3 down_grid((unsigned)(down.N / 32), (unsigned)tokens + 1);
    const size_t down_lds = (size_t)f.top_k * parts * 32 * 4;
    if (dtype == MOE355_DT_BF16) {
        hipLaunchKernelGGL(mx_up_few_kernel<MOE355_DT_BF16>, up_grid, up_threads, lds, st, up, f);
        hipLaunchKernelGGL(mx_down_few_kernel<MOE355_DT_BF16>, down_grid, down_threads, down_lds, st, down, f, parts);
    } else {
        hipLaunchKernelGGL(mx_up_few_kernel<MOE355_DT_F16>, up_grid, up_threads, lds, st, up, f);
        hipLaunchKernelGGL(mx_down_few_kernel<MOE355_DT_F16>, down_grid, down_threads, down_lds, st, down, f, parts);
    }
    return launch_status();
}

}  // namespace moe355
