// Rows times streamed weights: a wavefront takes 64 channels of an expert (32 gate channels and their 32 up channels for
// SwiGLU) and 32 or 64 of its rows through all of K or a part of it.  It keeps the loads of two windows of 256 K on their way, 8
// KiB of weights each, and nothing else waits for memory in between: HBM bound, and L2 bound in the tokens from some 32 rows
// on, since nothing is shared between wavefronts.
#pragma once

#include "gmm_mx.h"

namespace moe355 {

template <int EPI, int DT>
struct MxStream {
    const MxArgs& a;
    float* lds;               // [waves - 1][2][16][64]
    int lane, half;
    int wave, waves;          // that share the K
    int full, tail;           // windows of 256 K; steps of a last, shorter one
    int w_begin, w_end;       // this wavefront's windows
    int t0, t1;               // its blocks of channels
    bool store0, store1;
    __amdgpu_buffer_rsrc_t w0, w1, ws0, ws1, xb, xsb;
    uint32_t scale_end;

    struct Weights {
        v4i a[2][4];
        int s[2];
    };
    template <int MT>
    struct Tokens {
        v4i b[MT][4];
        MxRowScales s[MT];
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
            to.s[t].fetch(xsb, xs[t] + w * 8 + half * nb, scale_end);
        }
    }

    template <int MT, bool WHOLE>
    __device__ __forceinline__ void multiply(const Weights& w, const Tokens<MT>& x, const bool (&there)[MT], int nb,
                                             v16f (&acc)[2][MT]) const
    {
        int s[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) s[t] = there[t] ? x.s[t].get() : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (WHOLE || j < nb) {
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    acc[0][t] = mfma_mx(w.a[0][j], x.b[t][j], acc[0][t], w.s[0], s[t], j);
                    acc[1][t] = mfma_mx(w.a[1][j], x.b[t][j], acc[1][t], w.s[1], s[t], j);
                }
            }
    }

    __device__ __forceinline__ void operands(int e)
    {
        const int64_t tiles = a.N / 32, steps = a.K / 64, windows = (steps + 3) / 4, b0 = e * tiles + t0, b1 = e * tiles + t1;
        full = (int)(steps >> 2);
        tail = (int)(steps & 3);
        w0 = mx_buffer(a.w + b0 * steps * 1024, (uint32_t)steps * 1024);
        w1 = mx_buffer(a.w + b1 * steps * 1024, (uint32_t)steps * 1024);
        ws0 = mx_buffer(a.w_scale + b0 * windows * 256, (uint32_t)windows * 256);
        ws1 = mx_buffer(a.w_scale + b1 * windows * 256, (uint32_t)windows * 256);
        xb = mx_buffer(a.x, (uint32_t)(a.x_rows * (a.K / 2)));
        scale_end = mx_scale_bytes(a) - 4;
        xsb = mx_buffer(a.x_scale, scale_end + 4);
    }

    // rows r .. r + 32 MT - 1 of those up to row1; ONCE: nobody else reads these weights
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
            const int64_t token = a.row_token ? a.row_token[row] : row;
            there[t] = token >= 0 && token < a.x_rows;
            x[t] = there[t] ? (uint32_t)token * (uint32_t)(a.K / 2) : kMxNowhere;
            xs[t] = there[t] ? (uint32_t)token * (uint32_t)(a.K / 32) : 0;
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
                multiply<MT, true>(held[0], tokens[0], there, 4, acc);
                __builtin_amdgcn_sched_barrier(0);
                fetch_weights<ONCE>(w + 2, held[0]);
                fetch_tokens<MT>(w + 2, x, xs, tokens[0]);
                __builtin_amdgcn_sched_barrier(0);
                multiply<MT, true>(held[1], tokens[1], there, 4, acc);
                __builtin_amdgcn_sched_barrier(0);
            }
            for (; w < w_end; ++w) {  // at most two more, of which the last one may be short
                fetch_weights<ONCE>(w + 1, held[1]);
                fetch_tokens<MT>(w + 1, x, xs, tokens[1]);
                multiply<MT, false>(held[0], tokens[0], there, w < full ? 4 : tail, acc);
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
            const bool store = row < row1 && store0;
            if constexpr (EPI == MX_SWIGLU) {
                const MxBlock b = mx_swiglu(acc[0][t], acc[1][t], a.limit, store);
                if (store) {
                    *(uint2*)((uint8_t*)a.out + row * (a.N / 4) + t0 * 16 + 8 * half) = b.codes;
                    if (half == 0) a.out_scale[row * (a.N / 64) + t0] = (uint8_t)b.scale;
                }
            } else {
                uint16_t* to = (uint16_t*)a.out + row * a.N + 8 * half;
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const v4u v0 = mx_half<DT>(acc[0][t], p), v1 = mx_half<DT>(acc[1][t], p);
                    if (store) *(v4u*)(to + t0 * 32 + 16 * p) = v0;
                    if (row < row1 && store1) *(v4u*)(to + t1 * 32 + 16 * p) = v1;
                }
            }
        }
    }
};

}  // namespace moe355
