// What the kernels of the MXFP4 products share.
//
// An operand of v_mfma_scale_f32_32x32x64_f8f6f4 with 4-bit values is 32 rows x 64 K: lane l holds row l % 32 and 32 values of
// its K, one block, in 16 bytes, and the block's scale in a byte of a register (which one: an immediate).  Any order of K will
// do as long as both operands have it, so a window of 256 K is taken as two runs of blocks, one for either half of the lanes:
// lane l reads blocks 4 (l / 32) .. + 3 of its row, 64 bytes that follow each other, and their scales as one register.  A last
// window of nb < 4 steps (K = 64 nb) has runs of nb blocks.
//
// Weights are kept in that order: [E][N / 32][K / 64] operands of 1 KiB (lane l's 16 bytes at 16 l), scales [E][N / 32][windows]
// of 256 bytes (lane l's four at 4 l).
//
// Channels are the rows of the product and tokens its columns: lane l has token l % 32, and of channels 8 (i / 4) + 4 (l / 32) +
// i % 4 the i-th of its 16 results; so a block of 32 output channels of a token is in two lanes.
//
// Sums are exact in most cases: products are multiples of 2^(sx + sw - 2), and 24 bits hold the sum of thousands of them with
// scales that lie some powers of two apart.  So the order of K, and its split over wavefronts, hardly ever shows.
#pragma once

#include <type_traits>

#include "mx_common.h"

namespace moe355 {

// 16 bytes written through the L2 (gmm_common.h measures what that does for the outputs of large products)
__device__ __forceinline__ void store16_through(void* p, v4i v)
{
    asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" ::"v"(p), "v"(v) : "memory");
}

struct MxArgs {
    const uint8_t* x;           // [x_rows, K / 2] codes
    const uint8_t* x_scale;     // [x_rows, K / 32]
    const int32_t* row_token;   // sorted row -> row of x, or NULL: the rows of x are sorted
    const uint8_t* w;           // operands as above
    const uint8_t* w_scale;
    const int64_t* group_list;  // NULL: one expert, all rows
    int gl_type;
    int64_t rows, x_rows, K, N;
    int E;
    float limit;                // SwiGLU's clamp
    void* out;                  // 16-bit [rows, N], or codes [rows, N / 4] of the N / 2 values of SwiGLU
    uint8_t* out_scale;         // [rows, N / 64]
    bool far;                   // the 16-bit output is larger than the last cache
};

enum { MX_HALF = 0, MX_SWIGLU = 1 };

// A 16-bit output that the 256 MiB of the last cache do not hold is stored past it: 65536 rows of 768 -> 2048, 268 MB, 129 -> 107 us
// (half as many rows: no difference, and what reads them next finds them there).
inline bool mx_far(int64_t rows, int64_t n) { return rows * n >= (int64_t)96 << 20; }

__device__ __forceinline__ v16f mfma_mx(v4i a, v4i b, v16f c, int sa, int sb, int j)
{
    const v8i A = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, B = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    // 4: both operands e2m1; the byte of the scale registers is an immediate
    switch (j) {
    case 0: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, c, 4, 4, 0, sa, 0, sb);
    case 1: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, c, 4, 4, 1, sa, 1, sb);
    case 2: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, c, 4, 4, 2, sa, 2, sb);
    default: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, c, 4, 4, 3, sa, 3, sb);
    }
}

// `bytes` of memory for buffer loads: an offset past them reads as zero
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_buffer(const void* p, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00027000);
}

// A row that is not there has this offset: past the end of x, and of its scales, with any offset into a row added (2^19 at most),
// so zeros times 2^-127.
constexpr uint32_t kMxNowhere = 0xfff00000;

__device__ __forceinline__ uint32_t mx_scale_bytes(const MxArgs& a)
{
    const int64_t n = a.x_rows * (a.K / 32);
    return (uint32_t)(n < 4 ? 4 : n);  // (the caller's memory has four)
}
// Scales of a row from an offset on, the first one in the low byte, as many of four as there are: at the end of the memory the last
// four bytes, shifted where they are used (a shift behind the load would wait for it).
struct MxRowScales {
    uint32_t raw, shift;
    __device__ __forceinline__ void fetch(__amdgpu_buffer_rsrc_t scales, uint32_t want, uint32_t end)
    {
        const uint32_t at = want < end ? want : end;
        raw = __builtin_amdgcn_raw_buffer_load_b32(scales, at, 0, 0);
        shift = 8 * (want - at);
    }
    __device__ __forceinline__ int get() const { return (int)(raw >> shift); }
};

// Rows [row0, row1) of expert e, inside [0, rows) whatever the list holds.  Every lane of a wavefront calls it.
__device__ __forceinline__ void mx_expert_rows(const MxArgs& a, int e, int lane, int64_t& row0, int64_t& row1)
{
    if (!a.group_list) {
        row0 = 0;
        row1 = a.rows;
    } else if (a.gl_type == MOE355_GL_CUMSUM) {
        row0 = e > 0 ? a.group_list[e - 1] : 0;
        row1 = a.group_list[e];
    } else {
        int64_t total = 0;
        for (int i = lane; i < e; i += 64) {
            const int64_t n = a.group_list[i];
            total += n < 0 ? 0 : n < a.rows ? n : a.rows;  // at most 2^31 each
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) total += __shfl_xor(total, off, 64);
        row0 = total;
        const int64_t n = a.group_list[e];
        row1 = row0 + (n < 0 ? 0 : n < a.rows ? n : a.rows);
    }
    row0 = row0 < 0 ? 0 : row0 > a.rows ? a.rows : row0;
    row1 = row1 < row0 ? row0 : row1 > a.rows ? a.rows : row1;
}

// With fewer rows than experts: the expert that has rows and `index` others that have some in front of it, and its rows.  No such
// expert: false.  Every lane of a wavefront calls it.
__device__ __forceinline__ bool mx_find_expert(const MxArgs& a, int index, int lane, int& e, int64_t& row0, int64_t& row1)
{
    const int32_t rows = (int32_t)a.rows;  // below 2^15, so that 32 bits hold the sum of the list
    auto cut = [&](int64_t n) { return (int32_t)(n < 0 ? 0 : n < rows ? n : rows); };
    int seen = 0;
    int32_t before = 0;
    for (int base = 0; base < a.E; base += 256) {
        int32_t n[4], from[4] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = base + 64 * j + lane;
            n[j] = i < a.E ? cut(a.group_list[i]) : 0;
            if (a.gl_type == MOE355_GL_CUMSUM) from[j] = i > 0 && i < a.E ? cut(a.group_list[i - 1]) : 0;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (a.gl_type == MOE355_GL_CUMSUM) n[j] = n[j] > from[j] ? n[j] - from[j] : 0;
            const uint64_t has = __ballot(n[j] > 0);
            const int here = __builtin_popcountll(has);
            const int32_t inc = wave_scan_inclusive_i32(n[j]);
            if (index < seen + here) {
                const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(has >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0));
                const int who = __builtin_ctzll(__ballot(n[j] > 0 && rank == index - seen));
                const int32_t size = __builtin_amdgcn_readlane(n[j], who);
                const int32_t at = a.gl_type == MOE355_GL_CUMSUM ? __builtin_amdgcn_readlane(from[j], who)
                                                                : before + __builtin_amdgcn_readlane(inc, who) - size;
                e = base + 64 * j + who;
                row0 = at < rows ? at : rows;
                row1 = at + size < rows ? at + size : rows;
                return row0 < row1;
            }
            seen += here;
            before += __builtin_amdgcn_readlane(inc, 63);
        }
    }
    return false;
}

// silu(g) u from its definition in 64 bits, rounded once
__device__ __forceinline__ float swiglu_f64(float g, float u)
{
    const double d = (double)g;
    return (float)(d / (1.0 + exp(-d)) * (double)u);
}

// A block of 32 output channels of a token, of which this lane has 16: silu(gate) * up to MXFP4, codes of channels 0-15 in the
// lower half of the wavefront, of 16-31 in the upper one, the scale in both.  Both halves call it together; `exists`: whether the
// lane's token does.
struct MxBlock {
    uint2 codes;
    uint32_t scale;
};
//
// What is quantised is the value of the formula, rounded to binary32.  The hardware's exp2 and reciprocal make it in 13 issue
// slots a value (a transcendental instruction takes four; the IEEE sequence of the int8 epilogues takes 30), off by at most
// 48 units in the last place for gates above -32: |g| 7.5e-8 from the rounded argument of exp2, 4e-7 from the rest.  That shows
// in the codes only next to a border: the middles between two codes and the powers of two where the scale changes, all of
// which have a mantissa of two bits and then zeros.  A value within 64 units of such a number (6 in 10^5 of them; infinities
// and NaN look like one) is computed again in 64 bits, and so is one with a gate below -32, unless it is small enough beside its
// block to have the code of zero anyway.  The codes are therefore those of the formula, bit for bit.
__device__ __forceinline__ MxBlock mx_swiglu(v16f g, v16f u, float limit, bool exists)
{
    if (limit > 0.0f) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            g[i] = g[i] > limit ? limit : g[i];
            u[i] = u[i] > limit ? limit : u[i];
            u[i] = u[i] < -limit ? -limit : u[i];
        }
    }
    constexpr uint32_t kNear = 64;
    float y[16];
    uint32_t near = 0xffffffffu;
    float least = 0.0f, m = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(g[i] * -1.44269504088896341f);
        y[i] = g[i] * u[i] * __builtin_amdgcn_rcpf(1.0f + e);
        const uint32_t key = (__float_as_uint(y[i]) << 11) + (kNear << 11);
        near = key < near ? key : near;
        least = __builtin_fminf(least, g[i]);
        m = __builtin_fmaxf(m, __builtin_fabsf(y[i]));  // passes over NaN, which `near` sees
    }
    auto block_scale = [&](uint32_t bits) {
        const v2u both = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
        return mx_scale(max_u32(both[0], both[1]));
    };
    MxScale s = block_scale(__float_as_uint(m));
    // (a block of all but nothing, whose products may have lost bits below the normal numbers, too)
    const bool tiny = s.byte < 32 && m > 0.0f;
    if (__any(exists && (near < (2 * kNear << 11) || least < -32.0f || tiny))) {
        uint32_t todo = 0;
        // over 2^e a value below 0.1 has the code of zero, even if the block's scale turns out to be half as large
        const float small = 0.1f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t key = (__float_as_uint(y[i]) << 11) + (kNear << 11);
            // (false for NaN; below -80 the exponential ends)
            const bool nothing = s.finite && !tiny && g[i] >= -80.0f && __builtin_fabsf(y[i]) * s.inverse < small;
            if ((key < (2 * kNear << 11) || g[i] < -32.0f || tiny) && g[i] != 0.0f && u[i] != 0.0f && !nothing) todo |= 1u << i;
        }
        if (!exists) todo = 0;
        while (todo) {
            const int at = __builtin_ctz(todo);
            todo &= todo - 1;
            float gi = g[0], ui = u[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) gi = i == at ? g[i] : gi, ui = i == at ? u[i] : ui;
            const float v = swiglu_f64(gi, ui);
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = i == at ? v : y[i];
        }
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) bits = max_u32(bits, __float_as_uint(y[i]) & 0x7fffffffu);
        s = block_scale(bits);
    }
    float v[2][8];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i / 8][i % 8] = y[i] * s.inverse;
    // 16 codes: channels 0-3, 8-11 (+ 4 in the upper half) and 16-19, 24-27
    const uint32_t low = s.finite ? mx_codes8(v[0]) : 0, high = s.finite ? mx_codes8(v[1]) : 0;
    // lower half: channels 0-15 of the block, upper half: 16-31
    const v2u p = __builtin_amdgcn_permlane32_swap(low, high, false, false);
    return {make_uint2(__builtin_amdgcn_perm(p[1], p[0], 0x05040100), __builtin_amdgcn_perm(p[1], p[0], 0x07060302)), s.byte};
}

// 16 of 32 channels of a token as 16-bit values: 16 p .. 16 p + 7 in the lower half of the wavefront, + 8 in the upper one
template <int DT>
__device__ __forceinline__ v4u mx_half(const v16f& y, int p)
{
    uint32_t d[2][2];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = 8 * p + 4 * q + 2 * k;
            d[q][k] = (uint32_t)f32_to_half<DT>(y[i]) | (uint32_t)f32_to_half<DT>(y[i + 1]) << 16;
        }
    const v2u s0 = __builtin_amdgcn_permlane32_swap(d[0][0], d[1][0], false, false);
    const v2u s1 = __builtin_amdgcn_permlane32_swap(d[0][1], d[1][1], false, false);
    return (v4u){s0[0], s1[0], s0[1], s1[1]};
}

// (expert, rows) of the 128-row tiles, in the order of the experts
struct MxMap {
    int32_t* count;
    int32_t *expert, *begin, *end;
};
constexpr int kMxTileRows = 128;
inline int64_t mx_most_tiles(int64_t rows, int E) { return rows / kMxTileRows + (rows < E ? rows : E); }
size_t mx_map_bytes(int64_t rows, int num_experts);
MxMap mx_map_in(void* workspace, int64_t rows, int num_experts);  // 256-byte aligned, mx_map_bytes long

// How a product of this shape runs: every expert's weights streamed by its own workgroups, or tiles, found by each workgroup from
// the group list or in a list that a launch in front makes (mx_build_map, or the routing launch).
enum MxForm { MX_STREAM, MX_TILES, MX_LISTED };
MxForm mx_form(int64_t rows, int64_t n, int num_experts, bool swiglu, bool grouped);
// a launch has at most 2^32 - 1 threads: 256 for every tile that the product may have
constexpr int64_t kMxMostGroups = 0xffffffff / 256;
inline bool mx_launches(int64_t rows, int64_t n, int num_experts, bool swiglu)
{
    const int64_t columns = swiglu ? (n / 64 + 3) / 4 : (n / 32 + 7) / 8;
    return columns * (mx_most_tiles(rows, num_experts) + 8) <= kMxMostGroups;
}
void mx_build_map(const MxArgs& a, const MxMap& map, hipStream_t st);
int mx_check(const MxArgs& a, bool swiglu);
// map: of MX_LISTED.  The arguments have been checked.
int mx_launch(const MxArgs& a, bool swiglu, int out_dtype, MxForm form, const MxMap& map, hipStream_t st);
int launch_mx_tiled(const MxArgs& a, bool swiglu, int out_dtype, MxForm form, const MxMap& map, hipStream_t st);

}  // namespace moe355
