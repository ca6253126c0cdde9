// Products of MXFP4 rows and weights for many rows an expert.
//
// A workgroup of four wavefronts has a tile of 128 tokens x 256 channels (128 gate channels and their 128 up channels for
// SwiGLU), a wavefront 64 of those channels (a gate block and its up block) with all the tokens: 2 x 4 products of 32 x 32, 128
// accumulators a lane.  Tokens come through LDS, three windows of 256 K in a ring, by LDS-direct loads two windows ahead;
// weights go straight from the caches to registers in the order of their storage, as far ahead (a step's when the step that had
// its registers is done), since no other wavefront of the workgroup reads them.  A step of 64 K takes 8 matrix instructions of 32 cycles, 2 KiB of weights and 4 KiB of
// tokens a wavefront: while the matrix units do not pause, 64 of the 128 bytes a cycle that LDS gives and 48 of the 64 that a compute
// unit's L1 gets.  Two workgroups share a compute unit, so that the vector instructions of one's epilogue run beside the other's
// matrix instructions.
//
// us on the same buffers again / on buffers in turn: 65536 rows of 2048 -> 2 x 768 with SwiGLU 146 / 157 (2.8 / 2.6 PFLOP/s), of 768 ->
// 2048 105 / 123 (2.0 / 1.7; 3.8 / 3.3 TB/s), both with the list's 5; 2048 x 7168 x 4096 35 / 40 (3.4 / 3.0), 8192^3 258 on the same
// (4.3).  With the loads alone the first kernel takes 107, with the products and the start of a tile alone 104, with the epilogue 127:
// what is left is that neither hides all of the other.  By the counters its matrix units are busy for 35 % of the cycles, its L1s get
// 25 bytes a cycle, LDS loses 3 % to conflicts.
#include "gmm_mx_stream.h"

namespace moe355 {
namespace {

constexpr int kTileRows = kMxTileRows;
constexpr int kThreads = 256;
constexpr int kRing = 3;
constexpr int kStage = kTileRows * 128;  // tokens' bytes of a window
constexpr int kLds = kRing * (kStage + kTileRows * 8);

#define MOE355_LPTR(p) ((__attribute__((address_space(3))) void*)(p))

// One workgroup; thread t has the experts [t seg, (t + 1) seg).  Rows are cut to those that exist.
__global__ __launch_bounds__(1024) void mx_map_kernel(const int64_t* __restrict__ list, int gl_type, int E, int64_t rows, MxMap map,
                                                     int32_t most)
{
    __shared__ int64_t sums[16];
    __shared__ int32_t tiles_of[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, seg = (E + 1023) / 1024;
    const int e0 = tid * seg, e1 = e0 + seg < E ? e0 + seg : E;
    int64_t mine = 0, before = 0;
    if (gl_type == MOE355_GL_COUNT) {
        for (int e = e0; e < e1; ++e) {
            const int64_t n = list[e];
            mine += n < 0 ? 0 : n < rows ? n : rows;
        }
        int64_t inc = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int64_t o = __shfl_up(inc, off, 64);
            if (lane >= off) inc += o;
        }
        if (lane == 63) sums[wave] = inc;
        __syncthreads();
        before = inc - mine;
        for (int w = 0; w < wave; ++w) before += sums[w];
    }
    auto range = [&](int e, int64_t& row, int64_t& r0, int64_t& r1) {
        if (gl_type == MOE355_GL_COUNT) {
            const int64_t n = list[e];
            r0 = row;
            r1 = r0 + (n < 0 ? 0 : n < rows ? n : rows);
            row = r1;
        } else {
            r0 = e > 0 ? list[e - 1] : 0;
            r1 = list[e];
        }
        r0 = r0 < 0 ? 0 : r0 > rows ? rows : r0;
        r1 = r1 < r0 ? r0 : r1 > rows ? rows : r1;
    };
    int64_t row = before, r0, r1;
    int32_t tiles = 0;
    for (int e = e0; e < e1; ++e) {
        range(e, row, r0, r1);
        const int32_t n = (int32_t)((r1 - r0 + kTileRows - 1) / kTileRows);
        tiles = tiles + n < most ? tiles + n : most;  // (a list of sums that goes back and forth may name rows many times)
    }
    const int32_t inc = wave_scan_inclusive_i32(tiles);
    if (lane == 63) tiles_of[wave] = inc < 0 || inc > most ? most : inc;
    __syncthreads();
    int64_t at = inc < 0 ? most : inc - tiles, all = 0;
    for (int w = 0; w < 16; ++w) {
        if (w < wave) at += tiles_of[w];
        all += tiles_of[w];
    }
    if (tid == 0) map.count[0] = (int32_t)(all < most ? all : most);
    row = before;
    for (int e = e0; e < e1; ++e) {
        range(e, row, r0, r1);
        for (int64_t r = r0; r < r1 && at < most; r += kTileRows, ++at) {
            map.expert[at] = e;
            map.begin[at] = (int32_t)r;
            map.end[at] = (int32_t)r1;
        }
    }
}

// GRID: a workgroup has the tile (expert, one of those it may have) of its place in the grid, if there is one; otherwise one of the list, or
// of the one expert.  (Workgroups that stay and take turns through the list, with the next tile's place and rows known before they
// are through with one, were slower in every grouped product, 65536 rows of 2048 -> 2 x 768 179 us instead of 160: two that share a
// compute unit start their tiles together, and what the loop keeps does not fit the registers.)
template <int EPI, int DT, bool GRID>
__global__ __launch_bounds__(kThreads, 2) void gmm_mx_tiled_kernel(MxArgs a, MxMap map)
{
    // (not an array of a known size: the compiler would wait for every load on its way to it before each read)
    extern __shared__ __attribute__((aligned(16))) uint8_t mx_lds[];
    uint8_t* const tokens = mx_lds;
    int* const scales = (int*)(mx_lds + kRing * kStage);  // [kRing][rows][2]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int tiles = (int)(a.N / 32), steps = (int)(a.K / 64), windows = (steps + 3) / 4;
    const int columns = EPI == MX_SWIGLU ? (tiles / 2 + 3) / 4 : (tiles + 7) / 8;
    int e, column, tile;
    int64_t row0, row1;
    if constexpr (GRID) {
        e = blockIdx.y;
        column = blockIdx.x;
        tile = blockIdx.z;
        // an expert without rows for this workgroup: seen before anything else is read
        const int64_t n = min(a.group_list[e], a.rows), last = a.gl_type == MOE355_GL_CUMSUM && e > 0 ? a.group_list[e - 1] : 0;
        if (n - max(last, (int64_t)0) <= (int64_t)blockIdx.z * kTileRows) return;
        mx_expert_rows(a, e, lane, row0, row1);
        row0 += (int64_t)blockIdx.z * kTileRows;
        if (row0 >= row1) return;
    } else {
        // Consecutive workgroups run on different XCDs; an XCD takes a contiguous part of the tiles, all columns of a tile one
        // after the other, so that the tile's tokens and the expert's weights stay in its L2, in bands of 8 columns: the 64
        // workgroups of an XCD that run at a time share 8 tiles' tokens and 8 columns' weights (8192^3 330 -> 268 us).
        const uint32_t count = map.count ? map.count[0] : (uint32_t)((a.rows + kTileRows - 1) / kTileRows);
        const uint32_t items = count * columns, share = (items + 7) / 8, item = (blockIdx.x & 7) * share + (blockIdx.x >> 3);
        if ((blockIdx.x >> 3) >= share || item >= items) return;
        const uint32_t band = item / (count * 8), in = item - band * count * 8, wide = min(8u, (uint32_t)columns - band * 8);
        tile = (int)(in / wide);
        column = (int)(band * 8 + in - tile * wide);
        e = map.count ? map.expert[tile] : 0;
        row0 = map.count ? map.begin[tile] : (int64_t)tile * kTileRows;
        row1 = map.count ? map.end[tile] : a.rows;
    }

    // this wavefront's two blocks of channels (a block past the last one computes the last one again and is not stored)
    const int b0 = EPI == MX_SWIGLU ? column * 4 + wave : column * 8 + 2 * wave;
    const int last = EPI == MX_SWIGLU ? tiles / 2 - 1 : tiles - 1;
    const bool has0 = b0 <= last, has1 = EPI == MX_SWIGLU ? has0 : b0 + 1 <= last;
    const int t0 = has0 ? b0 : last, t1 = EPI == MX_SWIGLU ? t0 + tiles / 2 : has1 ? b0 + 1 : last;
    // A short tile: each wavefront by itself, without LDS.  The weights of an expert's only tile have no other reader; those of its
    // last tile are the other tiles' too, and stay in the caches (2500 tokens x 8 of 128 experts, 156 rows an expert: 2048 -> 2 x 768
    // 79 -> 70 us, 768 -> 2048 53 -> 46; without the hint in any tile 512 tokens of 7168 -> 2 x 2048 under Zipf(1.1) 295 -> 323).
    if (row1 - row0 <= 64) {
        MxStream<EPI, DT> s = {a, nullptr, lane, half, 0, 1, 0, 0, 0, windows, t0, t1, has0, has1};
        s.operands(e);
        const bool only = tile == 0 || (!GRID && map.count && map.expert[tile - 1] != e);
        if (row1 - row0 <= 32) return only ? s.template rows<1, true>(row0, row1) : s.template rows<1, false>(row0, row1);
        return only ? s.template rows<2, true>(row0, row1) : s.template rows<2, false>(row0, row1);
    }

    // Buffer loads: their offsets cost no registers, and what lies past the end of an operand is zero without being read.
    const auto w0 = mx_buffer(a.w + ((int64_t)e * tiles + t0) * steps * 1024, steps * 1024);
    const auto w1 = mx_buffer(a.w + ((int64_t)e * tiles + t1) * steps * 1024, steps * 1024);
    const auto ws0 = mx_buffer(a.w_scale + ((int64_t)e * tiles + t0) * windows * 256, windows * 256);
    const auto ws1 = mx_buffer(a.w_scale + ((int64_t)e * tiles + t1) * windows * 256, windows * 256);

    // Tokens' bytes of a window: row-major, 128 bytes a row, the 16-byte pieces exchanged by row pair so that the 16 lanes that
    // LDS serves at a time find theirs in different banks.  A load fills 8 rows; wavefront v has rows 32 v .. + 31.  Scales: thread
    // t has row t / 2, half t % 2.
    auto row_of = [&](int64_t row) -> int32_t { return row >= row1 ? -1 : a.row_token ? a.row_token[row] : (int32_t)row; };
    int32_t token[5];
#pragma unroll
    for (int i = 0; i < 4; ++i) token[i] = row_of(row0 + wave * 32 + i * 8 + (lane >> 3));
    token[4] = row_of(row0 + (threadIdx.x >> 1));
    const int tail = steps & 3, full = steps >> 2;  // steps of a last, shorter window; whole windows
    const auto xb = mx_buffer(a.x, (uint32_t)(a.x_rows * (a.K / 2)));
    auto there = [&](int32_t t) { return t >= 0 && t < a.x_rows; };
    uint32_t from[4];
    const int piece = (lane & 7) ^ (lane >> 4);  // of rows 8 i + lane / 8 with even i; with odd ones piece ^ 4
#pragma unroll
    for (int i = 0; i < 4; ++i)
        from[i] = there(token[i]) ? (uint32_t)token[i] * (uint32_t)(a.K / 2) + (piece ^ (i & 1) * 4) * 16 : kMxNowhere;
    const uint32_t scale_from = there(token[4]) ? (uint32_t)token[4] * (uint32_t)(a.K / 32) : kMxNowhere;

    auto fetch_tokens = [&](int w, int slot) {
        // (a shorter last window's last pieces are the next row's, and not used)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xb, MOE355_LPTR(tokens + slot * kStage + (wave * 4 + i) * 1024), 16,
                                                     from[i] + w * 128, 0, 0, 0);
    };
    const auto x_scales = mx_buffer(a.x_scale, mx_scale_bytes(a));
    const uint32_t scale_end = scale_from == kMxNowhere ? 0xffffffff : mx_scale_bytes(a) - 4;
    auto fetch_scale = [&](int w) {
        MxRowScales s;
        s.fetch(x_scales, scale_from + w * 8 + (threadIdx.x & 1) * (w < full ? 4 : tail), scale_end);
        return s;
    };
    struct Weights {
        v4i a[2][4];
        int s[2];
    };
    auto fetch_step = [&](int w, int j, Weights& to) {
        const int at = w * 4096 + lane * 16;
        to.a[0][j] = __builtin_amdgcn_raw_buffer_load_b128(w0, at + j * 1024, 0, 0);
        to.a[1][j] = __builtin_amdgcn_raw_buffer_load_b128(w1, at + j * 1024, 0, 0);
    };
    auto fetch_weight_scales = [&](int w, Weights& to) {
        const int at = w * 256 + lane * 4;
        to.s[0] = __builtin_amdgcn_raw_buffer_load_b32(ws0, at, 0, 0);
        to.s[1] = __builtin_amdgcn_raw_buffer_load_b32(ws1, at, 0, 0);
    };
    auto fetch_weights = [&](int w, Weights& to) {
#pragma unroll
        for (int j = 0; j < 4; ++j) fetch_step(w, j, to);
        fetch_weight_scales(w, to);
    };

    v16f acc[2][4] = {};
    const int row_in = lane & 31;
    auto compute = [&](int slot, Weights& w, int nb, int refill, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        int sb[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) sb[t] = scales[slot * (2 * kTileRows) + (t * 32 + row_in) * 2 + half];
        const uint8_t* base = tokens + slot * kStage + row_in * 128;
        v4i b[4];
        auto read = [&](int j, int t) { b[t] = *(const v4i*)(base + t * 32 * 128 + ((half * nb + j) ^ (row_in >> 1 & 7)) * 16); };
#pragma unroll
        for (int t = 0; t < 4; ++t) read(0, t);
        // the next step's tokens into the registers that this step's products have just used, six products ahead
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (WHOLE || j < nb) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    acc[0][t] = mfma_mx(w.a[0][j], b[t], acc[0][t], w.s[0], sb[t], j);
                    acc[1][t] = mfma_mx(w.a[1][j], b[t], acc[1][t], w.s[1], sb[t], j);
                    if (WHOLE ? j < 3 : j + 1 < nb) read(j + 1, t);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (WHOLE) fetch_step(refill, j, w);
        }
        if constexpr (WHOLE) fetch_weight_scales(refill, w);
    };

    Weights held[2];
    const int own = threadIdx.x, end = windows - 1;
    auto cut = [&](int w) { return w < end ? w : end; };
    // Prologue: windows 0 and 1 on their way, in this order: what waits for the scales of window 1 waits for the tokens of window 0
    // (the compiler does not know that the reads of LDS depend on them, and would move a load of tokens behind the scales).
    fetch_weights(0, held[0]);
    fetch_weights(1, held[1]);
    __builtin_amdgcn_sched_barrier(0);
    fetch_tokens(0, 0);
    __builtin_amdgcn_sched_barrier(0);
    const MxRowScales scale_first = fetch_scale(0);
    MxRowScales scale_next = fetch_scale(cut(1));
    __builtin_amdgcn_sched_barrier(0);
    fetch_tokens(cut(1), 1);
    __builtin_amdgcn_sched_barrier(0);
    scales[own] = scale_first.get();
    // Window w: its tokens and weights have been asked for two windows ago, a step's weights when the step that had their
    // registers was done.  Behind the barrier everybody has read window w - 1, whose place in the ring window w + 2 takes.
    int slot = 0;
    auto window = [&](int w, Weights& now, auto whole) {
        const int slot1 = slot == 2 ? 0 : slot + 1, slot2 = slot == 0 ? 2 : slot - 1;
        scales[slot1 * (2 * kTileRows) + own] = scale_next.get();
        // behind this window's tokens: the next window's 4 loads of tokens and 10 of weights, at least
        asm volatile("s_waitcnt vmcnt(14) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        scale_next = fetch_scale(cut(w + 2));
        __builtin_amdgcn_sched_barrier(0);
        fetch_tokens(cut(w + 2), slot2);
        __builtin_amdgcn_sched_barrier(0);
        compute(slot, now, decltype(whole)::value || w < full ? 4 : tail, w + 2, whole);
        __builtin_amdgcn_sched_barrier(0);
        slot = slot1;
    };
    // products before the vector instructions of the other workgroup's prologue and epilogue
    __builtin_amdgcn_s_setprio(1);
    constexpr std::true_type whole{};
    constexpr std::false_type part{};
    int w = 0;
    for (; w + 1 < full; w += 2) {
        window(w, held[0], whole);
        window(w + 1, held[1], whole);
    }
    for (; w < windows; ++w) {  // at most two more, of which the last one may be short
        window(w, held[0], part);
        held[0] = held[1];
    }
    __builtin_amdgcn_s_setprio(0);
    // The results go through LDS, which turns them into whole lines: once the loads past the end have landed and everybody has
    // read the last window.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const bool exists = row0 + t * 32 + row_in < row1;
        if constexpr (EPI == MX_SWIGLU) {
            // 64 bytes of codes a row, and four scales behind all of them
            const MxBlock b = mx_swiglu(acc[0][t], acc[1][t], a.limit, exists && has0);
            *(uint2*)(tokens + (t * 32 + row_in) * 64 + wave * 16 + 8 * half) = b.codes;
            if (half == 0) tokens[kTileRows * 64 + (t * 32 + row_in) * 4 + wave] = (uint8_t)b.scale;
        } else {
            // 128 bytes a row of this wavefront's 64 channels, the pieces exchanged as the tokens' are; three blocks in turn
            uint8_t* patch = tokens + (wave * 3 + t % 3) * 4096;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int p = 0; p < 2; ++p)
                    *(v4u*)(patch + row_in * 128 + ((c * 4 + p * 2 + half) ^ (row_in >> 1 & 7)) * 16) = mx_half<DT>(acc[c][t], p);
            wave_lds_order();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + (lane >> 3), piece = lane & 7;
                const int64_t row = row0 + t * 32 + r;
                const v4i v = *(const v4i*)(patch + r * 128 + (piece ^ (r >> 1 & 7)) * 16);
                if (row < row1 && (piece < 4 ? has0 : has1)) {
                    if (a.far) __builtin_nontemporal_store(v, (v4i*)((uint16_t*)a.out + row * a.N + b0 * 32 + piece * 8));
                    else store16_through((uint16_t*)a.out + row * a.N + b0 * 32 + piece * 8, v);
                }
            }
            wave_lds_order();
        }
    }
    if constexpr (EPI == MX_SWIGLU) {
        __syncthreads();
        // a thread has half of a row
        const int r = threadIdx.x >> 1, h = threadIdx.x & 1, left = last + 1 - column * 4;  // blocks of 32 channels
        const int64_t row = row0 + r;
        if (row < row1) {
            const v4i* held = (const v4i*)(tokens + r * 64 + h * 32);
            v4i* to = (v4i*)((uint8_t*)a.out + row * (a.N / 4) + column * 64 + h * 32);
            if (2 * h < left) to[0] = held[0];
            if (2 * h + 1 < left) to[1] = held[1];
            uint8_t* scale = a.out_scale + row * (a.N / 64) + column * 4 + h * 2;
            const uint8_t* held_scale = tokens + kTileRows * 64 + r * 4 + h * 2;
            if (2 * h < left) scale[0] = held_scale[0];
            if (2 * h + 1 < left) scale[1] = held_scale[1];
        }
    }
}

}  // namespace

size_t mx_map_bytes(int64_t rows, int num_experts)
{
    return (size_t)((64 + 3 * mx_most_tiles(rows, num_experts)) * 4 + 255) / 256 * 256;
}

MxMap mx_map_in(void* workspace, int64_t rows, int num_experts)
{
    int32_t* q = (int32_t*)workspace;
    const int64_t most = mx_most_tiles(rows, num_experts);
    return {q, q + 64, q + 64 + most, q + 64 + 2 * most};
}

void mx_build_map(const MxArgs& a, const MxMap& map, hipStream_t st)
{
    hipLaunchKernelGGL(mx_map_kernel, dim3(1), dim3(1024), 0, st, a.group_list, a.gl_type, a.E, a.rows, map,
                       (int32_t)mx_most_tiles(a.rows, a.E));
}

int launch_mx_tiled(const MxArgs& a, bool swiglu, int out_dtype, MxForm form, const MxMap& map, hipStream_t st)
{
    const int64_t columns = swiglu ? (a.N / 64 + 3) / 4 : (a.N / 32 + 7) / 8, tiles = (a.rows + kTileRows - 1) / kTileRows;
    const bool direct = form == MX_TILES && a.group_list;
    const int64_t most = (form == MX_LISTED ? mx_most_tiles(a.rows, a.E) : tiles) * columns, groups = (most + 7) / 8 * 8;
    const dim3 grid = direct ? dim3((unsigned)columns, (unsigned)a.E, (unsigned)tiles) : dim3((unsigned)groups);
#define MOE355_MXT(E_, D_)                                                                                       \
    do {                                                                                                         \
        if (direct)                                                                                              \
            hipLaunchKernelGGL((gmm_mx_tiled_kernel<E_, D_, true>), grid, dim3(kThreads), kLds, st, a, map);     \
        else                                                                                                     \
            hipLaunchKernelGGL((gmm_mx_tiled_kernel<E_, D_, false>), grid, dim3(kThreads), kLds, st, a, map);    \
    } while (0)
    if (swiglu) MOE355_MXT(MX_SWIGLU, MOE355_DT_BF16);
    else if (out_dtype == MOE355_DT_BF16) MOE355_MXT(MX_HALF, MOE355_DT_BF16);
    else MOE355_MXT(MX_HALF, MOE355_DT_F16);
#undef MOE355_MXT
    return launch_status();
}

}  // namespace moe355
