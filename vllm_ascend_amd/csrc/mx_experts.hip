// All MXFP4 experts of a layer on a batch whose routing is known, as one call: a few tokens in two launches (mx_few.hip); otherwise index
// maps (with the tokens' quantisation and the list of tiles where a product wants one, by the same launch), both products, combine.
#include "gmm_mx.h"
#include "layer_parts.h"
#include "mx_few.h"

namespace moe355 {
namespace {

struct MxBuffers {
    uint8_t *codes, *scale, *hidden, *hidden_scale;
    int32_t *dst, *row_token;
    void *out, *map_ws, *tiles;
    size_t map_bytes, total;
    MxForm form13, form2;
};

MxBuffers lay_out(int64_t T, int k, int64_t H, int64_t I, int E, bool quantised, void* base)
{
    const int64_t R = T * k;
    MxBuffers b = {};
    char* at = (char*)base;
    auto take = [&](size_t bytes) {
        char* p = at + b.total;
        b.total += (bytes + 255) & ~(size_t)255;
        return (void*)p;
    };
    if (!quantised) {
        b.codes = (uint8_t*)take((size_t)T * H / 2);
        b.scale = (uint8_t*)take((size_t)T * H / 32);
    }
    b.hidden = (uint8_t*)take((size_t)R * I / 2);
    b.hidden_scale = (uint8_t*)take((size_t)R * I / 32);
    b.dst = (int32_t*)take((size_t)R * 4);
    b.row_token = (int32_t*)take((size_t)R * 4);
    b.out = take((size_t)R * H * 2);
    b.map_bytes = moe355_init_routing_workspace(T, k, E);
    b.map_ws = take(b.map_bytes);
    b.form13 = mx_form(R, 2 * I, E, true, true);
    b.form2 = mx_form(R, H, E, false, true);
    if (b.form13 == MX_LISTED || b.form2 == MX_LISTED) b.tiles = take(mx_map_bytes(R, E));
    return b;
}

bool bad_sizes(int64_t T, int k, int64_t H, int64_t I, int E)
{
    return T < 0 || k <= 0 || H <= 0 || I <= 0 || E <= 0;
}
bool unsupported(int64_t T, int k, int64_t H, int64_t I, int E)
{
    if (H % 64 || I % 64 || H > (int64_t)1 << 20 || I > (int64_t)1 << 19 || k > 64 || E > 2048 || T > 0x7ffffffe / k ||
        T * (H / 2) > kMxNowhere || T * k * (I / 2) > kMxNowhere)
        return true;
    // (the combine has a workgroup a token)
    return T > kMxMostGroups || !mx_launches(T * k, 2 * I, E, true) || !mx_launches(T * k, H, E, false);
}

}  // namespace
}  // namespace moe355

using namespace moe355;

extern "C" size_t moe355_mx_experts_workspace(int64_t num_tokens, int top_k, int64_t hidden, int64_t intermediate, int num_experts,
                                              int quantised)
{
    if (bad_sizes(num_tokens, top_k, hidden, intermediate, num_experts) || num_tokens == 0 ||
        unsupported(num_tokens, top_k, hidden, intermediate, num_experts))
        return 0;
    return lay_out(num_tokens, top_k, hidden, intermediate, num_experts, quantised != 0, nullptr).total;
}

extern "C" int moe355_mx_experts(const void* x, const uint8_t* x_scale, int dtype, int64_t num_tokens, int64_t hidden,
                                 const int32_t* topk_ids, const void* topk_weights, int top_k, const uint8_t* w13,
                                 const uint8_t* w13_scale, const uint8_t* w2, const uint8_t* w2_scale, int64_t intermediate,
                                 int num_experts, float swiglu_limit, const void* residual, int64_t* expert_tokens, void* out,
                                 void* workspace, size_t workspace_bytes, void* stream)
{
    const int64_t T = num_tokens, H = hidden, I = intermediate, R = T * top_k;
    const int E = num_experts;
    if (bad_sizes(T, top_k, H, I, E) || (dtype != MOE355_DT_BF16 && dtype != MOE355_DT_F16)) return MOE355_E_ARG;
    if (unsupported(T, top_k, H, I, E)) return MOE355_E_SHAPE;
    if (T == 0) return MOE355_OK;
    if (!x || !topk_ids || !topk_weights || !w13 || !w13_scale || !w2 || !w2_scale || !expert_tokens || !out) return MOE355_E_ARG;
    const uintptr_t all = (uintptr_t)x | (uintptr_t)w13 | (uintptr_t)w2 | (uintptr_t)out | (uintptr_t)residual;
    if ((all & 15) || (((uintptr_t)w13_scale | (uintptr_t)w2_scale) & 3)) return MOE355_E_SHAPE;
    const MxBuffers b = lay_out(T, top_k, H, I, E, x_scale != nullptr, workspace);
    if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < b.total) return MOE355_E_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    int rc;
    const uint8_t *codes = (const uint8_t*)x, *scale = x_scale;
    const MxQuantJob job = {x, dtype, T, H, b.codes, b.scale};
    if (!x_scale) {
        codes = b.codes;
        scale = b.scale;
    }
    if (mx_few_takes(T, top_k, H, I, E)) {
        const MxArgs up = {nullptr, nullptr, nullptr, w13, w13_scale, nullptr, MOE355_GL_COUNT, R, T, H, 2 * I, E, swiglu_limit,
                           b.hidden, b.hidden_scale, false};
        const MxArgs down = {b.hidden, b.hidden_scale, nullptr, w2, w2_scale, nullptr, MOE355_GL_COUNT, R, R, I, H, E, 0.0f, out,
                             nullptr, false};
        const MxFew few = {x, x_scale, x_scale != nullptr, topk_ids, (const uint16_t*)topk_weights, (const uint16_t*)residual, top_k,
                           expert_tokens};
        return mx_few(up, down, few, dtype, T, st);
    }
    TileSpec spec = {};
    bool built = false;
    MxMap map = {};
    if (b.tiles) {
        map = mx_map_in(b.tiles, R, E);
        spec.tm = {map.count, map.expert, map.begin, map.end};
        spec.BM = kMxTileRows;
        spec.max_tiles = (int)mx_most_tiles(R, E);
    }
    if ((rc = route_map_impl(topk_ids, T, top_k, E, 1, b.dst, b.row_token, expert_tokens, b.map_ws, b.map_bytes, &spec,
                             b.tiles ? 1 : 0, &built, stream, nullptr, 0, x_scale ? nullptr : &job)))
        return rc;
    const MxArgs up = {codes, scale, b.row_token, w13, w13_scale, expert_tokens, MOE355_GL_COUNT, R, T, H, 2 * I, E, swiglu_limit,
                       b.hidden, b.hidden_scale, false};
    const MxArgs down = {b.hidden, b.hidden_scale, nullptr, w2, w2_scale, expert_tokens, MOE355_GL_COUNT, R, R, I, H, E, 0.0f, b.out,
                         nullptr, mx_far(R, H)};
    if (b.tiles && !built) mx_build_map(up, map, st);
    if ((rc = mx_launch(up, true, dtype, b.form13, map, st))) return rc;
    if ((rc = mx_launch(down, false, dtype, b.form2, map, st))) return rc;
    return moe355_token_unpermute(b.out, dtype, b.dst, topk_weights, T, top_k, H, R, residual, out, stream);
}
