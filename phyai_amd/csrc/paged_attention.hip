// Attention over pages: which kernel a call gets, and the kernels of plain calls over 16-bit pages (attention.h).
#include "attention.h"
#include "tuning.h"

#include <stdio.h>

namespace phyai {
namespace {

// magic = ceil(2^(31 + l) / d), l = ceil(log2 d)
Division division(uint32_t d) {
    if (d == 1) return {0, 0};
    uint32_t l = 1;
    while ((1ull << l) < d) ++l;
    return {(uint32_t)(((1ull << (31 + l)) + d - 1) / d), l - 1};
}

int64_t tiles_bound(int64_t T, int64_t B, int64_t group, int64_t rows) {
    return T * group / rows + (B < T ? B : T);   // every sequence with tokens adds less than one tile of its own
}
Plan make_plan(int64_t T, int64_t B, int64_t H, int64_t KV, int64_t D, int64_t max_kv, int64_t page_size) {
    Plan r = {};
    const int64_t group = H / KV;
    r.group_size = (int)group;
    r.page = division((uint32_t)page_size);
    r.group = division((uint32_t)group);
    // Many rows a workgroup once there are workgroups for most of the chip and rows enough to fill them.  Measured, many
    // against few: 104 workgroups of 256 dims 40 and 36 us, 208 of them 44 and 61 (156: 43 and 49); 136 of 128 dims 112 and 73, 264
    // of them 111 and 126; 288 of 64 dims (two to four fit a CU) 28 and 25, 576 of them 37 and 42.
    const int DP = padded_dim(D), waves = DP == 256 ? 4 : 8;
    const int64_t many = tiles_bound(T, B, group, 128) * KV;
    const char* forced = tuning_env("PHYAI_LAYER_ATTEND");   // 0: many rows; n: few rows, n splits
    r.many = forced != nullptr ? atoi(forced) == 0 : many >= (DP == 64 ? 512 : 192) && T * group >= 64 * B;
    r.tiles = (int)tiles_bound(T, B, group, r.many ? 128 : ROWS);
    r.splits = 1;
    if (!r.many) {
        // As many splits as workgroups run at once, and no more than give every wavefront a block: 32 tiles of 4096 keys 34 us
        // in one split, 18.5 in seven; 200 tiles of 816 keys 27.6 in one, 46 in two.
        const int64_t most = (max_kv + 32 * waves - 1) / (32 * waves), tiles = r.tiles * KV, at_once = DP == 64 ? 512 : 256;
        int64_t s = at_once / tiles;
        s = s < most ? s : most;
        if (forced != nullptr) s = atoi(forced);
        r.splits = (int)(s < 1 ? 1 : s < MAX_SPLITS ? s : MAX_SPLITS);
    }
    r.workers = division((uint32_t)(r.many ? 1 : r.splits * waves));
    return r;
}

// Calls that are more than plain ones.  PHYAI_LAYER_ATTEND_MORE = "many splits small shared_many shared_splits" (shared_splits 0: nothing is shared).
Plan make_plan_more(int64_t T, int64_t B, int64_t H, int64_t KV, int64_t D, int64_t max_kv, int64_t page_size, int64_t shared) {
    Plan r = make_plan(T, B, H, KV, D, max_kv, page_size);
    const int64_t group = H / KV;
    const int DP = padded_dim(D), waves = DP == 256 ? 4 : 8;
    int many = r.many, splits = r.splits, small = 0, shared_many = 0, shared_splits = 0;
    if (tuning_env("PHYAI_LAYER_ATTEND") == nullptr) {
        const int64_t at_once = DP == 64 ? 512 : 256;
        small = !many && r.tiles * KV >= at_once;
        if (shared > 0 && B > 1 && !many) {
            const int64_t once = (T * group + ROWS - 1) / ROWS;   // tiles of all rows together
            if (once < r.tiles) {
                // Workgroups with about as many keys each, as many as run at once, at least a block for every wavefront.
                const int64_t own = max_kv > shared ? max_kv - shared : 0, least = 32 * waves;
                int64_t keys = (once * KV * shared + r.tiles * KV * own + at_once - 1) / at_once;
                keys = keys < least ? least : keys;
                shared_splits = (int)((shared + keys - 1) / keys);
                splits = (int)((own + keys - 1) / keys);
            }
        }
    }
    if (const char* forced = tuning_env("PHYAI_LAYER_ATTEND_MORE")) sscanf(forced, "%d %d %d %d %d", &many, &splits, &small, &shared_many, &shared_splits);
    auto held = [](int v, int most) { return v < 1 ? 1 : v < most ? v : most; };
    r.many = many != 0;
    r.small = small != 0;
    r.tiles = (int)tiles_bound(T, B, group, r.many ? 128 : ROWS);
    if (shared > 0 && shared_splits > 0) {
        r.shared = (int)shared;
        r.shared_many = shared_many != 0;
        r.shared_tiles = (int)((T * group + (r.shared_many ? 128 : ROWS) - 1) / (r.shared_many ? 128 : ROWS));
        r.shared_splits = held(shared_splits, MAX_SPLITS / 2);
        splits = held(splits, MAX_SPLITS / 2);
    } else splits = held(splits, MAX_SPLITS);
    r.splits = r.shared_splits + splits;
    const int wide = r.small ? waves / 2 : waves;
    r.workers = division((uint32_t)(splits * (r.many ? 1 : wide)));
    if (r.shared > 0) r.shared_workers = division((uint32_t)(r.shared_splits * (r.shared_many ? 1 : wide)));
    return r;
}

}  // namespace

size_t paged_attention_workspace_bytes(int64_t T, int64_t B, int64_t H, int64_t KV, int64_t D, int64_t max_kv, int64_t shared, bool more) {
    if (T <= 0 || B <= 0) return 0;
    const Plan plan = more ? make_plan_more(T, B, H, KV, D, max_kv, 1, shared) : make_plan(T, B, H, KV, D, max_kv, 1);
    if (plan.splits == 1) return 0;
    return (size_t)plan.splits * T * H * (padded_dim(D) + 2) * sizeof(float);
}

hipError_t launch_paged_attention(const PagedAttention& p, hipStream_t stream) {
    const bool bf16 = p.type == HEAD_BF16;
    const int64_t max_kv = (int64_t)p.table_width * p.page_size;
    if (!p.more) {
        const Plan plan = make_plan(p.T, p.B, p.H, p.KV, p.D, max_kv, p.page_size);
        return bf16 ? launch_d<HEAD_BF16, 0>(p, plan, stream) : launch_d<HEAD_F16, 0>(p, plan, stream);
    }
    const Plan plan = make_plan_more(p.T, p.B, p.H, p.KV, p.D, max_kv, p.page_size, p.shared);
    if (p.k_scales != nullptr) return bf16 ? launch_attention_bf16_fp8(p, plan, stream) : launch_attention_f16_fp8(p, plan, stream);
    return bf16 ? launch_attention_bf16(p, plan, stream) : launch_attention_f16(p, plan, stream);
}

}  // namespace phyai
