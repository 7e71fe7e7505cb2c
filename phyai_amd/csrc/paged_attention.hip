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

// What a launch is expected to take, in us: workgroups of one kind, `n` of them with `keys` each, of which `at_once` run together.
struct Part {
    int64_t n;
    double each;
};
double together(const Part* parts, int count, int64_t at_once) {
    int64_t n = 0;
    double sum = 0, longest = 0;
    for (int i = 0; i < count; ++i) {
        n += parts[i].n;
        sum += (double)parts[i].n * parts[i].each;
        longest = longest > parts[i].each ? longest : parts[i].each;
    }
    return n <= at_once ? longest : sum / (double)at_once + 0.3 * longest > longest ? sum / (double)at_once + 0.3 * longest : longest;
}

// Calls that are more than plain ones: few rows a workgroup with all its wavefronts or half of them (two of those a CU), or many rows, each
// with the keys split or not, and shared keys beside the sequences' own, for few rows or many.  The
// choice with the least expected time; a workgroup takes its start (9 us for few rows, 12 for many, fitted to measured times: three turns of
// memory, and instructions that a cold cache does not have) and its blocks of 32 keys a wavefront, or steps of 64, at what they take where the
// CU is full; sums to be joined take 4.5.  Measured, few rows with all wavefronts / half of them / many rows, best number of splits each, 8 bits and
// 32 heads on 8 of 128 dims unless said, more than one token with a cap but for 4096 keys: 64 single tokens of 8192 keys 165 / 155 / -, 16 of them 48 / 43, 4 of them 18 / 18, 32 of
// 400 9 / 12, 256 of 1000 101 / 86; 256 tokens of 1024 19 / 26 / 30, 512 of 512 23 / 17 / 25, 512 of 4096 76 / 72 / 61, 2048 of 8192 583 / 530 / 358; 1000 of 1000 of 64
// dims 40 / 30 / 38; 16 x 816 of 816 of 256 dims in 16 bits 144 / 116 / 98.  64 tokens behind 8192 shared keys and up to 512 of their
// own in 16 bits: few and few rows 64, many and few 39 (16 shared splits; 43 with 8, 49 with 32), nothing shared 110; 16 of them 25 and 24.
// The rule's choices there: 166, 48, 17, 12, 87, 19, 17, 74, 383, 40, 99 and 40, 26; late by a third for 32 of 400 and 1000 of 64 dims, by a fifth for 512 of 4096.
// (few_only: kernels for caps above kWideCap are there for few rows with all wavefronts.)
// PHYAI_LAYER_ATTEND_MORE = "many splits small shared_many shared_splits" (shared_splits 0: nothing is shared) forces one.
Plan make_plan_more(int64_t T, int64_t B, int64_t H, int64_t KV, int64_t D, int64_t max_kv, int64_t page_size, int64_t shared, int64_t window, bool few_only) {
    Plan r = make_plan(T, B, H, KV, D, max_kv, page_size);
    const int64_t group = H / KV;
    const int DP = padded_dim(D), waves = DP == 256 ? 4 : 8;
    int many = r.many, splits = r.splits, small = 0, shared_many = 0, shared_splits = 0;
    if (tuning_env("PHYAI_LAYER_ATTEND") == nullptr) {
        const double block = DP == 256 ? 3.0 : 2.4, join = 4.5;
        const int64_t few = tiles_bound(T, B, group, ROWS) * KV, wide = tiles_bound(T, B, group, 128) * KV;
        const int64_t seen = window > 0 && window + T / B + 64 < max_kv ? window + T / B + 64 : max_kv;   // keys of a tile
        auto ceiling = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
        auto few_rows = [&](int64_t tiles, int64_t keys, int s, int half) {
            return Part{tiles * s, 9.0 + (double)ceiling(keys, 32 * (half ? waves / 2 : waves) * s) * block};
        };
        auto many_rows = [&](int64_t tiles, int64_t keys, int s) {
            const double step = DP == 256 ? 3.5 : DP == 128 ? (tiles * s <= 256 ? 1.9 : 2.5) : tiles * s <= 256 ? 1.6 : 2.2;
            return Part{tiles * s, 12.0 + (double)ceiling(keys, 64 * s) * step};
        };
        const int64_t at_once_many = DP == 256 ? 256 : 512, at_once_mixed = DP == 64 ? 768 : at_once_many;
        auto at_once_few = [&](int half) -> int64_t { return DP == 64 ? (half ? 768 : 512) : half ? 512 : 256; };
        auto moved = [&](int s) { return s > 1 ? join + (double)(T * H) * DP * s / 1.5e6 : 0.0; };   // (the sums of all splits)
        double best = 1e30;
        auto take = [&](double t, int m, int s, int h, int sm, int ss) {
            if (t >= best) return;
            best = t;
            many = m; splits = s; small = h; shared_many = sm; shared_splits = ss;
        };
        for (int s = 1; s <= MAX_SPLITS; s = s < 8 ? s + 1 : s + s / 4) {
            for (int h = 0; h < 2; ++h) {
                const Part p = few_rows(few, seen, s, h);
                if (s == 1 || seen >= 32 * (h ? waves / 2 : waves) * (s - 1)) take(together(&p, 1, at_once_few(h)) + moved(s), 0, s, h, 0, 0);
            }
            const Part p = many_rows(wide, seen, s);
            if (s == 1 || seen >= 128 * s) take(together(&p, 1, at_once_many) + moved(s), 1, s, 0, 0, 0);
        }
        if (shared > 0 && B > 1 && few < (1 << 20)) {   // (beyond, a launch of all of them could have 2^32 threads)
            const int64_t own = max_kv > shared ? max_kv - shared : 1, once = ceiling(T * group, ROWS) * KV, once_wide = ceiling(T * group, 128) * KV;
            for (int ss = 1; ss <= MAX_SPLITS / 2; ss *= 2)
                for (int s = 1; s <= 4; s *= 2)
                    for (int h = 0; h < 2; ++h) {
                        const Part both[2] = {few_rows(once, shared, ss, h), few_rows(few, own, s, h)};
                        const Part before = many_rows(once_wide, shared, ss), wide_own = many_rows(wide, own, s);
                        const Part all_many[2] = {before, wide_own}, mixed[2] = {before, both[1]};
                        take(together(both, 2, at_once_few(h)) + moved(ss + s), 0, s, h, 0, ss);
                        if (shared >= 128 * ss && h == (DP != 256)) take(together(mixed, 2, at_once_mixed) + moved(ss + s), 0, s, h, 1, ss);
                        if (shared >= 128 * ss && h == 0) take(together(all_many, 2, at_once_many) + moved(ss + s), 1, s, 0, 1, ss);
                    }
        }
    }
    if (const char* forced = tuning_env("PHYAI_LAYER_ATTEND_MORE")) sscanf(forced, "%d %d %d %d %d", &many, &splits, &small, &shared_many, &shared_splits);
    if (few_only) many = small = shared_many = 0;   // (as many sums, so no other workspace)
    auto held = [](int v, int most) { return v < 1 ? 1 : v < most ? v : most; };
    r.many = many != 0;
    r.small = shared > 0 && shared_splits > 0 && shared_many != 0 && many == 0 ? DP != 256 : small != 0;   // (in one launch: four wavefronts)
    r.tiles = (int)tiles_bound(T, B, group, r.many ? 128 : ROWS);
    if (shared > 0 && shared_splits > 0) {
        r.shared = (int)shared;
        r.shared_many = shared_many != 0 || many != 0;   // (nobody has many rows of his own and few with the others)
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

size_t paged_attention_workspace_bytes(int64_t T, int64_t B, int64_t H, int64_t KV, int64_t D, int64_t max_kv, int64_t shared, int64_t window, bool more) {
    if (T <= 0 || B <= 0) return 0;
    const Plan plan = more ? make_plan_more(T, B, H, KV, D, max_kv, 1, shared, window, false) : make_plan(T, B, H, KV, D, max_kv, 1);
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
    const Plan plan = make_plan_more(p.T, p.B, p.H, p.KV, p.D, max_kv, p.page_size, p.shared, p.window, p.cap > kWideCap);
    if (p.k_scales != nullptr) return bf16 ? launch_attention_bf16_fp8(p, plan, stream) : launch_attention_f16_fp8(p, plan, stream);
    return bf16 ? launch_attention_bf16(p, plan, stream) : launch_attention_f16(p, plan, stream);
}

}  // namespace phyai
