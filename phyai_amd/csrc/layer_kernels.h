// Problems and launchers of the kernels behind include/phyai_layer.h: the block-scaled fp8 linear, head norms with
// rotation, attention over pages.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace phyai {

// Launches a kernel and says whether that went well - of this launch, whatever older error the thread may have.
template <typename T>
struct SameType {
    using type = T;
};
template <typename... P>
inline hipError_t enqueue(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t stream, typename SameType<P>::type... args) {
    void* list[] = {static_cast<void*>(&args)...};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, list, 0, stream);
}

// ---- block-scaled linear ---------------------------------------------------------------------------------------
struct BlockLinear {
    const uint16_t* x;        // bf16 activations [M, ldx], or null when codes are given
    int64_t ldx;
    const uint8_t* xq;        // codes, rows of ldq bytes
    int64_t ldq;
    const float* xs;          // scale of row m, block g: xs[m * xs_row + g * xs_block]
    int64_t xs_row, xs_block;
    const uint8_t* w;         // [N, K] row-major codes
    const float* ws;          // [ceil(N / 128), ceil(K / 128)]
    const uint16_t* bias;     // [N] or null
    uint16_t* out;
    int64_t ldo;
    int M, N, K;
};
// Codes of x (rows of ldq bytes, zeros between K and ldq) and the scales.
hipError_t launch_block_quant(const uint16_t* x, int64_t ldx, int64_t M, int64_t K, uint8_t* xq, int64_t ldq, float* xs, int64_t xs_row,
                        int64_t xs_block, hipStream_t stream);
bool block_linear_small(int64_t M, int64_t N, int64_t K);         // one launch, rows quantized where they are multiplied
hipError_t launch_block_linear_small(const BlockLinear& p, hipStream_t stream);
hipError_t launch_block_gemm(const BlockLinear& p, hipStream_t stream);

// ---- head norms, rotation, cache write ---------------------------------------------------------------------------
enum HeadType : int { HEAD_BF16 = 0, HEAD_F16 = 1 };
struct HeadRope {
    const uint16_t* qkv;      // [T, (H + 2 KV) * D], row stride ld
    int64_t ld;
    const uint16_t *q_weight, *k_weight;   // [D] or null: no norm
    const float* cos_sin;     // [positions, rot]: cosines, then sines
    int64_t table_rows;
    const int64_t* positions; // [T]
    uint16_t* q_out;          // [T, H, D] dense
    uint16_t* k_out;          // [T, KV, D] dense, or null: into the cache
    void *k_pages, *v_pages;               // elements of the heads' type or, with scales, codes of e4m3
    int64_t k_stride[3], v_stride[3];      // elements between pages, tokens of a page, heads
    uint8_t *k_scales, *v_scales;          // pages in 8 bits: a byte b for each token and head, the power 2^(b - 127)
    int64_t k_scale_stride[3], v_scale_stride[3];
    const int64_t* slots;     // [T]: page * page_size + token, anything outside the cache: not written
    int64_t n_slots;
    int T, H, KV, D, rot, page_size;
    float eps;
    int gemma, interleaved, type;
};
hipError_t launch_head_rope(const HeadRope& p, hipStream_t stream);

// ---- attention over pages -----------------------------------------------------------------------------------------
struct PagedAttention {
    const uint16_t* q;        // [T, H, D]: strides of a token and of a head
    int64_t q_token, q_head;
    const void *k_pages, *v_pages;         // elements of q's type or, with scales, codes of e4m3
    int64_t kv_stride[3];     // elements between pages, tokens of a page, heads: of K and of V
    int64_t n_pages;
    const int32_t* table;     // [B, table_width], row stride table_ld
    int64_t table_ld;
    const int32_t* q_offsets; // [B + 1]
    const int32_t* kv_lens;   // [B]
    uint16_t* out;            // [T, H, D] dense
    float scale;
    int T, B, H, KV, D, page_size, table_width, causal, window, type;
    void* workspace;          // where split sums go, or null
    // what a plain call leaves at zero
    const uint8_t *k_scales, *v_scales;    // of pages in 8 bits: bytes b of powers 2^(b - 127)
    int64_t scale_stride[3];  // between pages, tokens of a page, heads
    const int32_t* prefix_lens;            // [B]: keys that a causal row sees whatever its position
    float cap, cap_by;        // scores become cap tanh: the cap times log2(e); 2 log2(e) scale / cap (above kWideCap: scale / cap)
    float cap_most;           // cap / scale
    int more;                 // not a plain call (also where everything below is zero)
    int shared;               // leading keys that lie in the same pages for all sequences, as the caller says
};
constexpr float kWideCap = 256.0f * 1.4426950408889634f;   // (as cap above)
// Division by a number known on the host: its magic number and shift (magic 0: by one).
struct AttentionDivision {
    uint32_t magic, shift;
};
// What the host works out once per call.
struct AttentionPlan {
    AttentionDivision page, group, workers;
    int group_size, tiles, splits, many;
    // leading keys computed once for all, with tiles of all sequences' rows together; of the splits the first ones are theirs
    int shared, shared_tiles, shared_splits, shared_many;
    AttentionDivision shared_workers;
    int small;                // few rows: half the wavefronts a workgroup
};
size_t paged_attention_workspace_bytes(int64_t T, int64_t B, int64_t H, int64_t KV, int64_t D, int64_t max_kv, int64_t shared, int64_t window,
                                       bool more);
hipError_t launch_paged_attention(const PagedAttention& p, hipStream_t stream);

// ---- residual, norm, quantizer ---------------------------------------------------------------------------------------
struct AddNorm {
    const uint16_t *x, *residual;          // bf16 [M, D], row strides ldx, ldr
    int64_t ldx, ldr;
    const uint16_t* weight;   // [D]
    uint16_t* total;          // bf16(x + residual), row stride ldt; may be x or residual
    int64_t ldt;
    uint8_t* xq;              // codes [M, D] dense
    float* scale;             // of row m, block g: scale[m * xs_row + g * xs_block]
    int64_t xs_row, xs_block;
    int64_t M;
    int D, gemma, per_block;
    float eps;
};
hipError_t launch_add_norm(const AddNorm& p, hipStream_t stream);

// ---- a cache in 8 bits, read back ------------------------------------------------------------------------------------
struct CacheRead {
    const uint8_t *k_pages, *v_pages;
    int64_t k_stride[3], v_stride[3];
    const uint8_t *k_scales, *v_scales;
    int64_t k_scale_stride[3], v_scale_stride[3];
    const int64_t* slots;     // [T]
    int64_t n_slots;
    uint16_t *k_out, *v_out;  // [T, KV, D] dense
    int T, KV, D, page_size, type;
};
hipError_t launch_cache_read(const CacheRead& p, hipStream_t stream);

}  // namespace phyai
