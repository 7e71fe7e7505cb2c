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
    uint16_t *k_pages, *v_pages;
    int64_t k_stride[3], v_stride[3];      // elements between pages, tokens of a page, heads
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
    const uint16_t *k_pages, *v_pages;
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
};
size_t paged_attention_workspace_bytes(int64_t T, int64_t B, int64_t H, int64_t KV, int64_t D, int64_t max_kv);
hipError_t launch_paged_attention(const PagedAttention& p, hipStream_t stream);

}  // namespace phyai
