// extern "C" boundary of include/phyai_layer.h: arguments are checked here, nothing is allocated, nothing synchronises.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "../../include/phyai_fp8.h"
#include "../../include/phyai_layer.h"
#include "layer_kernels.h"

namespace {

thread_local char g_error[256] = "";

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
    return code;
}
int launched(const char* fn, hipError_t e) {
    return e == hipSuccess ? PHYAI_FP8_OK : fail(PHYAI_FP8_ELAUNCH, "%s: %s", fn, hipGetErrorString(e));
}
bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

constexpr int64_t kMost = (int64_t)1 << 31;
constexpr int64_t kBlock = 128;
int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

// Workspace of a linear, behind the header: codes (rows padded to whole blocks), then scales, one row of them per block.
size_t codes_bytes(int64_t M, int64_t K) { return align_up((size_t)M * (size_t)(blocks_of(K) * kBlock), 256); }

int check_rows(const char* fn, const void* x, int64_t ldx, int64_t M, int64_t K) {
    if (M < 0 || K <= 0) return fail(PHYAI_FP8_EINVAL, "%s: bad shape M=%lld K=%lld", fn, (long long)M, (long long)K);
    if (M == 0) return 0;
    if (!x || !aligned(x, 16)) return fail(PHYAI_FP8_EINVAL, "%s: x must be a 16-byte aligned pointer", fn);
    if (K % 8 != 0) return fail(PHYAI_FP8_EUNSUPPORTED, "%s: K=%lld must be a multiple of 8", fn, (long long)K);
    if (ldx < K || ldx % 8 != 0) return fail(PHYAI_FP8_EINVAL, "%s: row stride %lld must be >= K and a multiple of 8", fn, (long long)ldx);
    if (M >= kMost || K >= kMost / 2 || M * (blocks_of(K) * kBlock) >= kMost)
        return fail(PHYAI_FP8_EUNSUPPORTED, "%s: more than 2^31 elements", fn);
    return 0;
}

int check_linear(const char* fn, const void* w, const float* w_scale, const void* bias, const void* out, int64_t ldo, int64_t M, int64_t N, int64_t K) {
    if (M < 0 || N <= 0 || K <= 0)
        return fail(PHYAI_FP8_EINVAL, "%s: bad shape M=%lld N=%lld K=%lld", fn, (long long)M, (long long)N, (long long)K);
    if (N % 16 != 0 || K % 16 != 0) return fail(PHYAI_FP8_EUNSUPPORTED, "%s: N=%lld and K=%lld must be multiples of 16", fn, (long long)N, (long long)K);
    if (M == 0) return 0;
    if (!w || !w_scale || !out) return fail(PHYAI_FP8_EINVAL, "%s: null pointer", fn);
    if (!aligned(w, 16) || !aligned(w_scale, 4) || !aligned(out, 8) || !aligned(bias, 2))
        return fail(PHYAI_FP8_EINVAL, "%s: w must be 16-byte, out 8-byte, w_scale 4-byte and bias 2-byte aligned", fn);
    if (ldo < N || ldo % 4 != 0) return fail(PHYAI_FP8_EINVAL, "%s: row stride %lld of out must be >= N and a multiple of 4", fn, (long long)ldo);
    if (M >= kMost || N >= kMost || K >= kMost || M * K >= kMost || N * K >= kMost)
        return fail(PHYAI_FP8_EUNSUPPORTED, "%s: operand of more than 2^31 elements", fn);
    return 0;
}

// Do M rows of `a` bytes from p, `lda` bytes apart, and M of `b` bytes from q share memory?  Rows of equal strides may lie beside each
// other in one buffer.
bool overlap(const void* p, int64_t lda, int64_t a, const void* q, int64_t ldb, int64_t b, int64_t M) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
    if (x + (uintptr_t)((M - 1) * lda + a) <= y || y + (uintptr_t)((M - 1) * ldb + b) <= x) return false;
    if (M == 1 || lda != ldb) return true;
    const int64_t off = y >= x ? (int64_t)((y - x) % (uintptr_t)lda) : lda - 1 - (int64_t)((x - y - 1) % (uintptr_t)lda);
    return off < a || off + b > lda;
}

}  // namespace

extern "C" {

int phyai_layer_abi_version(void) { return PHYAI_LAYER_ABI_VERSION; }

const char* phyai_layer_last_error(void) { return g_error; }

int phyai_layer_block_quant(const void* x, int64_t ldx, int64_t M, int64_t K, void* xq, float* x_scale, int64_t xs_row, int64_t xs_block,
                            void* stream) {
    const char* fn = "phyai_layer_block_quant";
    if (int rc = check_rows(fn, x, ldx, M, K)) return rc;
    if (M == 0) return PHYAI_FP8_OK;
    if (!xq || !x_scale || !aligned(xq, 8) || !aligned(x_scale, 4)) return fail(PHYAI_FP8_EINVAL, "%s: xq must be 8-byte and x_scale 4-byte aligned", fn);
    if (xs_row <= 0 || xs_block <= 0) return fail(PHYAI_FP8_EINVAL, "%s: strides of x_scale must be positive", fn);
    return launched(fn, phyai::launch_block_quant(static_cast<const uint16_t*>(x), ldx, M, K, static_cast<uint8_t*>(xq), K, x_scale, xs_row, xs_block,
                                                  static_cast<hipStream_t>(stream)));
}

int phyai_layer_block_gemm(const void* xq, const float* x_scale, int64_t xs_row, int64_t xs_block, const void* w, const float* w_scale,
                           const void* bias, void* out, int64_t ldo, int64_t M, int64_t N, int64_t K, void* stream) {
    const char* fn = "phyai_layer_block_gemm";
    if (int rc = check_linear(fn, w, w_scale, bias, out, ldo, M, N, K)) return rc;
    if (M == 0) return PHYAI_FP8_OK;
    if (!xq || !x_scale || !aligned(xq, 16) || !aligned(x_scale, 4)) return fail(PHYAI_FP8_EINVAL, "%s: xq must be 16-byte and x_scale 4-byte aligned", fn);
    if (xs_row < 0 || xs_block < 0 || xs_row >= kMost || xs_block >= kMost ||
        ((M - 1) * xs_row + (blocks_of(K) - 1) * xs_block + 1) * 4 >= kMost)
        return fail(PHYAI_FP8_EUNSUPPORTED, "%s: strides of x_scale must not be negative and reach less than 2^29 elements", fn);
    if (overlap(xq, K, K, out, ldo * 2, N * 2, M)) return fail(PHYAI_FP8_EINVAL, "%s: out overlaps xq", fn);
    phyai::BlockLinear p = {};
    p.xq = static_cast<const uint8_t*>(xq);
    p.ldq = K;
    p.xs = x_scale;
    p.xs_row = xs_row;
    p.xs_block = xs_block;
    p.w = static_cast<const uint8_t*>(w);
    p.ws = w_scale;
    p.bias = static_cast<const uint16_t*>(bias);
    p.out = static_cast<uint16_t*>(out);
    p.ldo = ldo;
    p.M = (int)M; p.N = (int)N; p.K = (int)K;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return launched(fn, phyai::block_linear_small(M, N, K) ? phyai::launch_block_linear_small(p, st) : phyai::launch_block_gemm(p, st));
}

size_t phyai_layer_block_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || M >= kMost || K >= kMost || phyai::block_linear_small(M, N, K)) return 0;
    return PHYAI_FP8_WORKSPACE_HEADER_BYTES + codes_bytes(M, K) + (size_t)M * (size_t)blocks_of(K) * sizeof(float);
}

int phyai_layer_block_linear(const void* x, int64_t ldx, const void* w, const float* w_scale, const void* bias, void* out, int64_t ldo,
                             int64_t M, int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
    const char* fn = "phyai_layer_block_linear";
    if (int rc = check_rows(fn, x, ldx, M, K)) return rc;
    if (int rc = check_linear(fn, w, w_scale, bias, out, ldo, M, N, K)) return rc;
    if (M == 0) return PHYAI_FP8_OK;
    phyai::BlockLinear p = {};
    p.w = static_cast<const uint8_t*>(w);
    p.ws = w_scale;
    p.bias = static_cast<const uint16_t*>(bias);
    p.out = static_cast<uint16_t*>(out);
    p.ldo = ldo;
    p.M = (int)M; p.N = (int)N; p.K = (int)K;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const uint16_t* rows = static_cast<const uint16_t*>(x);
    if (phyai::block_linear_small(M, N, K)) {
        if (overlap(x, ldx * 2, K * 2, out, ldo * 2, N * 2, M))
            return fail(PHYAI_FP8_EINVAL, "%s: out overlaps x, of whose few rows some are read while others are written", fn);
        p.x = rows;
        p.ldx = ldx;
        return launched(fn, phyai::launch_block_linear_small(p, st));
    }
    const size_t need = phyai_layer_block_linear_workspace_bytes(M, N, K);
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < need)
        return fail(PHYAI_FP8_EWORKSPACE, "%s: workspace of %zu bytes is missing, unaligned or smaller than %zu", fn, workspace ? workspace_bytes : (size_t)0, need);
    uint8_t* codes = static_cast<uint8_t*>(workspace) + PHYAI_FP8_WORKSPACE_HEADER_BYTES;
    float* scales = reinterpret_cast<float*>(codes + codes_bytes(M, K));
    p.xq = codes;
    p.ldq = blocks_of(K) * kBlock;
    p.xs = scales;
    p.xs_row = 1;
    p.xs_block = M;
    const hipError_t e = phyai::launch_block_quant(rows, ldx, M, K, codes, p.ldq, scales, p.xs_row, p.xs_block, st);
    return launched(fn, e != hipSuccess ? e : phyai::launch_block_gemm(p, st));
}

int phyai_layer_head_rope(const void* qkv, int64_t ld, const void* q_weight, const void* k_weight, const float* cos_sin, int64_t table_rows,
                          const int64_t* positions, void* q_out, void* k_out, void* k_pages, void* v_pages, const int64_t* k_strides,
                          const int64_t* v_strides, const int64_t* slots, int64_t n_pages, int64_t page_size, int64_t T, int64_t heads,
                          int64_t kv_heads, int64_t head_dim, int64_t rot, float eps, int gemma, int interleaved, int type, void* stream) {
    const char* fn = "phyai_layer_head_rope";
    if (T < 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || rot < 0 || rot > head_dim || heads > 65535 || kv_heads > 65535)
        return fail(PHYAI_FP8_EINVAL, "%s: bad shape T=%lld heads=%lld kv_heads=%lld head_dim=%lld rot=%lld", fn, (long long)T, (long long)heads,
                    (long long)kv_heads, (long long)head_dim, (long long)rot);
    if (head_dim % 8 != 0 || rot % 8 != 0 || head_dim > 512)
        return fail(PHYAI_FP8_EUNSUPPORTED, "%s: head_dim=%lld and rot=%lld must be multiples of 8, head_dim at most 512", fn, (long long)head_dim, (long long)rot);
    if (type != PHYAI_LAYER_BF16 && type != PHYAI_LAYER_F16) return fail(PHYAI_FP8_EINVAL, "%s: unknown type %d", fn, type);
    if ((q_weight == nullptr) != (k_weight == nullptr)) return fail(PHYAI_FP8_EINVAL, "%s: q_weight and k_weight go together", fn);
    if (k_out == nullptr && (!k_pages || !v_pages || !k_strides || !v_strides || !slots || n_pages < 0 || page_size <= 0))
        return fail(PHYAI_FP8_EINVAL, "%s: without k_out the pages, their strides and the slots are needed", fn);
    if (T == 0) return PHYAI_FP8_OK;
    if (!qkv || (rot > 0 && !cos_sin) || !positions || !q_out) return fail(PHYAI_FP8_EINVAL, "%s: null pointer", fn);
    if (table_rows <= 0) return fail(PHYAI_FP8_EINVAL, "%s: the table of angles is empty", fn);
    const int64_t width = (heads + 2 * kv_heads) * head_dim;
    if (T >= kMost || ld < width || ld % 8 != 0) return fail(PHYAI_FP8_EINVAL, "%s: row stride %lld must be at least %lld and a multiple of 8", fn, (long long)ld, (long long)width);
    if (!aligned(qkv, 16) || !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(cos_sin, 16) || !aligned(positions, 8) || !aligned(q_out, 16) ||
        !aligned(k_out, 16) || !aligned(slots, 8))
        return fail(PHYAI_FP8_EINVAL, "%s: operands must be 16-byte aligned (positions and slots 8-byte)", fn);
    phyai::HeadRope p = {};
    if (k_out == nullptr) {
        for (int i = 0; i < 3; ++i) {
            if (k_strides[i] < 0 || v_strides[i] < 0 || k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0)
                return fail(PHYAI_FP8_EINVAL, "%s: strides of the pages must be multiples of 8", fn);
            p.k_stride[i] = k_strides[i];
            p.v_stride[i] = v_strides[i];
        }
        if (!aligned(k_pages, 16) || !aligned(v_pages, 16)) return fail(PHYAI_FP8_EINVAL, "%s: pages must be 16-byte aligned", fn);
        if (page_size >= kMost || (n_pages > 0 && page_size > (kMost - 1) / n_pages))
            return fail(PHYAI_FP8_EUNSUPPORTED, "%s: a cache of 2^31 tokens or more", fn);
    }
    p.qkv = static_cast<const uint16_t*>(qkv);
    p.ld = ld;
    p.q_weight = static_cast<const uint16_t*>(q_weight);
    p.k_weight = static_cast<const uint16_t*>(k_weight);
    p.cos_sin = cos_sin;
    p.table_rows = table_rows;
    p.positions = positions;
    p.q_out = static_cast<uint16_t*>(q_out);
    p.k_out = static_cast<uint16_t*>(k_out);
    p.k_pages = static_cast<uint16_t*>(k_pages);
    p.v_pages = static_cast<uint16_t*>(v_pages);
    p.slots = slots;
    p.n_slots = k_out == nullptr ? n_pages * page_size : 0;
    p.T = (int)T; p.H = (int)heads; p.KV = (int)kv_heads; p.D = (int)head_dim; p.rot = (int)rot;
    p.page_size = k_out == nullptr ? (int)page_size : 1;
    p.eps = eps;
    p.gemma = gemma ? 1 : 0;
    p.interleaved = interleaved ? 1 : 0;
    p.type = type;
    return launched(fn, phyai::launch_head_rope(p, static_cast<hipStream_t>(stream)));
}

size_t phyai_layer_paged_attention_workspace_bytes(int64_t T, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_kv) {
    if (T <= 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || heads % kv_heads != 0 || T >= kMost || T * heads >= kMost) return 0;
    const size_t n = phyai::paged_attention_workspace_bytes(T, batch, heads, kv_heads, head_dim, max_kv);
    return n == 0 ? 0 : PHYAI_FP8_WORKSPACE_HEADER_BYTES + n;
}

int phyai_layer_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k_pages, const void* v_pages,
                                const int64_t* kv_strides, int64_t n_pages, int64_t page_size, const int32_t* page_table, int64_t table_stride,
                                int64_t table_width, const int32_t* q_offsets, const int32_t* kv_lens, void* out, int64_t T, int64_t batch,
                                int64_t heads, int64_t kv_heads, int64_t head_dim, float scale, int causal, int64_t window, int type,
                                void* workspace, size_t workspace_bytes, void* stream) {
    const char* fn = "phyai_layer_paged_attention";
    if (T < 0 || batch < 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || n_pages < 0 || page_size <= 0 || table_width < 0)
        return fail(PHYAI_FP8_EINVAL, "%s: bad shape T=%lld batch=%lld heads=%lld kv_heads=%lld head_dim=%lld page_size=%lld", fn, (long long)T,
                    (long long)batch, (long long)heads, (long long)kv_heads, (long long)head_dim, (long long)page_size);
    if (heads % kv_heads != 0) return fail(PHYAI_FP8_EINVAL, "%s: heads=%lld must be a multiple of kv_heads=%lld", fn, (long long)heads, (long long)kv_heads);
    if (head_dim % 8 != 0 || head_dim > 256) return fail(PHYAI_FP8_EUNSUPPORTED, "%s: head_dim=%lld must be a multiple of 8 up to 256", fn, (long long)head_dim);
    if (type != PHYAI_LAYER_BF16 && type != PHYAI_LAYER_F16) return fail(PHYAI_FP8_EINVAL, "%s: unknown type %d", fn, type);
    if (!(scale > 0.f) || isinf(scale * 1.4426950408889634f))   // (scores are taken to base 2)
        return fail(PHYAI_FP8_EINVAL, "%s: scale must be a positive number, and times log2(e) a finite one", fn);
    if (window < 0) return fail(PHYAI_FP8_EINVAL, "%s: window=%lld must not be negative", fn, (long long)window);
    if (T == 0 || batch == 0) return PHYAI_FP8_OK;
    if (!q || !out || !q_offsets || !kv_lens) return fail(PHYAI_FP8_EINVAL, "%s: null pointer", fn);
    if (!kv_strides || (n_pages > 0 && (!k_pages || !v_pages)) || (table_width > 0 && !page_table)) return fail(PHYAI_FP8_EINVAL, "%s: null pointer", fn);
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(page_table, 4) || !aligned(q_offsets, 4) || !aligned(kv_lens, 4))
        return fail(PHYAI_FP8_EINVAL, "%s: q, out and pages must be 16-byte aligned, the tables 4-byte", fn);
    if (q_token_stride < 0 || q_head_stride < 0 || q_token_stride % 8 != 0 || q_head_stride % 8 != 0)
        return fail(PHYAI_FP8_EINVAL, "%s: strides of q must be multiples of 8", fn);
    for (int i = 0; i < 3; ++i)
        if (kv_strides[i] < 0 || kv_strides[i] % 8 != 0) return fail(PHYAI_FP8_EINVAL, "%s: strides of the pages must be multiples of 8", fn);
    if (T >= kMost / 2 || heads >= kMost / 2 || T * heads >= kMost / 2 || batch >= kMost / 2 || n_pages >= kMost || kv_heads > 65535)
        return fail(PHYAI_FP8_EUNSUPPORTED, "%s: T * heads and batch must be below 2^30, n_pages below 2^31, kv_heads below 2^16", fn);
    if (table_width >= kMost / 4 || page_size >= kMost || (table_width > 0 && page_size > (kMost / 2 - 1) / table_width))
        return fail(PHYAI_FP8_EUNSUPPORTED, "%s: table width * page size must be below 2^30", fn);
    if (table_width > 0 && batch > 1 && table_stride != 0 && table_stride < table_width)
        return fail(PHYAI_FP8_EINVAL, "%s: row stride of the page table is smaller than its width", fn);
    if (kv_strides[1] >= (int64_t)1 << 28) return fail(PHYAI_FP8_EUNSUPPORTED, "%s: stride between a page's tokens of 2^28 or more", fn);
    const size_t need = phyai_layer_paged_attention_workspace_bytes(T, batch, heads, kv_heads, head_dim, table_width * page_size);
    if (need > 0 && (!workspace || !aligned(workspace, 256) || workspace_bytes < need))
        return fail(PHYAI_FP8_EWORKSPACE, "%s: workspace of %zu bytes is missing, unaligned or smaller than %zu", fn, workspace ? workspace_bytes : (size_t)0, need);
    phyai::PagedAttention p = {};
    p.q = static_cast<const uint16_t*>(q);
    p.q_token = q_token_stride;
    p.q_head = q_head_stride;
    p.k_pages = static_cast<const uint16_t*>(k_pages);
    p.v_pages = static_cast<const uint16_t*>(v_pages);
    for (int i = 0; i < 3; ++i) p.kv_stride[i] = kv_strides[i];
    p.n_pages = n_pages;
    p.table = page_table;
    p.table_ld = table_stride;
    p.q_offsets = q_offsets;
    p.kv_lens = kv_lens;
    p.out = static_cast<uint16_t*>(out);
    p.scale = scale;
    p.T = (int)T; p.B = (int)batch; p.H = (int)heads; p.KV = (int)kv_heads; p.D = (int)head_dim;
    p.page_size = (int)page_size; p.table_width = (int)table_width;
    p.causal = causal ? 1 : 0;
    p.window = window > kMost - 1 ? (int)(kMost - 1) : (int)window;
    p.type = type;
    p.workspace = need > 0 ? static_cast<uint8_t*>(workspace) + PHYAI_FP8_WORKSPACE_HEADER_BYTES : nullptr;
    return launched(fn, phyai::launch_paged_attention(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
