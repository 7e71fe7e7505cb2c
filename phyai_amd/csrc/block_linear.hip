// The W8A8 linear with a scale for each block of 128 (gfx950):
//
//     s[m, g]  = max(amax of the 128 values of block g of row m, 1e-12) / 448          (fp32, rounded division)
//     q[m, k]  = e4m3(x[m, k] / s[m, g])                                               (rounded quotient, nearest even)
//     y[m, n]  = bf16(sum_g s[m, g] * ws[n / 128, g] * (sum over block g of q[m, k] * w[n, k]) + bias[n])
//
// The inner sum of one block is exactly one v_mfma_f32_16x16x128 with C = 0; its result is scaled and added in fp32 with
// one fused multiply-add per value.  With the weights as operand A a lane ends up with four neighbouring columns of ONE
// token, so the scale is one product per 16 tokens and block, and the four values leave as one 8-byte store.
#include "fp8_device.h"
#include "layer_kernels.h"
#include "quant_device.h"
#include "tuning.h"

namespace phyai {
namespace {

constexpr int QB = 128;   // elements per scale
constexpr float kBlockAmaxFloor = 1e-12f;

// max over the lanes l, l ^ 16, l ^ 32, l ^ 48: the four lanes that hold one row of an MFMA operand.
__device__ __forceinline__ uint32_t quad_rows_max(uint32_t v) {
    auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = a[0] > a[1] ? a[0] : a[1];
    auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return b[0] > b[1] ? b[0] : b[1];
}

__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
    const float a = bf16_bits_to_f32(amax_bits);
    return (a < kBlockAmaxFloor ? kBlockAmaxFloor : a) / kFp8Max;   // (a NaN stays one)
}

// Codes of eight values.  Fast: the correctly rounded quotient in three instructions (quant_device.h); |x / s| is at most
// one step above 448, which rounds to 448.  A scale that is not finite, or out of that range, takes the division.
__device__ __forceinline__ uint2 block_encode8(uint4 q, const RowDivisor& d) {
    if (d.fast) return encode8<QUANT_WEIGHT>(q, d);
    return encode8<QUANT_ACT_DYNAMIC>(q, d);   // (d.fast is false: divides, NaN and Inf give NaN codes)
}

// ---- the quantizer on its own -----------------------------------------------------------------------------------
// Sixteen lanes a block, eight values (16 bytes) a lane; the block's maximum by four DPP steps inside the row of lanes.
// One pass over the data, bound by memory.
__global__ __launch_bounds__(256) void block_quant_kernel(const uint16_t* __restrict__ x, int64_t ldx, int K, int blocks, int64_t items,
                                                          uint8_t* __restrict__ xq, int64_t ldq, float* __restrict__ xs, int64_t xs_row,
                                                          int64_t xs_block) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t item = i >> 4;
    if (item >= items) return;   // (whole rows of 16 lanes leave together)
    const int c = (int)(i & 15);
    const int64_t m = item / blocks;
    const int g = (int)(item - m * blocks);
    const int k = g * QB + c * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (k < K) v = *reinterpret_cast<const uint4*>(x + m * ldx + k);
    uint32_t a = absmax8(v, 0u), o;
    o = dpp_move_u32<0xB1>(a);  a = o > a ? o : a;
    o = dpp_move_u32<0x4E>(a);  a = o > a ? o : a;
    o = dpp_move_u32<0x141>(a); a = o > a ? o : a;
    o = dpp_move_u32<0x140>(a); a = o > a ? o : a;
    const float s = block_scale(a);
    const RowDivisor d = make_divisor<QUANT_WEIGHT>(s);
    const uint2 codes = block_encode8(v, d);
    if (k < ldq) *reinterpret_cast<uint2*>(xq + m * ldq + k) = codes;
    if (c == 0) xs[m * xs_row + g * xs_block] = s;
}

// ---- few tokens: the weights streamed once ------------------------------------------------------------------------
// A workgroup owns 16 * NT weight rows and up to 16 * MB tokens; its wavefronts take the blocks of K in turn, each
// loads its weight block and the tokens' values straight into the MFMA's registers (lane q of a row: bytes 16 q and
// 64 + 16 q), quantizes the values there - the whole block of a row is in four lanes - and the partial sums meet in LDS,
// added in wavefront order.
constexpr int SMALL_WAVES = 8;

template <int MB, int NT, bool CODES>
__global__ __launch_bounds__(SMALL_WAVES * 64) void block_small_kernel(const BlockLinear p, int n_tiles) {
    __shared__ float sums[SMALL_WAVES][MB * NT][64][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
    const int m0 = blockIdx.y * (16 * MB), n0 = blockIdx.x * (16 * NT);
    const int blocks = (p.K + QB - 1) / QB;
    v4f acc[NT][MB];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[t][b] = v4f{0, 0, 0, 0};
    const uint8_t* wrow[NT];
    int nblk[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        int n = n0 + t * 16 + l16;
        n = n < p.N ? n : p.N - 1;
        wrow[t] = p.w + (size_t)n * p.K + q * 16;
        nblk[t] = __builtin_amdgcn_readfirstlane((n0 + t * 16 < p.N ? n0 + t * 16 : p.N - 1) / QB);
    }
    for (int g = wave; g < blocks; g += SMALL_WAVES) {
        const int k = g * QB;
        const bool lo = k + q * 16 < p.K, hi = k + 64 + q * 16 < p.K;
        v8i wf[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            v4i a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
            if (lo) a = *reinterpret_cast<const v4i*>(wrow[t] + k);
            if (hi) b = *reinterpret_cast<const v4i*>(wrow[t] + k + 64);
            wf[t] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            const int m = m0 + b * 16 + l16;
            const bool row = m < p.M;
            v8i xf;
            float s;
            if constexpr (CODES) {
                v4i a = {0, 0, 0, 0}, c = {0, 0, 0, 0};
                if (row && lo) a = *reinterpret_cast<const v4i*>(p.xq + m * p.ldq + k + q * 16);
                if (row && hi) c = *reinterpret_cast<const v4i*>(p.xq + m * p.ldq + k + 64 + q * 16);
                xf = __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7);
                s = row ? p.xs[m * p.xs_row + g * p.xs_block] : 0.f;
            } else {
                uint4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = make_uint4(0, 0, 0, 0);
                    if (row && (i < 2 ? lo : hi)) v[i] = *reinterpret_cast<const uint4*>(p.x + m * p.ldx + k + (i >> 1) * 64 + q * 16 + (i & 1) * 8);
                }
                uint32_t m2 = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) m2 = absmax8_pk(v[i], m2);
                s = block_scale(quad_rows_max(absmax_finish(m2)));
                const RowDivisor d = make_divisor<QUANT_WEIGHT>(s);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint2 c = block_encode8(v[i], d);
                    xf[2 * i] = (int)c.x;
                    xf[2 * i + 1] = (int)c.y;
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const v4f d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[t], xf, v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
                const float f = s * p.ws[(size_t)nblk[t] * blocks + g];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][b][e] = __builtin_fmaf(d[e], f, acc[t][b][e]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b) *reinterpret_cast<v4f*>(sums[wave][t * MB + b][lane]) = acc[t][b];
    __syncthreads();
    for (int tile = wave; tile < MB * NT; tile += SMALL_WAVES) {
        const int t = tile / MB, b = tile % MB;
        v4f y = *reinterpret_cast<const v4f*>(sums[0][tile][lane]);
#pragma unroll
        for (int w = 1; w < SMALL_WAVES; ++w) {
            const v4f o = *reinterpret_cast<const v4f*>(sums[w][tile][lane]);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += o[e];
        }
        const int m = m0 + b * 16 + l16, n = n0 + t * 16 + q * 4;
        if (m < p.M && n < p.N) {
            if (p.bias != nullptr) {
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] += bf16_bits_to_f32(p.bias[n + e]);
            }
            *reinterpret_cast<uint2*>(p.out + (size_t)m * p.ldo + n) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
        }
    }
}

// ---- many tokens: tiles through LDS -------------------------------------------------------------------------------
// Stage = one block of K (128 bytes a row) of the tile's tokens and weight rows and the tokens' scales of that block,
// copied straight into LDS; chunk c of row r lies in slot c ^ ((r >> 1) & 7), so the sixteen rows that a quarter of a
// wavefront reads together are in sixteen different bank groups.  Copies go through buffer resources: rows past the
// matrix repeat its last one, bytes past K arrive as zeros.
template <int TM, int TN, int WM, int WN, int DEPTH>
struct BlockTile {
    static constexpr int BM = 16 * TM * WM, BN = 16 * TN * WN, WAVES = WM * WN;
    static constexpr int STAGE = (BM + BN) * QB + (BM > 64 * WAVES ? BM : 64 * WAVES) * 4;
    static constexpr int CA = BM / 8 / WAVES, CB = BN / 8 / WAVES, CS = (BM + 64 * WAVES - 1) / (64 * WAVES);
    static constexpr int COPIES = CA + CB + CS;
    static constexpr int LDS = STAGE * DEPTH;
};

__device__ __forceinline__ uint32_t block_swizzle(int row) { return (uint32_t)(row >> 1) & 7u; }

template <int TM, int TN, int WM, int WN, int DEPTH>
__global__ __launch_bounds__(WM * WN * 64) void block_gemm_kernel(const BlockLinear p, int m_tiles, int n_tiles) {
    using T = BlockTile<TM, TN, WM, WN, DEPTH>;
    __shared__ __align__(16) uint8_t lds[T::LDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, q = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    const int bid = blockIdx.x;
    const int mt = bid % m_tiles, nt = bid / m_tiles;
    const int m0 = mt * T::BM, n0 = nt * T::BN;
    const int blocks = (p.K + QB - 1) / QB;

    uint32_t aoff[T::CA], boff[T::CB], soff[T::CS];
    uint32_t a_gone[2], b_gone[2];
    const int tail = p.K & (QB - 1);
#pragma unroll
    for (int i = 0; i < T::CA; ++i) {
        const int r = (wave * T::CA + i) * 8 + (lane >> 3);
        const int m = m0 + r < p.M ? m0 + r : p.M - 1;
        const uint32_t c = (uint32_t)(lane & 7) ^ block_swizzle(r);
        aoff[i] = (uint32_t)m * (uint32_t)p.ldq + c * 16;
        if (i < 2) a_gone[i] = tail != 0 && (int)(c * 16) >= tail ? kCopyNothing : 0u;
    }
#pragma unroll
    for (int i = 0; i < T::CB; ++i) {
        const int r = (wave * T::CB + i) * 8 + (lane >> 3);
        const int n = n0 + r < p.N ? n0 + r : p.N - 1;
        const uint32_t c = (uint32_t)(lane & 7) ^ block_swizzle(r);
        boff[i] = (uint32_t)n * (uint32_t)p.K + c * 16;
        if (i < 2) b_gone[i] = tail != 0 && (int)(c * 16) >= tail ? kCopyNothing : 0u;
    }
#pragma unroll
    for (int i = 0; i < T::CS; ++i) {
        const int r = (i * T::WAVES + wave) * 64 + lane;
        const int m = r < T::BM && m0 + r < p.M ? m0 + r : p.M - 1;
        soff[i] = (uint32_t)m * (uint32_t)p.xs_row * 4u;
    }
    static_assert(T::CA % 2 == 0 || T::CA == 1, "the swizzle repeats every two groups of eight rows");
    const v4i a_src = copy_source(p.xq, (uint32_t)((int64_t)(p.M - 1) * p.ldq + p.K));
    const v4i b_src = copy_source(p.w, (uint32_t)p.N * (uint32_t)p.K);
    const v4i s_src = copy_source(reinterpret_cast<const uint8_t*>(p.xs), (uint32_t)(((int64_t)(p.M - 1) * p.xs_row + (int64_t)(blocks - 1) * p.xs_block + 1) * 4));
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    auto issue = [&](int d) {
        const uint32_t at = base + (uint32_t)(d % DEPTH) * T::STAGE;
        const uint32_t last = d == blocks - 1 ? ~0u : 0u;
        const uint32_t k = (uint32_t)d * QB;
#pragma unroll
        for (int i = 0; i < T::CA; ++i)
            copy16_to_lds_checked(a_src, aoff[i] | (a_gone[i & 1] & last), k, __builtin_amdgcn_readfirstlane(at + (wave * T::CA + i) * 1024));
#pragma unroll
        for (int i = 0; i < T::CB; ++i)
            copy16_to_lds_checked(b_src, boff[i] | (b_gone[i & 1] & last), k, __builtin_amdgcn_readfirstlane(at + T::BM * QB + (wave * T::CB + i) * 1024));
#pragma unroll
        for (int i = 0; i < T::CS; ++i)
            asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds"
                         :: "v"(soff[i]), "s"(s_src), "s"((uint32_t)d * (uint32_t)p.xs_block * 4u),
                            "s"(__builtin_amdgcn_readfirstlane(at + (T::BM + T::BN) * QB + (i * T::WAVES + wave) * 256)) : "memory", "m0");
    };
    v4f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = v4f{0, 0, 0, 0};

    static_assert(QB % (16 * TN) == 0, "a wavefront's columns lie in one block of weight scales");
    int nb = (n0 + wn * 16 * TN) / QB;
    const int n_blocks = (p.N + QB - 1) / QB;
    nb = nb < n_blocks ? nb : n_blocks - 1;
    const float* wsrow = p.ws + (size_t)nb * blocks;
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d)
        if (d < blocks) issue(d);
    for (int d = 0; d < blocks; ++d) {
        // stage d is complete (this wavefront's copies by the wait, the others' by the barrier) and stage d - 1 has been read
        if (DEPTH > 2 && d + DEPTH - 2 < blocks) wait_copies<(DEPTH - 2) * T::COPIES>();
        else wait_copies<0>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (d + DEPTH - 1 < blocks) issue(d + DEPTH - 1);
        const uint8_t* stage = lds + (d % DEPTH) * T::STAGE;
        const uint8_t* wbuf = stage + T::BM * QB;
        const float* sbuf = reinterpret_cast<const float*>(stage + (T::BM + T::BN) * QB);
        const float wscale = wsrow[d];
        v8i wf[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int r = (wn * TN + j) * 16 + l16;
            const uint32_t z = block_swizzle(r);
            const v4i a = *reinterpret_cast<const v4i*>(wbuf + r * QB + (((uint32_t)q ^ z) << 4));
            const v4i b = *reinterpret_cast<const v4i*>(wbuf + r * QB + (((uint32_t)(q + 4) ^ z) << 4));
            wf[j] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int r = (wm * TM + i) * 16 + l16;
            const uint32_t z = block_swizzle(r);
            const v4i a = *reinterpret_cast<const v4i*>(stage + r * QB + (((uint32_t)q ^ z) << 4));
            const v4i b = *reinterpret_cast<const v4i*>(stage + r * QB + (((uint32_t)(q + 4) ^ z) << 4));
            const v8i xf = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
            const float f = sbuf[r] * wscale;
            v4f t[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) t[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], xf, v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(t[j][e], f, acc[i][j][e]);
        }
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int n = n0 + (wn * TN + j) * 16 + q * 4;
        if (n >= p.N) continue;
        float b[4] = {0, 0, 0, 0};
        if (p.bias != nullptr) {
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = bf16_bits_to_f32(p.bias[n + e]);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int m = m0 + (wm * TM + i) * 16 + l16;
            if (m >= p.M) continue;
            const v4f y = acc[i][j];
            *reinterpret_cast<uint2*>(p.out + (size_t)m * p.ldo + n) = make_uint2(pack_bf16x2(y[0] + b[0], y[1] + b[1]), pack_bf16x2(y[2] + b[2], y[3] + b[3]));
        }
    }
}

template <int TM, int TN, int WM, int WN, int DEPTH>
hipError_t launch_tile(const BlockLinear& p, hipStream_t stream) {
    using T = BlockTile<TM, TN, WM, WN, DEPTH>;
    const int mt = (p.M + T::BM - 1) / T::BM, nt = (p.N + T::BN - 1) / T::BN;
    return enqueue(block_gemm_kernel<TM, TN, WM, WN, DEPTH>, dim3((uint32_t)mt * nt), dim3(T::WAVES * 64), stream, p, mt, nt);
}

template <int MB, bool CODES>
hipError_t launch_small(const BlockLinear& p, hipStream_t stream) {
    const int nt = (p.N + 15) / 16;
    return enqueue(block_small_kernel<MB, 1, CODES>, dim3((uint32_t)nt, (uint32_t)((p.M + 16 * MB - 1) / (16 * MB))), dim3(SMALL_WAVES * 64), stream, p, nt);
}

}  // namespace

hipError_t launch_block_quant(const uint16_t* x, int64_t ldx, int64_t M, int64_t K, uint8_t* xq, int64_t ldq, float* xs, int64_t xs_row,
                        int64_t xs_block, hipStream_t stream) {
    const int blocks = (int)((K + QB - 1) / QB);
    const int64_t items = M * blocks;
    return enqueue(block_quant_kernel, dim3((uint32_t)((items + 15) / 16)), dim3(256), stream, x, ldx, (int)K, blocks, items, xq, ldq, xs,
                       xs_row, xs_block);
}

bool block_linear_small(int64_t M, int64_t, int64_t) {
    const char* forced = tuning_env("PHYAI_LAYER_BLOCK");   // 0: few tokens; 1, 2, 3: tiles of 256, 128, 64
    return forced != nullptr ? atoi(forced) == 0 : M <= 64;
}

hipError_t launch_block_linear_small(const BlockLinear& p, hipStream_t stream) {
    const bool codes = p.x == nullptr;
    if (p.M <= 16) return codes ? launch_small<1, true>(p, stream) : launch_small<1, false>(p, stream);
    if (p.M <= 32) return codes ? launch_small<2, true>(p, stream) : launch_small<2, false>(p, stream);
    return codes ? launch_small<4, true>(p, stream) : launch_small<4, false>(p, stream);
}

hipError_t launch_block_gemm(const BlockLinear& p, hipStream_t stream) {
    const int64_t big = (int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256);
    const int64_t mid = (int64_t)((p.M + 127) / 128) * ((p.N + 127) / 128);
    const char* forced = tuning_env("PHYAI_LAYER_BLOCK");
    const int shape = forced != nullptr ? atoi(forced) : big >= 256 ? 1 : mid >= 256 ? 2 : 3;
    if (shape == 1) return launch_tile<8, 4, 2, 4, 2>(p, stream);
    if (shape == 2) return launch_tile<4, 4, 2, 2, 2>(p, stream);
    return launch_tile<2, 2, 2, 2, 4>(p, stream);
}

}  // namespace phyai
