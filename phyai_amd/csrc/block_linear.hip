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

// Codes of a block's values, N of them in `v` of this lane: the correctly rounded quotient by three instructions
// (quant_device.h), for scales below 2^60; |x / s| is at most one step above 448, which rounds to 448.  A block whose
// scale is not of that kind is first brought there: a large one with its values by 2^-64 (what underflows has the code
// zero anyway), one with an infinity by zero - which leaves zeros, and NaN for the infinities - and one with a NaN by NaN.
template <int N>
__device__ __forceinline__ void block_encode(uint4 (&v)[N], float s, uint2 (&codes)[N]) {
    const bool plain = s < 1.152921504606846976e18f;
    if (__any(!plain)) {
        const bool finite = s < __builtin_huge_valf();
        const float by = plain ? 1.0f : finite ? 5.421010862427522e-20f : s != s ? s : 0.0f;
        s = plain || finite ? s * by : 1.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(__uint_as_float(w[j] << 16) * by, __uint_as_float(w[j] & 0xFFFF0000u) * by);
            v[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    RowDivisor d;
    d.s = s;
    d.r = 1.0f / s;
    d.fast = true;
#pragma unroll
    for (int i = 0; i < N; ++i) codes[i] = encode8<QUANT_WEIGHT>(v[i], d);
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
    uint4 v[1] = {make_uint4(0, 0, 0, 0)};
    if (k < K) v[0] = *reinterpret_cast<const uint4*>(x + m * ldx + k);
    uint32_t a = absmax8(v[0], 0u), o;
    o = dpp_move_u32<0xB1>(a);  a = o > a ? o : a;
    o = dpp_move_u32<0x4E>(a);  a = o > a ? o : a;
    o = dpp_move_u32<0x141>(a); a = o > a ? o : a;
    o = dpp_move_u32<0x140>(a); a = o > a ? o : a;
    const float s = block_scale(a);
    uint2 codes[1];
    block_encode(v, s, codes);
    if (k < ldq) *reinterpret_cast<uint2*>(xq + m * ldq + k) = codes[0];
    if (c == 0) xs[m * xs_row + g * xs_block] = s;
}

// ---- few tokens: the weights streamed once ------------------------------------------------------------------------
// A workgroup owns 16 * NT weight rows and 16 * MB tokens; its wavefronts take the blocks of K in turn, each loads its
// weight block and the tokens' values straight into the MFMA's registers (lane q of a row: bytes 16 q and 64 + 16 q),
// DEPTH blocks ahead, quantizes the values there - the whole block of a row is in four lanes - and the partial sums meet in
// LDS, added in wavefront order.
constexpr int SMALL_WAVES = 8;

template <int MB, int NT, int DEPTH, bool CODES>
__global__ __launch_bounds__(SMALL_WAVES * 64) void block_small_kernel(const BlockLinear p) {
    __shared__ float sums[SMALL_WAVES][MB * NT][64][4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, q = lane >> 4;
    const int m0 = blockIdx.y * (16 * MB), n0 = blockIdx.x * (16 * NT);
    const int blocks = (p.K + QB - 1) / QB;
    struct Stage {
        v4i w[NT][2];
        uint4 x[MB][CODES ? 2 : 4];
        float s[MB], ws[NT];
    } stage[DEPTH];
    v4f acc[NT][MB];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[t][b] = v4f{0, 0, 0, 0};
    const uint8_t* wrow[NT];
    const float* wsrow[NT];
    const uint8_t* xrow[MB];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int n = n0 + t * 16 + l16, first = n0 + t * 16 < p.N ? n0 + t * 16 : p.N - 1;
        wrow[t] = p.w + (size_t)(n < p.N ? n : p.N - 1) * p.K + q * 16;
        wsrow[t] = p.ws + (size_t)(first / QB) * blocks;
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        const int m = m0 + b * 16 + l16;
        const int64_t row = m < p.M ? m : p.M - 1;   // (rows past the last repeat it; nobody stores their sums)
        xrow[b] = CODES ? p.xq + row * p.ldq + q * 16 : reinterpret_cast<const uint8_t*>(p.x + row * p.ldx + q * 16);
    }
    auto load = [&](int g, Stage& o) {
        const int k = g * QB;
        const bool lo = k + q * 16 < p.K, hi = k + 64 + q * 16 < p.K;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            o.w[t][0] = lo ? *reinterpret_cast<const v4i*>(wrow[t] + k) : v4i{0, 0, 0, 0};
            o.w[t][1] = hi ? *reinterpret_cast<const v4i*>(wrow[t] + k + 64) : v4i{0, 0, 0, 0};
            o.ws[t] = wsrow[t][g];
        }
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            if constexpr (CODES) {
                o.x[b][0] = lo ? *reinterpret_cast<const uint4*>(xrow[b] + k) : make_uint4(0, 0, 0, 0);
                o.x[b][1] = hi ? *reinterpret_cast<const uint4*>(xrow[b] + k + 64) : make_uint4(0, 0, 0, 0);
                const int m = m0 + b * 16 + l16;
                o.s[b] = p.xs[(m < p.M ? m : p.M - 1) * p.xs_row + g * p.xs_block];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o.x[b][i] = (i < 2 ? lo : hi) ? *reinterpret_cast<const uint4*>(xrow[b] + 2 * k + (i >> 1) * 128 + (i & 1) * 16) : make_uint4(0, 0, 0, 0);
            }
        }
    };
    auto multiply = [&](Stage& o) {
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            v8i xf;
            float s;
            if constexpr (CODES) {
                xf = __builtin_shufflevector(__builtin_bit_cast(v4i, o.x[b][0]), __builtin_bit_cast(v4i, o.x[b][1]), 0, 1, 2, 3, 4, 5, 6, 7);
                s = o.s[b];
            } else {
                uint32_t m2 = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) m2 = absmax8_pk(o.x[b][i], m2);
                s = block_scale(quad_rows_max(absmax_finish(m2)));
                uint2 c[4];
                block_encode(o.x[b], s, c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    xf[2 * i] = (int)c[i].x;
                    xf[2 * i + 1] = (int)c[i].y;
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const v8i wf = __builtin_shufflevector(o.w[t][0], o.w[t][1], 0, 1, 2, 3, 4, 5, 6, 7);
                const v4f d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
                const float f = s * o.ws[t];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][b][e] = __builtin_fmaf(d[e], f, acc[t][b][e]);
            }
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (wave + d * SMALL_WAVES < blocks) load(wave + d * SMALL_WAVES, stage[d]);
    for (int g = wave; g < blocks; g += DEPTH * SMALL_WAVES) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int now = g + d * SMALL_WAVES, next = now + DEPTH * SMALL_WAVES;
            if (now < blocks) multiply(stage[d]);
            if (next < blocks) load(next, stage[d]);
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
    static constexpr int GA = BM / 8, GB = BN / 8, GS = (BM + 63) / 64 + 1;   // copies of a stage: eight rows; 64 scales, of the columns last
    static constexpr int STAGE = (BM + BN) * QB + GS * 256;
    static constexpr int EACH = (GA + GB + WAVES - 1) / WAVES, EACH_S = (GS + WAVES - 1) / WAVES;   // of a wavefront, at most
    static constexpr int LEAST = (GA + GB) / WAVES;                                                // and at least
    static constexpr int LDS = STAGE * DEPTH;
};

__device__ __forceinline__ uint32_t block_swizzle(int row) { return (uint32_t)(row >> 1) & 7u; }

template <int TM, int TN, int WM, int WN, int DEPTH>
__global__ __launch_bounds__(WM * WN * 64) void block_gemm_kernel(const BlockLinear p, int m_tiles, int n_tiles, int band, int per_xcd) {
    using T = BlockTile<TM, TN, WM, WN, DEPTH>;
    __shared__ __align__(16) uint8_t lds[T::LDS];
    // Workgroup i runs on XCD i % 8: each takes a run of the tiles, in bands of `band` tile rows, column after column
    int tile = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per_xcd || tile >= m_tiles * n_tiles) return;
    const int of_band = tile / (band * n_tiles), in_band = tile - of_band * band * n_tiles;
    const int rows_here = m_tiles - of_band * band < band ? m_tiles - of_band * band : band;
    const int nt = in_band / rows_here, mt = of_band * band + in_band - nt * rows_here;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, q = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    const int m0 = mt * T::BM, n0 = nt * T::BN;
    const int blocks = (p.K + QB - 1) / QB;

    // A wavefront's copies of a stage are those numbered wave, wave + WAVES, ...: token rows, weight rows, scales
    const int lr = lane >> 3;
    const uint32_t chunk = ((uint32_t)(lane & 7) ^ block_swizzle((wave & 1) * 8 + lr)) * 16;   // (WAVES is even: one parity of eight-row groups)
    const int tail = p.K & (QB - 1);
    const uint32_t gone = tail != 0 && (int)chunk >= tail ? kCopyNothing : 0u;
    uint32_t off[T::EACH], soff[T::EACH_S], sstep[T::EACH_S];
#pragma unroll
    for (int i = 0; i < T::EACH; ++i) {
        const int c = wave + i * T::WAVES;
        const int m = m0 + c * 8 + lr, n = n0 + (c - T::GA) * 8 + lr;
        off[i] = c < T::GA ? (uint32_t)(m < p.M ? m : p.M - 1) * (uint32_t)p.ldq + chunk : (uint32_t)(n < p.N ? n : p.N - 1) * (uint32_t)p.K + chunk;
    }
    static_assert(T::WAVES % 2 == 0 && T::GA % 2 == 0 && T::GB % 2 == 0, "the swizzle repeats every two groups of eight rows");
    const int n_blocks = (p.N + QB - 1) / QB;
    const v4i a_src = copy_source(p.xq, (uint32_t)((int64_t)(p.M - 1) * p.ldq + p.K));
    const v4i b_src = copy_source(p.w, (uint32_t)p.N * (uint32_t)p.K);
    const v4i s_src = copy_source(reinterpret_cast<const uint8_t*>(p.xs), (uint32_t)(((int64_t)(p.M - 1) * p.xs_row + (int64_t)(blocks - 1) * p.xs_block + 1) * 4));
    const v4i ws_src = copy_source(reinterpret_cast<const uint8_t*>(p.ws), (uint32_t)n_blocks * (uint32_t)blocks * 4u);
#pragma unroll
    for (int i = 0; i < T::EACH_S; ++i) {
        const int c = wave + i * T::WAVES, m = m0 + c * 64 + lane, nb = n0 / QB + lane;
        soff[i] = c < T::GS - 1 ? (uint32_t)(m < p.M ? m : p.M - 1) * (uint32_t)p.xs_row * 4u : (uint32_t)(nb < n_blocks ? nb : n_blocks - 1) * (uint32_t)blocks * 4u;
        sstep[i] = c < T::GS - 1 ? (uint32_t)p.xs_block * 4u : 4u;
    }
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    auto issue = [&](int d) {
        const uint32_t at = base + (uint32_t)(d % DEPTH) * T::STAGE;
        const uint32_t drop = d == blocks - 1 ? gone : 0u, k = (uint32_t)d * QB;
#pragma unroll
        for (int i = 0; i < T::EACH_S; ++i) {
            const int c = wave + i * T::WAVES;
            if (c >= T::GS) continue;
            const uint32_t to = __builtin_amdgcn_readfirstlane(at + (T::GA + T::GB) * 1024 + c * 256);
            asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds"
                         :: "v"(soff[i]), "s"(c < T::GS - 1 ? s_src : ws_src), "s"((uint32_t)d * __builtin_amdgcn_readfirstlane(sstep[i])), "s"(to) : "memory", "m0");
        }
#pragma unroll
        for (int i = 0; i < T::EACH; ++i) {
            const int c = wave + i * T::WAVES;
            if ((i + 1) * T::WAVES > T::GA + T::GB && c >= T::GA + T::GB) continue;
            const v4i src = (i + 1) * T::WAVES <= T::GA ? a_src : i * T::WAVES >= T::GA ? b_src : c < T::GA ? a_src : b_src;
            copy16_to_lds_checked(src, off[i] | drop, k, __builtin_amdgcn_readfirstlane(at + c * 1024));
        }
    };
    v4f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = v4f{0, 0, 0, 0};

    static_assert(QB % (16 * TN) == 0 && (T::BN % QB == 0 || QB % T::BN == 0), "a wavefront's columns lie in one block of weight scales");
    // fragments: row l16 of a block of 16, chunks q and q + 4; (every block of 16 rows has the same swizzle)
    const uint32_t f0 = (uint32_t)l16 * QB + (((uint32_t)q ^ block_swizzle(l16)) << 4);
    auto fragment = [&](const uint8_t* rows) -> v8i {
        const v4i a = *reinterpret_cast<const v4i*>(rows + f0), b = *reinterpret_cast<const v4i*>(rows + (f0 ^ 64u));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    };
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d)
        if (d < blocks) issue(d);
    for (int d = 0; d < blocks; ++d) {
        // stage d is complete (this wavefront's copies by the wait, the others' by the barrier) and stage d - 1 has been read
        if (DEPTH > 2 && d + DEPTH - 2 < blocks) wait_copies<(DEPTH - 2) * T::LEAST>();   // (some wavefronts have more in flight, and wait for a few too many)
        else wait_copies<0>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (d + DEPTH - 1 < blocks) issue(d + DEPTH - 1);
        const uint8_t* stage = lds + (d % DEPTH) * T::STAGE;
        const uint8_t *xbuf = stage + wm * TM * 16 * QB, *wbuf = stage + (T::BM + wn * TN * 16) * QB;
        const float* sbuf = reinterpret_cast<const float*>(stage + (T::BM + T::BN) * QB) + wm * TM * 16 + l16;
        const float wscale = reinterpret_cast<const float*>(stage + (T::BM + T::BN) * QB)[(T::GS - 1) * 64 + wn * 16 * TN / QB];
        v8i wf[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) wf[j] = fragment(wbuf + j * 16 * QB);
        // the products of row block i run while those of i - 1 are scaled and added
        v4f t[2][TN];
        v8i xf = fragment(xbuf);
        float f[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) f[i] = sbuf[i * 16] * wscale;
#pragma unroll
        for (int i = 0; i <= TM; ++i) {
            if (i < TM) {
                const v8i x = xf;
                if (i + 1 < TM) xf = fragment(xbuf + (i + 1) * 16 * QB);
#pragma unroll
                for (int j = 0; j < TN; ++j) t[i & 1][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], x, v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
            }
            if (i > 0) {
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i - 1][j][e] = __builtin_fmaf(t[(i - 1) & 1][j][e], f[i - 1], acc[i - 1][j][e]);
            }
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
    const int per = (mt * nt + 7) / 8, band = 1024 / T::BM;
    return enqueue(block_gemm_kernel<TM, TN, WM, WN, DEPTH>, dim3((uint32_t)per * 8), dim3(T::WAVES * 64), stream, p, mt, nt, band, per);
}

template <int MB, int NT, int DEPTH>
hipError_t launch_small(const BlockLinear& p, hipStream_t stream) {
    const dim3 grid((uint32_t)((p.N + 16 * NT - 1) / (16 * NT)), (uint32_t)((p.M + 16 * MB - 1) / (16 * MB)));
    return p.x == nullptr ? enqueue(block_small_kernel<MB, NT, DEPTH, true>, grid, dim3(SMALL_WAVES * 64), stream, p)
                          : enqueue(block_small_kernel<MB, NT, DEPTH, false>, grid, dim3(SMALL_WAVES * 64), stream, p);
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
    const char* forced = tuning_env("PHYAI_LAYER_BLOCK");   // 0: few tokens; 14 .. 18, 2, 3: tiles of 128 .. 256 x 256, 128, 64
    return forced != nullptr ? atoi(forced) == 0 : M <= 64;
}

hipError_t launch_block_linear_small(const BlockLinear& p, hipStream_t stream) {
    const int rows = (p.M + 15) / 16, cols = (p.N + 15) / 16;
    int mb = 1, nt = 1;
    while (mb < 4 && mb < rows && cols * ((rows + 2 * mb - 1) / (2 * mb)) >= 256) mb *= 2;
    if ((cols + 1) / 2 * ((rows + mb - 1) / mb) >= 512) nt = 2;
    if (const char* forced = tuning_env("PHYAI_LAYER_SMALL")) {   // 10 * token blocks + weight tiles of a workgroup
        mb = atoi(forced) / 10;
        nt = atoi(forced) % 10;
    }
    if (mb == 1) return nt == 1 ? launch_small<1, 1, 4>(p, stream) : launch_small<1, 2, 4>(p, stream);
    if (mb == 2) return nt == 1 ? launch_small<2, 1, 2>(p, stream) : launch_small<2, 2, 2>(p, stream);
    return nt == 1 ? launch_small<4, 1, 2>(p, stream) : launch_small<4, 2, 2>(p, stream);
}

hipError_t launch_block_gemm(const BlockLinear& p, hipStream_t stream) {
    const char* forced = tuning_env("PHYAI_LAYER_BLOCK");
    const int64_t mid = (int64_t)((p.M + 127) / 128) * ((p.N + 127) / 128);
    int shape;
    if (forced != nullptr) shape = atoi(forced);
    else if (mid >= 512) {
        // 256 columns, 128 to 256 rows: rounds of 256 workgroups, each a step longer than its row blocks
        int64_t best = INT64_MAX;
        shape = 1;
        for (int tm = 8; tm >= 4; --tm) {
            const int64_t tiles = (int64_t)((p.M + 32 * tm - 1) / (32 * tm)) * ((p.N + 255) / 256), cost = (tiles + 255) / 256 * (tm + 1);
            if (cost < best) {
                best = cost;
                shape = 10 + tm;
            }
        }
    } else shape = mid >= 200 ? 2 : 3;
    switch (shape) {
        case 14: return launch_tile<4, 4, 2, 4, 2>(p, stream);
        case 15: return launch_tile<5, 4, 2, 4, 2>(p, stream);
        case 16: return launch_tile<6, 4, 2, 4, 2>(p, stream);
        case 17: return launch_tile<7, 4, 2, 4, 2>(p, stream);
        case 1:
        case 18: return launch_tile<8, 4, 2, 4, 2>(p, stream);
        case 2: return launch_tile<4, 4, 2, 2, 2>(p, stream);
        default: return launch_tile<2, 2, 2, 2, 4>(p, stream);
    }
}

}  // namespace phyai
