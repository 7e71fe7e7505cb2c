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

__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
    const float a = bf16_max_to_f32(amax_bits);
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
// One pass over the data, bound by memory: 13056 x 16384 in 111 to 121 us, 5.3 to 5.8 TB/s of reads and writes.
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

// ---- a token or a few: the weights streamed once ------------------------------------------------------------------------
// A workgroup owns 16 * NT weight rows and all tokens, up to eight.  It quantizes its tokens' values into LDS, a stretch of K
// at a time (sixteen lanes a block of a row, as above), while the first weights are on their way; then its wavefronts take
// the blocks of K in turn, each with its weights straight from memory in the MFMA's registers (lane q of a row: bytes
// 16 q and 64 + 16 q), DEPTH blocks ahead.  The partial sums meet in LDS, added in wavefront order.  1 x 2560 x 1024: 3.5 us
// in a graph, the launch and two trips to memory; 2 x 22656 x 5632: 36.5 us, 3.5 TB/s of weights.
constexpr int FEW_WAVES = 8;

template <int NT>
struct FewShape {
    static constexpr int ROWS = 8, BLOCKS = 32;                     // of K in LDS at a time
    static constexpr int ROW = BLOCKS * QB + QB;               // bytes between rows: an odd number of lines, for the banks
    static constexpr int SCALES_AT = ROWS * ROW, CODES = SCALES_AT + ROWS * BLOCKS * 4, SUMS = FEW_WAVES * NT * 1024;
    static constexpr int LDS = CODES > SUMS ? CODES : SUMS;
};

template <int NT, int DEPTH, bool CODES>
__global__ __launch_bounds__(FEW_WAVES * 64) void block_few_kernel(const BlockLinear p) {
    using S = FewShape<NT>;
    __shared__ __align__(16) uint8_t lds[S::LDS];
    float* const scales = reinterpret_cast<float*>(lds + S::SCALES_AT);   // [block][token]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * (16 * NT), rows = p.M;
    const int blocks = (p.K + QB - 1) / QB;
    struct Stage {
        v4i w[NT][2];
        float ws[NT];
    } stage[DEPTH];
    const uint8_t* wrow[NT];
    const float* wsrow[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int n = n0 + t * 16 + l16, first = n0 + t * 16 < p.N ? n0 + t * 16 : p.N - 1;
        wrow[t] = p.w + (size_t)(n < p.N ? n : p.N - 1) * p.K + q * 16;
        wsrow[t] = p.ws + (size_t)(first / QB) * blocks;
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
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (wave + d * FEW_WAVES < blocks) load(wave + d * FEW_WAVES, stage[d]);

    v4f acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = v4f{0, 0, 0, 0};
    const int xrow = l16 < S::ROWS ? l16 : 0;   // (columns of the products past the last token are nobody's)
    static_assert(S::BLOCKS % (FEW_WAVES) == 0, "a stretch is whole turns of the wavefronts");
    for (int first = 0; first < blocks; first += S::BLOCKS) {
        const int here = blocks - first < S::BLOCKS ? blocks - first : S::BLOCKS;
        if (first > 0) __syncthreads();   // (the stretch before has been read)
        // codes of `rows` tokens and `here` blocks, four of them per sixteen lanes in flight
        const int c = threadIdx.x & 15;
        for (int item = threadIdx.x >> 4; item < rows * here; item += 4 * FEW_WAVES * 4) {
            int r[4], g[4];
            uint4 v[4];
            uint2 e[4];
            float s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int it = item + i * 4 * FEW_WAVES;
                r[i] = it < rows * here ? (int)((uint32_t)it / (uint32_t)here) : 0;
                g[i] = it < rows * here ? it - r[i] * here : 0;
                const int k = (first + g[i]) * QB + c * 8;
                if constexpr (CODES) {
                    e[i] = k < p.K ? *reinterpret_cast<const uint2*>(p.xq + (int64_t)r[i] * p.ldq + k) : make_uint2(0, 0);
                    s[i] = p.xs[(int64_t)r[i] * p.xs_row + (first + g[i]) * p.xs_block];
                } else {
                    v[i] = k < p.K ? *reinterpret_cast<const uint4*>(p.x + (int64_t)r[i] * p.ldx + k) : make_uint4(0, 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (!CODES) {
                    uint32_t a = absmax8(v[i], 0u), o;
                    o = dpp_move_u32<0xB1>(a);  a = o > a ? o : a;
                    o = dpp_move_u32<0x4E>(a);  a = o > a ? o : a;
                    o = dpp_move_u32<0x141>(a); a = o > a ? o : a;
                    o = dpp_move_u32<0x140>(a); a = o > a ? o : a;
                    s[i] = block_scale(a);
                    uint4 one[1] = {v[i]};
                    uint2 code[1];
                    block_encode(one, s[i], code);
                    e[i] = code[0];
                }
                if (item + i * 4 * FEW_WAVES >= rows * here) continue;
                *reinterpret_cast<uint2*>(lds + r[i] * S::ROW + g[i] * QB + (((uint32_t)(c >> 1) ^ ((uint32_t)(r[i] >> 1) & 7u)) << 4) + (c & 1) * 8) = e[i];
                if (c == 0) scales[g[i] * S::ROWS + r[i]] = s[i];
            }
        }
        __syncthreads();
        for (int g0 = wave; g0 < S::BLOCKS; g0 += FEW_WAVES * DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const int g = g0 + d * FEW_WAVES;
                if (S::BLOCKS / FEW_WAVES % DEPTH != 0 && g >= S::BLOCKS) continue;
                Stage& o = stage[d];
                if (g < here) {
                    const uint8_t* xr = lds + xrow * S::ROW + g * QB;
                    const uint32_t z = (uint32_t)(xrow >> 1) & 7u;
                    const v4i x0 = *reinterpret_cast<const v4i*>(xr + (((uint32_t)q ^ z) << 4)), x1 = *reinterpret_cast<const v4i*>(xr + (((uint32_t)(q + 4) ^ z) << 4));
                    const v8i xf = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
                    const float s = scales[g * S::ROWS + xrow];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const v8i wf = __builtin_shufflevector(o.w[t][0], o.w[t][1], 0, 1, 2, 3, 4, 5, 6, 7);
                        const v4f y = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
                        const float f = s * o.ws[t];
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[t][i] = __builtin_fmaf(y[i], f, acc[t][i]);
                    }
                }
                const int next = first + g + DEPTH * FEW_WAVES;
                if (next < blocks) load(next, o);
            }
        }
    }
    __syncthreads();
    v4f* const sums = reinterpret_cast<v4f*>(lds);
#pragma unroll
    for (int t = 0; t < NT; ++t) sums[(wave * NT + t) * 64 + lane] = acc[t];
    __syncthreads();
    if (wave >= NT) return;
    v4f y = sums[wave * 64 + lane];
#pragma unroll
    for (int w = 1; w < FEW_WAVES; ++w) {
        const v4f o = sums[(w * NT + wave) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] += o[e];
    }
    const int n = n0 + wave * 16 + q * 4;
    if (l16 < p.M && n < p.N) {
        if (p.bias != nullptr) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += bf16_bits_to_f32(p.bias[n + e]);
        }
        *reinterpret_cast<uint2*>(p.out + (size_t)l16 * p.ldo + n) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    }
}

// max over the lanes l, l ^ 16, l ^ 32, l ^ 48: the four lanes that hold one row of an MFMA operand.
__device__ __forceinline__ uint32_t quad_rows_max(uint32_t v) {
    auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = a[0] > a[1] ? a[0] : a[1];
    auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return b[0] > b[1] ? b[0] : b[1];
}

// ---- few tokens: the same, quantized where they are multiplied ------------------------------------------------------
// A workgroup owns 16 * NT weight rows and 16 tokens; its wavefronts take the blocks of K in turn, each loads its weight
// block and the tokens' values straight into the MFMA's registers (lane q of a row: bytes 16 q and 64 + 16 q), DEPTH
// blocks ahead, and quantizes the values there - the whole block of a row is in four lanes - while the others' loads are on
// their way.  The partial sums meet in LDS, added in wavefront order.  (More than 16 tokens a workgroup, so that weights are read
// fewer times, is slower: every size from 17 to 64 tokens, most by a third; the second reading comes out of the L2.)
// Bound by the quantizer's eight instructions a value, done once per 16 NT columns (blocks further ahead change nothing): 50 x 1024 x
// 4096 8.7 us, 3.6 of them that.
template <int NT, int WAVES, int DEPTH, bool CODES>
__global__ __launch_bounds__(WAVES * 64) void block_small_kernel(const BlockLinear p) {
    __shared__ float sums[WAVES][NT][64][4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, q = lane >> 4;
    const int m0 = blockIdx.y * 16, n0 = blockIdx.x * (16 * NT);
    const int blocks = (p.K + QB - 1) / QB;
    struct Stage {
        v4i w[NT][2];
        uint4 x[CODES ? 2 : 4];
        float s, ws[NT];
    } stage[DEPTH];
    v4f acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = v4f{0, 0, 0, 0};
    const uint8_t* wrow[NT];
    const float* wsrow[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int n = n0 + t * 16 + l16, first = n0 + t * 16 < p.N ? n0 + t * 16 : p.N - 1;
        wrow[t] = p.w + (size_t)(n < p.N ? n : p.N - 1) * p.K + q * 16;
        wsrow[t] = p.ws + (size_t)(first / QB) * blocks;
    }
    const int m = m0 + l16;
    const int64_t row = m < p.M ? m : p.M - 1;   // (rows past the last repeat it; nobody stores their sums)
    const uint8_t* xrow = CODES ? p.xq + row * p.ldq + q * 16 : reinterpret_cast<const uint8_t*>(p.x + row * p.ldx + q * 16);
    auto load = [&](int g, Stage& o) {
        const int k = g * QB;
        const bool lo = k + q * 16 < p.K, hi = k + 64 + q * 16 < p.K;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            o.w[t][0] = lo ? *reinterpret_cast<const v4i*>(wrow[t] + k) : v4i{0, 0, 0, 0};
            o.w[t][1] = hi ? *reinterpret_cast<const v4i*>(wrow[t] + k + 64) : v4i{0, 0, 0, 0};
            o.ws[t] = wsrow[t][g];
        }
        if constexpr (CODES) {
            o.x[0] = lo ? *reinterpret_cast<const uint4*>(xrow + k) : make_uint4(0, 0, 0, 0);
            o.x[1] = hi ? *reinterpret_cast<const uint4*>(xrow + k + 64) : make_uint4(0, 0, 0, 0);
            o.s = p.xs[row * p.xs_row + g * p.xs_block];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o.x[i] = (i < 2 ? lo : hi) ? *reinterpret_cast<const uint4*>(xrow + 2 * k + (i >> 1) * 128 + (i & 1) * 16) : make_uint4(0, 0, 0, 0);
        }
    };
    auto multiply = [&](Stage& o) {
        v8i xf;
        float s;
        if constexpr (CODES) {
            xf = __builtin_shufflevector(__builtin_bit_cast(v4i, o.x[0]), __builtin_bit_cast(v4i, o.x[1]), 0, 1, 2, 3, 4, 5, 6, 7);
            s = o.s;
        } else {
            uint32_t m2 = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) m2 = absmax8_pk(o.x[i], m2);
            s = block_scale(quad_rows_max(absmax_finish(m2)));
            uint2 c[4];
            block_encode(o.x, s, c);
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
            for (int e = 0; e < 4; ++e) acc[t][e] = __builtin_fmaf(d[e], f, acc[t][e]);
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (wave + d * WAVES < blocks) load(wave + d * WAVES, stage[d]);
    for (int g = wave; g < blocks; g += DEPTH * WAVES) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int now = g + d * WAVES, next = now + DEPTH * WAVES;
            if (now < blocks) multiply(stage[d]);
            if (next < blocks) load(next, stage[d]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) *reinterpret_cast<v4f*>(sums[wave][t][lane]) = acc[t];
    __syncthreads();
    if (wave >= NT) return;
    v4f y = *reinterpret_cast<const v4f*>(sums[0][wave][lane]);
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
        const v4f o = *reinterpret_cast<const v4f*>(sums[w][wave][lane]);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] += o[e];
    }
    const int n = n0 + wave * 16 + q * 4;
    if (m < p.M && n < p.N) {
        if (p.bias != nullptr) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += bf16_bits_to_f32(p.bias[n + e]);
        }
        *reinterpret_cast<uint2*>(p.out + (size_t)m * p.ldo + n) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    }
}

// ---- many tokens: tiles through LDS -------------------------------------------------------------------------------
// Stage = one block of K (128 bytes a row) of the tile's tokens and weight rows and the tokens' scales of that block,
// copied straight into LDS; chunk c of row r lies in slot c ^ ((r >> 1) & 7), so the sixteen rows that a quarter of a
// wavefront reads together are in sixteen different bank groups.  Copies go through buffer resources: rows past the
// matrix repeat its last one, bytes past K arrive as zeros.  777 x 1168 x 4304: 12.9 us in 247 tiles of 64 x 64, one round of workgroups
// that each wait for 17 steps; 2225 x 6912 x 2176 with its quantizer 51 us, 1.3 PFLOP/s.
template <int TM, int TN, int WM, int WN, int WK, int DEPTH>
struct BlockTile {
    static constexpr int BM = 16 * TM * WM, BN = 16 * TN * WN, WAVES = WM * WN;
    static constexpr int GA = BM / 8, GB = BN / 8, GS = (BM + 63) / 64 + 1;   // copies of a stage: eight rows; 64 scales, of the columns last
    static constexpr int STAGE = (BM + BN) * QB + GS * 256;
    static constexpr int EACH = (GA + GB + WAVES - 1) / WAVES, EACH_S = (GS + WAVES - 1) / WAVES;   // of a wavefront, at most
    static constexpr int LEAST = (GA + GB) / WAVES;                                                // and at least
    static constexpr int LDS = STAGE * WK * DEPTH;
};

__device__ __forceinline__ uint32_t block_swizzle(int row) { return (uint32_t)(row >> 1) & 7u; }

template <int TM, int TN, int WM, int WN, int WK, int DEPTH>
__global__ __launch_bounds__(WM * WN * WK * 64) void block_gemm_kernel(const BlockLinear p, int m_tiles, int n_tiles, int band, int per_xcd) {
    using T = BlockTile<TM, TN, WM, WN, WK, DEPTH>;
    __shared__ __align__(16) uint8_t lds[T::LDS];
    // Workgroup i runs on XCD i % 8: each takes a run of the tiles, in bands of `band` tile rows, column after column
    int tile = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per_xcd || tile >= m_tiles * n_tiles) return;
    const int of_band = tile / (band * n_tiles), in_band = tile - of_band * band * n_tiles;
    const int rows_here = m_tiles - of_band * band < band ? m_tiles - of_band * band : band;
    const int nt = in_band / rows_here, mt = of_band * band + in_band - nt * rows_here;
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, q = lane >> 4;
    // WK groups of WM x WN wavefronts take the blocks of K in turn and add their sums at the end
    const int group = WK > 1 ? __builtin_amdgcn_readfirstlane(tid / (T::WAVES * 64)) : 0, wave = __builtin_amdgcn_readfirstlane(tid >> 6) - group * T::WAVES;
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
    const int steps = (blocks + WK - 1) / WK;
    // (a block past the last is copied as zeros, without an access)
    auto issue = [&](int step) {
        const int d = step * WK + group;
        const uint32_t at = base + (uint32_t)((step % DEPTH) * WK + group) * T::STAGE;
        const uint32_t drop = d < blocks - 1 ? 0u : d == blocks - 1 ? gone : kCopyNothing, k = (uint32_t)d * QB;
#pragma unroll
        for (int i = 0; i < T::EACH_S; ++i) {
            const int c = wave + i * T::WAVES;
            if (c >= T::GS) continue;
            const uint32_t to = __builtin_amdgcn_readfirstlane(at + (T::GA + T::GB) * 1024 + c * 256);
            asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds"
                         :: "v"(d < blocks ? soff[i] : kCopyNothing), "s"(c < T::GS - 1 ? s_src : ws_src), "s"((uint32_t)d * __builtin_amdgcn_readfirstlane(sstep[i])), "s"(to) : "memory", "m0");
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
        if (d < steps) issue(d);
    for (int d = 0; d < steps; ++d) {
        // stage d is complete (this wavefront's copies by the wait, the others' by the barrier) and stage d - 1 has been read
        if (DEPTH > 2 && d + DEPTH - 2 < steps) wait_copies<(DEPTH - 2) * T::LEAST>();   // (some wavefronts have more in flight, and wait for a few too many)
        else wait_copies<0>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (d + DEPTH - 1 < steps) issue(d + DEPTH - 1);
        const uint8_t* stage = lds + ((d % DEPTH) * WK + group) * T::STAGE;
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
    if constexpr (WK > 1) {
        // the groups' sums, in order: the first one's registers, then the others' through LDS (no copy is in flight)
        static_assert((WK - 1) * T::WAVES * TM * TN * 1024 <= T::LDS, "the sums fit where the stages were");
        __syncthreads();
        v4f* sums = reinterpret_cast<v4f*>(lds);
        if (group > 0) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) sums[(((group - 1) * T::WAVES + wave) * TM * TN + i * TN + j) * 64 + lane] = acc[i][j];
        }
        __syncthreads();
        if (group > 0) return;
#pragma unroll
        for (int g = 0; g < WK - 1; ++g)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    const v4f o = sums[((g * T::WAVES + wave) * TM * TN + i * TN + j) * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] += o[e];
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

// The largest problems: 32 TM x 256 tiles, eight wavefronts of 16 TM x 64, two per SIMD.  What a step costs beside its
// products is the beginning: eight wavefronts behind a barrier that all want their first operands from LDS.  So the weight
// fragments of a step are read at the end of the one before it - the stages of weights run one step further ahead than
// those of tokens, in three buffers instead of two - and the last row block of a step is scaled and added behind the
// barrier, while the first token fragment comes; the copies are issued between the products.  13056 x 2048 x 16384: 417 us, 2.1 PFLOP/s
// with the MFMA busy 58 % of the time at the clock that the chip's power leaves.
template <int TM>
struct WideTile {
    static constexpr int TN = 4, WM = 2, WN = 4, WAVES = 8, BM = 32 * TM, BN = 256;
    static constexpr int GA = BM / 8, GB = BN / 8, GS = (BM + 63) / 64 + 1;
    static constexpr int A_STAGE = BM * QB, B_STAGE = BN * QB, S_STAGE = GS * 256;
    static constexpr int B_AT = 2 * A_STAGE, S_AT = B_AT + 3 * B_STAGE, LDS = S_AT + 2 * S_STAGE;
    static constexpr int EACH_A = (GA + WAVES - 1) / WAVES, EACH_B = GB / WAVES;
};

template <int TM>
__global__ __launch_bounds__(512) void block_wide_kernel(const BlockLinear p, int m_tiles, int n_tiles, int band, int per_xcd) {
    using T = WideTile<TM>;
    constexpr int TN = T::TN;
    __shared__ __align__(16) uint8_t lds[T::LDS];
    int tile = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per_xcd || tile >= m_tiles * n_tiles) return;
    const int of_band = tile / (band * n_tiles), in_band = tile - of_band * band * n_tiles;
    const int rows_here = m_tiles - of_band * band < band ? m_tiles - of_band * band : band;
    const int nt = in_band / rows_here, mt = of_band * band + in_band - nt * rows_here;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, q = lane >> 4;
    const int wm = wave / T::WN, wn = wave % T::WN;
    const int m0 = mt * T::BM, n0 = nt * T::BN;
    const int blocks = (p.K + QB - 1) / QB;

    const int lr = lane >> 3;
    const uint32_t chunk = ((uint32_t)(lane & 7) ^ block_swizzle((wave & 1) * 8 + lr)) * 16;   // (groups wave, wave + 8, ...: one parity)
    const int tail = p.K & (QB - 1);
    const uint32_t gone = tail != 0 && (int)chunk >= tail ? kCopyNothing : 0u;
    uint32_t aoff[T::EACH_A], boff[T::EACH_B], soff;
#pragma unroll
    for (int i = 0; i < T::EACH_A; ++i) {
        const int m = m0 + (wave + i * 8) * 8 + lr;
        aoff[i] = (uint32_t)(m < p.M ? m : p.M - 1) * (uint32_t)p.ldq + chunk;
    }
#pragma unroll
    for (int i = 0; i < T::EACH_B; ++i) {
        const int n = n0 + (wave + i * 8) * 8 + lr;
        boff[i] = (uint32_t)(n < p.N ? n : p.N - 1) * (uint32_t)p.K + chunk;
    }
    const int n_blocks = (p.N + QB - 1) / QB;
    const v4i a_src = copy_source(p.xq, (uint32_t)((int64_t)(p.M - 1) * p.ldq + p.K));
    const v4i b_src = copy_source(p.w, (uint32_t)p.N * (uint32_t)p.K);
    // the scales: wavefronts 0 .. GS - 2 bring 64 of the tokens each, the others those of the columns (the same bytes to the same place)
    const int scales = wave < T::GS - 1 ? wave : T::GS - 1;
    const bool of_rows = scales < T::GS - 1;
    const v4i s_src = of_rows ? copy_source(reinterpret_cast<const uint8_t*>(p.xs), (uint32_t)(((int64_t)(p.M - 1) * p.xs_row + (int64_t)(blocks - 1) * p.xs_block + 1) * 4))
                              : copy_source(reinterpret_cast<const uint8_t*>(p.ws), (uint32_t)n_blocks * (uint32_t)blocks * 4u);
    {
        const int m = m0 + wave * 64 + lane, nb = n0 / QB + lane;
        soff = of_rows ? (uint32_t)(m < p.M ? m : p.M - 1) * (uint32_t)p.xs_row * 4u : (uint32_t)(nb < n_blocks ? nb : n_blocks - 1) * (uint32_t)blocks * 4u;
    }
    const uint32_t sstep = of_rows ? (uint32_t)p.xs_block * 4u : 4u;
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    // Steps that do not exist are copied too, as zeros and without an access (kCopyNothing): no branches in the loop.
    auto part_of = [&](int d) -> uint32_t { return d < blocks - 1 ? 0u : d == blocks - 1 ? gone : kCopyNothing; };
    auto issue_a = [&](int d, uint32_t drop, int i) {
        if ((i + 1) * 8 > T::GA && wave + i * 8 >= T::GA) return;
        copy16_to_lds_checked(a_src, aoff[i] | drop, (uint32_t)d * QB, __builtin_amdgcn_readfirstlane(base + (uint32_t)(d & 1) * T::A_STAGE + (wave + i * 8) * 1024));
    };
    auto issue_b = [&](int d, uint32_t drop, uint32_t slot, int i) {
        copy16_to_lds_checked(b_src, boff[i] | drop, (uint32_t)d * QB, __builtin_amdgcn_readfirstlane(base + T::B_AT + slot * T::B_STAGE + (wave + i * 8) * 1024));
    };
    auto issue_s = [&](int d) {
        asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds"
                     :: "v"(d < blocks ? soff : kCopyNothing), "s"(s_src), "s"((uint32_t)d * sstep),
                        "s"(__builtin_amdgcn_readfirstlane(base + T::S_AT + (uint32_t)(d & 1) * T::S_STAGE + scales * 256)) : "memory", "m0");
    };
    const uint32_t f0 = (uint32_t)l16 * QB + (((uint32_t)q ^ block_swizzle(l16)) << 4);
    auto fragment = [&](const uint8_t* rows) -> v8i {
        const v4i a = *reinterpret_cast<const v4i*>(rows + f0), b = *reinterpret_cast<const v4i*>(rows + (f0 ^ 64u));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    v4f acc[TM][TN], t[2][TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[i][j] = v4f{0, 0, 0, 0};
        t[(TM - 1) & 1][j] = v4f{0, 0, 0, 0};
    }
    float late = 0.f;   // scale of the row block that is still to be added
    issue_s(0);
#pragma unroll
    for (int i = 0; i < T::EACH_A; ++i) issue_a(0, part_of(0), i);
#pragma unroll
    for (int i = 0; i < T::EACH_B; ++i) {
        issue_b(0, part_of(0), 0, i);
        issue_b(1, part_of(1), 1, i);
    }
    v8i wf[TN];
    uint32_t b_next = 1, b_fill = 2;   // buffers of the weights of steps d + 1 and d + 2
#pragma unroll 1
    for (int d = 0; d < blocks; ++d) {
        // tokens of step d and weights of step d + 1 are complete (this wavefront's copies by the wait, the others' by the
        // barrier), and the buffers that are filled next have been read
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const uint8_t* xbuf = lds + (d & 1) * T::A_STAGE + wm * TM * 16 * QB;
        const float* sbuf = reinterpret_cast<const float*>(lds + T::S_AT + (d & 1) * T::S_STAGE);
        if (d == 0) {
#pragma unroll
            for (int j = 0; j < TN; ++j) wf[j] = fragment(lds + T::B_AT + (wn * TN + j) * 16 * QB);
        }
        v8i xf = fragment(xbuf);
        float f[TM];
        const float wscale = sbuf[(T::GS - 1) * 64 + wn * 16 * TN / QB];
#pragma unroll
        for (int i = 0; i < TM; ++i) f[i] = sbuf[(wm * TM + i) * 16 + l16];
        uint32_t drop1 = part_of(d + 1), drop2 = part_of(d + 2);
        asm volatile("" : "+v"(drop1), "+v"(drop2));   // (or every offset is kept twice, with and without it)
        const uint8_t* wnext = lds + T::B_AT + b_next * T::B_STAGE + wn * TN * 16 * QB;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const v8i x = xf;
            if (i + 1 < TM) xf = fragment(xbuf + (i + 1) * 16 * QB);
            // the row block before this one: of the last step if this is the first
            const float s = i == 0 ? late : f[i - 1] * wscale;
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const v4f y = t[i == 0 ? (TM - 1) & 1 : (i - 1) & 1][j];
                t[i & 1][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], x, v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
                if (i == TM - 1) wf[j] = fragment(wnext + j * 16 * QB);
                const int o = i == 0 ? TM - 1 : i - 1;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[o][j][e] = __builtin_fmaf(y[e], s, acc[o][j][e]);
            }
            if (i == 0) {
                issue_s(d + 1);
#pragma unroll
                for (int c = 0; c < T::EACH_A; ++c) issue_a(d + 1, drop1, c);
            }
            if (i == 1) {
#pragma unroll
                for (int c = 0; c < T::EACH_B; ++c) issue_b(d + 2, drop2, b_fill, c);
            }
            __builtin_amdgcn_sched_barrier(0);   // (row blocks run into each other otherwise, and out of registers)
        }
        late = f[TM - 1] * wscale;
        b_next = b_fill;
        b_fill = b_fill == 2 ? 0 : b_fill + 1;
    }
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[TM - 1][j][e] = __builtin_fmaf(t[(TM - 1) & 1][j][e], late, acc[TM - 1][j][e]);
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

template <int TM>
hipError_t launch_wide(const BlockLinear& p, hipStream_t stream) {
    using T = WideTile<TM>;
    const int mt = (p.M + T::BM - 1) / T::BM, nt = (p.N + T::BN - 1) / T::BN;
    const int per = (mt * nt + 7) / 8, band = 1024 / T::BM;
    return enqueue(block_wide_kernel<TM>, dim3((uint32_t)per * 8), dim3(512), stream, p, mt, nt, band, per);
}

template <int TM, int TN, int WM, int WN, int WK, int DEPTH>
hipError_t launch_tile(const BlockLinear& p, hipStream_t stream) {
    using T = BlockTile<TM, TN, WM, WN, WK, DEPTH>;
    const int mt = (p.M + T::BM - 1) / T::BM, nt = (p.N + T::BN - 1) / T::BN;
    const int per = (mt * nt + 7) / 8, band = 1024 / T::BM;
    return enqueue(block_gemm_kernel<TM, TN, WM, WN, WK, DEPTH>, dim3((uint32_t)per * 8), dim3(T::WAVES * WK * 64), stream, p, mt, nt, band, per);
}

template <int NT, int DEPTH>
hipError_t launch_few(const BlockLinear& p, hipStream_t stream) {
    const dim3 grid((uint32_t)((p.N + 16 * NT - 1) / (16 * NT)));
    return p.x == nullptr ? enqueue(block_few_kernel<NT, DEPTH, true>, grid, dim3(FEW_WAVES * 64), stream, p)
                          : enqueue(block_few_kernel<NT, DEPTH, false>, grid, dim3(FEW_WAVES * 64), stream, p);
}

template <int NT, int WAVES, int DEPTH>
hipError_t launch_small(const BlockLinear& p, hipStream_t stream) {
    const dim3 grid((uint32_t)((p.N + 16 * NT - 1) / (16 * NT)), (uint32_t)((p.M + 15) / 16));
    return p.x == nullptr ? enqueue(block_small_kernel<NT, WAVES, DEPTH, true>, grid, dim3(WAVES * 64), stream, p)
                          : enqueue(block_small_kernel<NT, WAVES, DEPTH, false>, grid, dim3(WAVES * 64), stream, p);
}

}  // namespace

hipError_t launch_block_quant(const uint16_t* x, int64_t ldx, int64_t M, int64_t K, uint8_t* xq, int64_t ldq, float* xs, int64_t xs_row,
                        int64_t xs_block, hipStream_t stream) {
    const int blocks = (int)((K + QB - 1) / QB);
    const int64_t items = M * blocks;
    return enqueue(block_quant_kernel, dim3((uint32_t)((items + 15) / 16)), dim3(256), stream, x, ldx, (int)K, blocks, items, xq, ldq, xs,
                       xs_row, xs_block);
}

// ---- which kernel ---------------------------------------------------------------------------------------------------
namespace {
// Microseconds of M x N x K, as fitted to event-timed graphs of 60 shapes from 1 x 256 x 256 to 13056 x 32768 x 2048.  What they choose is
// 0.7 % behind the best kernel in the geometric mean over 68 shapes of that range, three of them more than 8 % (100 x 2560 x 1024: 9.2 us
// chosen, 7.6 in tiles of 64 x 64; 8 x 32768 x 2048 16.5 and 14.9); the microseconds themselves are within a fifth at 47 of 59 for
// few tokens and at 249 of 272 for the tiles.
constexpr int FEW_ROWS = 4;   // up to here quantizing into LDS first wins: 1 x 12288 x 2048 7.4 us, 8.0 where they are multiplied; 16 x 2048 x 16384 41 and 26
enum Shape { SHAPE_SMALL, SHAPE_64_SPLIT, SHAPE_64, SHAPE_128, SHAPE_224 };
// Weight tiles of a workgroup of the kernels for few tokens.  For up to FEW_ROWS one, or four once there are workgroups for every
// CU all the same: 1 x 8192 x 8192 15.1 us with one and 20.1 with four, 1 x 12288 x 2048 7.8 and 7.1.  Beyond,
// about one workgroup per CU, each with all the weights that go with the rows it quantizes: 16 x 16384 x 1024 12.3 / 8.8 / 6.3 us with
// 1 / 2 / 4, 32 x 2048 x 2048 6.0 / 6.7 / 8.5.
int small_tiles(int64_t M, int64_t N) {
    const int64_t units = (N + 15) / 16 * ((M + 15) / 16);
    if (M <= FEW_ROWS) return units < 640 ? 1 : 4;
    return units <= 288 ? 1 : units <= 576 ? 2 : 4;
}
// Wavefronts of block_small_kernel: 16 for long K and up to two weight tiles, whose instructions then fill the SIMDs' gaps: 14 x 896 x
// 7024 11.6 us with 8 and 10.3 with 16, 50 x 1024 x 4096 9.5 and 8.7, 40 x 2048 x 4096 11.4 and 10.1; 16 x 2560 x 1024 4.2 and 4.4.
bool small_wide(int nt, int64_t K) { return nt <= 2 && K >= 2048; }
double small_cost(int64_t M, int64_t N, int64_t K) {
    const int nt = small_tiles(M, N);
    const int64_t groups = ((N + 16 * nt - 1) / (16 * nt)) * ((M + 15) / 16), turns = (K + QB * 8 - 1) / (QB * 8);
    return 2.6 + turns * (nt == 1 ? 1.5 : nt == 2 ? 2.05 : 3.1) * (groups <= 256 ? 1.0 : groups / 256.0);
}
// The quantizer, and a tile kernel: rounds of workgroups (one per CU, or two), each K block the dearer the more CUs are busy.
double tile_cost(Shape s, int64_t M, int64_t N, int64_t K) {
    const int64_t bm = s == SHAPE_224 ? 224 : s == SHAPE_128 ? 128 : 64, bn = s == SHAPE_224 ? 256 : s == SHAPE_128 ? 128 : 64;
    const bool two = s == SHAPE_64 || s == SHAPE_128;
    const double tiles = (double)(((M + bm - 1) / bm) * ((N + bn - 1) / bn)), slots = two ? 512.0 : 256.0, load = tiles < slots ? tiles / slots : 1.0;
    const double rounds = tiles <= slots ? 1.0 : two ? tiles / slots + 0.25 : (double)(int64_t)((tiles + slots - 1) / slots);
    static constexpr double idle[] = {0, 0.2, 0.28, 0.6, 1.2}, busy[] = {0, 0.15, 0.3, 0.5, 0.35}, leave[] = {0, 0.5, 0.5, 1.0, 3.0};
    return 5.5 + (double)M * (double)K * 0.7e-6 + rounds * ((double)((K + QB - 1) / QB) * (idle[s] + busy[s] * load) + leave[s]);
}
Shape choose(int64_t M, int64_t N, int64_t K) {
    if (const char* forced = tuning_env("PHYAI_LAYER_BLOCK")) return (Shape)atoi(forced);
    if (M <= FEW_ROWS) return SHAPE_SMALL;
    Shape best = SHAPE_64_SPLIT;
    for (Shape s : {SHAPE_64, SHAPE_128, SHAPE_224})
        if (tile_cost(s, M, N, K) < tile_cost(best, M, N, K)) best = s;
    return M <= 1024 && small_cost(M, N, K) < tile_cost(best, M, N, K) ? SHAPE_SMALL : best;
}
}  // namespace

bool block_linear_small(int64_t M, int64_t N, int64_t K) { return choose(M, N, K) == SHAPE_SMALL; }

hipError_t launch_block_linear_small(const BlockLinear& p, hipStream_t stream) {
    int nt = small_tiles(p.M, p.N);
    bool few = p.M <= FEW_ROWS, wide = small_wide(nt, p.K);
    if (const char* forced = tuning_env("PHYAI_LAYER_SMALL")) {   // weight tiles of a workgroup (of a few tokens: 1, else 4); + 10: not the kernel of a few tokens; + 30: nor 8 wavefronts
        nt = atoi(forced) % 10;
        few = p.M <= 8 && atoi(forced) < 10;
        wide = nt <= 2 && atoi(forced) >= 30;
    }
    if (few) return nt == 1 ? launch_few<1, 4>(p, stream) : launch_few<4, 2>(p, stream);
    if (wide) return nt == 1 ? launch_small<1, 16, 2>(p, stream) : launch_small<2, 16, 1>(p, stream);
    return nt == 1 ? launch_small<1, 8, 4>(p, stream) : nt == 2 ? launch_small<2, 8, 4>(p, stream) : launch_small<4, 8, 2>(p, stream);
}

hipError_t launch_block_gemm(const BlockLinear& p, hipStream_t stream) {
    switch (choose(p.M, p.N, p.K)) {
        case SHAPE_64_SPLIT: return launch_tile<2, 2, 2, 2, 2, 4>(p, stream);
        case SHAPE_64: return launch_tile<2, 2, 2, 2, 2, 2>(p, stream);
        case SHAPE_128: return launch_tile<4, 2, 2, 4, 1, 2>(p, stream);
        default: return launch_wide<7>(p, stream);
    }
}

}  // namespace phyai
