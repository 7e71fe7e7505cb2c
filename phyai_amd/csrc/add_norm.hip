// The residual's addition, the root-mean-square norm of the sum and its quantization to e4m3, in one pass (gfx950).  For a row:
//
//     t = bf16(x + residual)                                 (written: the residual stream goes on with it)
//     n[i] = t[i] * rsqrt(mean(t^2) + eps) * w[i]            (w + 1 in the Gemma form), fp32, not rounded in between
//     scale_g = max(amax of n over group g, 1e-12) / 448     (fp32; groups of 128 elements, or the row)
//     codes = e4m3(n / scale_g)                              (round to nearest even)
//
// A workgroup has a row, in registers: both inputs are read once, the sum and the codes written once.  Sixteen lanes of eight
// elements are a group of 128, so its maximum takes four steps inside a row of lanes; a row's goes through LDS.  Bound by memory, seven
// bytes an element: 13056 x 2048 in 31.4 us, 6.0 TB/s (the last states of a loop are still in the caches; 34.8, 5.4, where three take
// turns), where a large copy runs at 4.9; one row 2.6 us, the launch and a turn of memory.
#include "fp8_device.h"
#include "layer_kernels.h"
#include "quant_device.h"
#include "tuning.h"

namespace phyai {
namespace {

__device__ __forceinline__ void unpack8(const v4i& q, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float((uint32_t)q[i] << 16);
        f[2 * i + 1] = __uint_as_float((uint32_t)q[i] & 0xFFFF0000u);
    }
}
// bf16(x + residual), eight of them
__device__ __forceinline__ v4i add8(const v4i& x, const v4i& r) {
    float a[8], b[8];
    unpack8(x, a);
    unpack8(r, b);
    v4i t;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = (int)pack_bf16x2(a[2 * i] + b[2 * i], a[2 * i + 1] + b[2 * i + 1]);
    return t;
}
// Maxima of magnitudes as bit patterns: a NaN wins.
__device__ __forceinline__ uint32_t amax8(const float* n) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = __float_as_uint(n[i]) & 0x7FFFFFFFu;
        m = b > m ? b : m;
    }
    return m;
}
__device__ __forceinline__ uint32_t max_of_16_lanes(uint32_t v) {
    uint32_t o;
    o = dpp_move_u32<0xB1>(v);  v = o > v ? o : v;
    o = dpp_move_u32<0x4E>(v);  v = o > v ? o : v;
    o = dpp_move_u32<0x141>(v); v = o > v ? o : v;
    o = dpp_move_u32<0x140>(v); v = o > v ? o : v;
    return v;
}
__device__ __forceinline__ float scale_of(uint32_t amax) {
    const float a = __uint_as_float(amax);
    return (a < 1e-12f ? 1e-12f : a) / kFp8Max;   // (a NaN stays one)
}
// Quotients by a reciprocal and a correction step (StaticDivisor), which differ from a division's at most in the last bit; the
// division itself outside that step's range.
__device__ __forceinline__ uint2 encode8(const float* n, const StaticDivisor& d) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = d.fast ? quotient(n[i], n[i] * d.r, d.s, d.r) : n[i] / d.s;
    if (__builtin_expect(!d.fast, 0))   // (there may be NaNs)
        return make_uint2(e4m3_pack2(v[0], v[1]) | e4m3_pack2(v[2], v[3]) << 16, e4m3_pack2(v[4], v[5]) | e4m3_pack2(v[6], v[7]) << 16);
    return make_uint2(encode4(v[0], v[1], v[2], v[3]), encode4(v[4], v[5], v[6], v[7]));
}
// (The product of two bf16 values is exact in fp32: one rounding, that of r's product.  With gemma w + 1 may round as well, and its product with t.)
__device__ __forceinline__ void normed8(const v4i& t, const v4i& w, float r, float more, float* n) {
    float wf[8];
    unpack8(t, n);
    unpack8(w, wf);
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = n[i] * (wf[i] + more) * r;
}

// Over the workgroup's wavefronts, whose words are in LDS, in their order.
__device__ __forceinline__ float sum_of_all(float v, float* words) {
    const int waves = blockDim.x / kWave;
    v = wave_sum_f32(v);
    if (waves > 1) {
        if (threadIdx.x % kWave == 0) words[threadIdx.x / kWave] = v;
        __syncthreads();
        v = words[0];
        for (int i = 1; i < waves; ++i) v += words[i];
    }
    return v;
}
__device__ __forceinline__ uint32_t max_of_all(uint32_t v, uint32_t* words) {
    const int waves = blockDim.x / kWave;
    v = wave_max_u32(v);
    if (waves > 1) {
        if (threadIdx.x % kWave == 0) words[threadIdx.x / kWave] = v;
        __syncthreads();
        v = words[0];
        for (int i = 1; i < waves; ++i) v = words[i] > v ? words[i] : v;
    }
    return v;
}

template <int CHUNKS, bool BLOCKS>
__global__ __launch_bounds__(1024) void add_norm_kernel(const AddNorm p) {
    __shared__ float sums[1024 / kWave];
    __shared__ uint32_t maxima[1024 / kWave];
    const int threads = blockDim.x;
    const int64_t row = blockIdx.x;
    const uint16_t *x = p.x + row * p.ldx, *residual = p.residual + row * p.ldr;
    v4i t[CHUNKS], w[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int k = (c * threads + threadIdx.x) * 8;
        t[c] = v4i{0, 0, 0, 0};
        w[c] = v4i{0, 0, 0, 0};
        if (k < p.D) {
            t[c] = add8(*reinterpret_cast<const v4i*>(x + k), *reinterpret_cast<const v4i*>(residual + k));
            w[c] = *reinterpret_cast<const v4i*>(p.weight + k);
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int k = (c * threads + threadIdx.x) * 8;
        if (k < p.D) *reinterpret_cast<v4i*>(p.total + row * p.ldt + k) = t[c];
        float f[8];
        unpack8(t[c], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(f[i], f[i], ss);
    }
    ss = sum_of_all(ss, sums);
    const float r = 1.0f / __builtin_sqrtf(ss / (float)p.D + p.eps), more = p.gemma ? 1.0f : 0.0f;
    uint8_t* codes = p.xq + row * (int64_t)p.D;
    float* scale = p.scale + row * p.xs_row;
    if constexpr (BLOCKS) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int k = (c * threads + threadIdx.x) * 8;
            float n[8];
            normed8(t[c], w[c], r, more, n);
            const float s = scale_of(max_of_16_lanes(amax8(n)));
            if (k >= p.D) continue;
            if ((k & 127) == 0) scale[(int64_t)(k >> 7) * p.xs_block] = s;
            *reinterpret_cast<uint2*>(codes + k) = encode8(n, make_static_divisor(s));
        }
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            float n[8];
            normed8(t[c], w[c], r, more, n);
            const uint32_t a = amax8(n);
            m = a > m ? a : m;
        }
        const float s = scale_of(max_of_all(m, maxima));
        if (threadIdx.x == 0) scale[0] = s;
        const StaticDivisor d = make_static_divisor(s);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int k = (c * threads + threadIdx.x) * 8;
            float n[8];
            normed8(t[c], w[c], r, more, n);
            if (k < p.D) *reinterpret_cast<uint2*>(codes + k) = encode8(n, d);
        }
    }
}

// Rows too long for registers: the sum is written and read again, by the same threads.
template <bool BLOCKS>
__global__ __launch_bounds__(512) void add_norm_long_kernel(const AddNorm p) {
    __shared__ float sums[8];
    __shared__ uint32_t maxima[8];
    const int64_t row = blockIdx.x;
    const uint16_t *x = p.x + row * p.ldx, *residual = p.residual + row * p.ldr;
    uint16_t* total = p.total + row * p.ldt;
    float ss = 0.f;
    for (int k = threadIdx.x * 8; k < p.D; k += 512 * 8) {
        const v4i t = add8(*reinterpret_cast<const v4i*>(x + k), *reinterpret_cast<const v4i*>(residual + k));
        *reinterpret_cast<v4i*>(total + k) = t;
        float f[8];
        unpack8(t, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(f[i], f[i], ss);
    }
    ss = sum_of_all(ss, sums);
    const float r = 1.0f / __builtin_sqrtf(ss / (float)p.D + p.eps), more = p.gemma ? 1.0f : 0.0f;
    uint8_t* codes = p.xq + row * (int64_t)p.D;
    float* scale = p.scale + row * p.xs_row;
    StaticDivisor d = {};
    if constexpr (!BLOCKS) {
        uint32_t m = 0;
        for (int k = threadIdx.x * 8; k < p.D; k += 512 * 8) {
            float n[8];
            normed8(*reinterpret_cast<const v4i*>(total + k), *reinterpret_cast<const v4i*>(p.weight + k), r, more, n);
            const uint32_t a = amax8(n);
            m = a > m ? a : m;
        }
        const float s = scale_of(max_of_all(m, maxima));
        if (threadIdx.x == 0) scale[0] = s;
        d = make_static_divisor(s);
    }
    const int steps = (p.D + 512 * 8 - 1) / (512 * 8);
    for (int c = 0; c < steps; ++c) {   // (all lanes: they exchange maxima)
        const int k = (c * 512 + threadIdx.x) * 8;
        float n[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (k < p.D) normed8(*reinterpret_cast<const v4i*>(total + k), *reinterpret_cast<const v4i*>(p.weight + k), r, more, n);
        if constexpr (BLOCKS) {
            const float s = scale_of(max_of_16_lanes(amax8(n)));
            if (k < p.D && (k & 127) == 0) scale[(int64_t)(k >> 7) * p.xs_block] = s;
            d = make_static_divisor(s);
        }
        if (k < p.D) *reinterpret_cast<uint2*>(codes + k) = encode8(n, d);
    }
}

template <bool BLOCKS>
hipError_t launch_blocks(const AddNorm& p, hipStream_t stream) {
    const dim3 grid((uint32_t)p.M);
    // One chunk of eight elements a thread where few rows leave most of the chip empty: a row is then one turn of memory.  With more, two or
    // three, whichever leaves fewer lanes without work: wavefronts of a row wait for each other less.  us with 1 / 2 / 3 chunks: 1 x
    // 2048 2.6 / 3.2 / 3.3, 816 x 2048 4.4 / 4.6 / 4.8, 777 x 4304 8.7 / 8.3 / 7.8, 6000 x 1152 11.6 / 11.7 / 11.1, 3264 x 8192 37.2 / 32.4 / 33.2, 13056 x 2048
    // 32.7 / 31.4 / 31.9.
    const int lanes = (p.D + 7) / 8;
    auto threads_of = [&](int c) { return ((lanes + c - 1) / c + kWave - 1) / kWave * kWave; };
    int chunks = 1;
    if (p.M * threads_of(1) > 4096 * kWave) chunks = threads_of(3) * 3 < threads_of(2) * 2 ? 3 : 2;
    if (lanes <= kWave) chunks = 1;
    if (const char* forced = tuning_env("PHYAI_LAYER_ADD_NORM")) {   // (what is no number of chunks changes nothing)
        const int n = atoi(forced);
        if (n >= 1 && n <= 4) chunks = n;
    }
    while (threads_of(chunks) > 1024) ++chunks;
    const dim3 threads((uint32_t)threads_of(chunks));
    if (lanes > 4096) return enqueue(add_norm_long_kernel<BLOCKS>, grid, dim3(512), stream, p);
    switch (chunks) {
        case 1: return enqueue(add_norm_kernel<1, BLOCKS>, grid, threads, stream, p);
        case 2: return enqueue(add_norm_kernel<2, BLOCKS>, grid, threads, stream, p);
        case 3: return enqueue(add_norm_kernel<3, BLOCKS>, grid, threads, stream, p);
        default: return enqueue(add_norm_kernel<4, BLOCKS>, grid, threads, stream, p);
    }
}

}  // namespace

hipError_t launch_add_norm(const AddNorm& p, hipStream_t stream) {
    return p.per_block ? launch_blocks<true>(p, stream) : launch_blocks<false>(p, stream);
}

}  // namespace phyai
