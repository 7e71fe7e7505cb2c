// Norms of the query and key heads of a fused projection, the position rotation, and the write of keys and values into
// a paged cache, in one pass (gfx950).  For a head x[0 .. D) of the query or key part of a token at position t:
//
//     n[i] = x[i] * rsqrt(mean(x^2) + eps) * w[i]            (w + 1 in the Gemma form; no weights: n = x)
//     (n[a], n[b]) -> (n[a] cos - n[b] sin, n[b] cos + n[a] sin)   for the rot / 2 pairs (a, b)
//
// with (a, b) = (i, i + rot / 2) or, interleaved, (2 i, 2 i + 1); cos and sin from row t of a table.  Everything between
// the load and the one rounding at the end is fp32.  Value heads are copied.
//
// A group of lanes owns a head: each lane holds two runs of V elements that make up whole pairs, so the rotation needs
// no exchange, and the sum of squares is a few lane shuffles.  The angles are loaded once for the heads of a token that
// a group goes through.  Bound by memory: every element is read once and written once; 13056 tokens of 8 + 2 heads of 256 in
// 32.1 us, 4.6 TB/s, where a large copy runs at 5.2; one token 4.5 us, the launch.
#include "fp8_device.h"
#include "layer_kernels.h"

namespace phyai {
namespace {

template <int TYPE>
__device__ __forceinline__ float head_to_f32(uint32_t h) {
    if constexpr (TYPE == HEAD_BF16) return __uint_as_float(h << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
template <int TYPE>
__device__ __forceinline__ uint32_t head_pack2(float a, float b) {
    if constexpr (TYPE == HEAD_BF16) return pack_bf16x2(a, b);
    else {   // (both at once: no instruction that writes half a register)
        typedef float two __attribute__((ext_vector_type(2)));
        typedef _Float16 pair __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(two{a, b}, pair));
    }
}

template <int V>
struct Run {
    uint32_t w[V / 2];
};
template <int V>
__device__ __forceinline__ Run<V> load_run(const uint16_t* p) {
    Run<V> r;
    if constexpr (V == 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        r.w[0] = v.x; r.w[1] = v.y;
    }
    return r;
}
template <int V>
__device__ __forceinline__ void store_run(uint16_t* p, const Run<V>& r) {
    if constexpr (V == 8) *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(r.w[0], r.w[1]);
}

// LP lanes a head (a power of two, at least D / (2 V)); `heads_per_group` heads of one token, neighbours, per group.
template <int TYPE, int V>
__global__ __launch_bounds__(256) void head_rope_kernel(const HeadRope p, int lp_log, int heads_per_group, int groups_per_token, int64_t groups) {
    const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> lp_log;
    const int c = threadIdx.x & ((1 << lp_log) - 1);
    if (group >= groups) return;   // (a head's lanes leave together)
    const int t = (int)(group / groups_per_token);
    const int first = (int)(group - (int64_t)t * groups_per_token) * heads_per_group;
    const int heads = p.H + 2 * p.KV;
    const int last = first + heads_per_group < heads ? first + heads_per_group : heads;
    const bool active = c * 2 * V < p.D;
    // the lane's two runs: pairs of the rotated part, or a stretch behind it
    const int half = p.rot >> 1;
    const bool turned = p.interleaved ? c * 2 * V < p.rot : c * V < half;
    int a, b;
    if (turned && !p.interleaved) { a = c * V; b = half + c * V; }
    else if (p.interleaved) { a = c * 2 * V; b = a + V; }
    else { a = p.rot + (c * V - half) * 2; b = a + V; }

    float cs[V], sn[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { cs[i] = 1.f; sn[i] = 0.f; }
    if (active && turned && first < p.H + p.KV) {
        const int64_t pos = p.positions[t];
        const bool known = pos >= 0 && pos < p.table_rows;
        const float* row = p.cos_sin + (known ? pos : 0) * p.rot + (p.interleaved ? c * V : a);
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const v4f x = *reinterpret_cast<const v4f*>(row + i), y = *reinterpret_cast<const v4f*>(row + half + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                cs[i + e] = known ? x[e] : __builtin_nanf("");   // a position that the table does not have: NaN, not a wrong angle
                sn[i + e] = known ? y[e] : __builtin_nanf("");
            }
        }
    }
    int64_t page = 0, at = 0;
    bool write = false;
    if (p.k_out == nullptr && last > p.H) {
        const int64_t slot = p.slots[t];
        write = slot >= 0 && slot < p.n_slots;
        page = write ? (int64_t)((uint32_t)slot / (uint32_t)p.page_size) : 0;
        at = write ? slot - page * p.page_size : 0;
    }
    const uint16_t* row = p.qkv + (int64_t)t * p.ld;
    for (int h = first; h < last; ++h) {
        Run<V> ra = {}, rb = {};
        if (active) {
            ra = load_run<V>(row + (int64_t)h * p.D + a);
            rb = load_run<V>(row + (int64_t)h * p.D + b);
        }
        if (h >= p.H + p.KV) {
            if (active && write) {
                uint16_t* o = p.v_pages + page * p.v_stride[0] + at * p.v_stride[1] + (h - p.H - p.KV) * p.v_stride[2];
                store_run<V>(o + a, ra);
                store_run<V>(o + b, rb);
            }
            continue;
        }
        float x[V], y[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            x[i] = head_to_f32<TYPE>((ra.w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
            y[i] = head_to_f32<TYPE>((rb.w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
        }
        const uint16_t* weight = h < p.H ? p.q_weight : p.k_weight;
        if (weight != nullptr) {   // (uniform)
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) ss = __builtin_fmaf(x[i], x[i], __builtin_fmaf(y[i], y[i], ss));
            for (int m = 1; m < (1 << lp_log); m <<= 1) ss += __shfl_xor(ss, m);
            const float r = 1.0f / __builtin_sqrtf(ss / (float)p.D + p.eps);
            Run<V> wa = {}, wb = {};
            if (active) {
                wa = load_run<V>(weight + a);
                wb = load_run<V>(weight + b);
            }
            const float more = p.gemma ? 1.0f : 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                x[i] = x[i] * r * (head_to_f32<TYPE>((wa.w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu) + more);
                y[i] = y[i] * r * (head_to_f32<TYPE>((wb.w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu) + more);
            }
        }
        if (turned) {
            if (p.interleaved) {
                // pairs (0, 1), (2, 3), ... of the first run, then of the second: angle i of the lane's V
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const float u = x[i], v = x[i + 1], f = y[i], g = y[i + 1];
                    const float c0 = cs[i >> 1], s0 = sn[i >> 1], c1 = cs[(V + i) >> 1], s1 = sn[(V + i) >> 1];
                    x[i] = u * c0 - v * s0; x[i + 1] = v * c0 + u * s0;
                    y[i] = f * c1 - g * s1; y[i + 1] = g * c1 + f * s1;
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float u = x[i], v = y[i];
                    x[i] = u * cs[i] - v * sn[i];
                    y[i] = v * cs[i] + u * sn[i];
                }
            }
        }
        if (!active) continue;
        uint16_t* o;
        if (h < p.H) o = p.q_out + ((int64_t)t * p.H + h) * p.D;
        else if (p.k_out != nullptr) o = p.k_out + ((int64_t)t * p.KV + (h - p.H)) * p.D;
        else if (write) o = p.k_pages + page * p.k_stride[0] + at * p.k_stride[1] + (h - p.H) * p.k_stride[2];
        else continue;
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            ra.w[i >> 1] = head_pack2<TYPE>(x[i], x[i + 1]);
            rb.w[i >> 1] = head_pack2<TYPE>(y[i], y[i + 1]);
        }
        store_run<V>(o + a, ra);
        store_run<V>(o + b, rb);
    }
}

template <int TYPE, int V>
hipError_t launch_v(const HeadRope& p, hipStream_t stream) {
    int lp_log = 0;
    while ((1 << lp_log) * 2 * V < p.D) ++lp_log;
    // without a cache the value heads are nobody's work
    const int heads = p.k_out != nullptr ? p.H + p.KV : p.H + 2 * p.KV;
    // Two heads a group, which then loads a token's angles once for both, where there are more threads than the chip holds:
    // 13056 tokens of 10 heads of 256 26.3 us, 29.3 with one and 28.1 with four; 816 of them 6.2 and 5.4 (graphs of the same call).
    const int per_group = ((int64_t)p.T * heads << lp_log) > 256 * 2048 ? 2 : 1;
    const int per_token = (heads + per_group - 1) / per_group;
    const int64_t groups = (int64_t)p.T * per_token;
    const int64_t threads = groups << lp_log;
    return enqueue(head_rope_kernel<TYPE, V>, dim3((uint32_t)((threads + 255) / 256)), dim3(256), stream, p, lp_log, per_group, per_token, groups);
}

}  // namespace

hipError_t launch_head_rope(const HeadRope& p, hipStream_t stream) {
    // runs of eight elements where half the rotated part and what lies behind it are whole runs (pairs of them), else of four
    const bool wide = (p.interleaved ? p.rot % 16 == 0 : (p.rot / 2) % 8 == 0) && (p.D - p.rot) % 16 == 0;
    if (p.type == HEAD_BF16) return wide ? launch_v<HEAD_BF16, 8>(p, stream) : launch_v<HEAD_BF16, 4>(p, stream);
    return wide ? launch_v<HEAD_F16, 8>(p, stream) : launch_v<HEAD_F16, 4>(p, stream);
}

}  // namespace phyai
