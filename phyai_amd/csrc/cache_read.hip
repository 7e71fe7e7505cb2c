// Keys and values of single tokens out of a paged cache in 8 bits: out[t, h, :] = code * 2^(b - 127) in the element type (what
// it holds of that exactly: widen.h; gfx950).  Sixteen codes a thread, one load and two stores; bound by memory, three bytes an element: 13056 tokens
// of one head of 256 in 6.0 us, 3.3 TB/s with the launch's 2 us in it; one token 1.6 us.
#include "fp8_device.h"
#include "layer_kernels.h"
#include "widen.h"

namespace phyai {
namespace {

template <int TYPE>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheRead p, uint32_t chunks, uint32_t items) {
    const uint32_t item = blockIdx.x * 256u + threadIdx.x;   // (token, key or value, head, chunk of sixteen)
    if (item >= items) return;
    const uint32_t part = item / chunks, t = part / (2u * (uint32_t)p.KV);
    const int chunk = (int)(item - part * chunks), head = (int)(part - t * (2u * (uint32_t)p.KV));
    const bool value = head >= p.KV;
    const int h = value ? head - p.KV : head;
    const int64_t slot = p.slots[t];
    v4i codes = {0, 0, 0, 0};
    uint32_t power = 127;
    if (slot >= 0 && slot < p.n_slots) {
        const int64_t page = (int64_t)((uint32_t)slot / (uint32_t)p.page_size), at = slot - page * p.page_size;
        const int64_t *s = value ? p.v_stride : p.k_stride, *b = value ? p.v_scale_stride : p.k_scale_stride;
        codes = *reinterpret_cast<const v4i*>((value ? p.v_pages : p.k_pages) + page * s[0] + at * s[1] + h * s[2] + chunk * 16);
        power = (value ? p.v_scales : p.k_scales)[page * b[0] + at * b[1] + h * b[2]];
    }
    if (power == 255) codes = v4i{(int)kNanCodes, (int)kNanCodes, (int)kNanCodes, (int)kNanCodes};
    v4i out[2];
    widen16<TYPE>(codes, power, out);
    uint16_t* o = (value ? p.v_out : p.k_out) + ((int64_t)t * p.KV + h) * p.D + chunk * 16;
    *reinterpret_cast<v4i*>(o) = out[0];
    *reinterpret_cast<v4i*>(o + 8) = out[1];
}

}  // namespace

hipError_t launch_cache_read(const CacheRead& p, hipStream_t stream) {
    const uint32_t chunks = (uint32_t)p.D / 16, items = (uint32_t)p.T * 2u * (uint32_t)p.KV * chunks;   // (less than 2^32, by the checks of its arguments)
    const dim3 grid((uint32_t)(((int64_t)items + 255) / 256));
    return p.type == HEAD_BF16 ? enqueue(cache_read_kernel<HEAD_BF16>, grid, dim3(256), stream, p, chunks, items)
                               : enqueue(cache_read_kernel<HEAD_F16>, grid, dim3(256), stream, p, chunks, items);
}

}  // namespace phyai
