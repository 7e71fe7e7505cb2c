// Attention of each sequence's new tokens over its pages (gfx950).  Row (i, g) of sequence b and key head h - new token i,
// query head h G + g, position kv_b - q_b + i - sees the keys j with lo <= j < hi (causal: hi = position + 1, window: lo =
// position - window + 1) and gets sum_j softmax_j(scale q.k_j) v_j, zero where it sees nothing.
//
// One pass over the keys with a running maximum m and sum l per row, in the base-2 domain.  Both products are computed
// transposed: S^T = K Q^T by v_mfma_f32_32x32x16, so a lane holds 16 of the 32 keys' scores of ONE row (the other 16 are in
// the lane 32 further) and the softmax needs a single exchange; P^T then lies in the registers exactly as the B operand of
// O^T = V^T P^T wants it, if V's keys are taken in the same order - which the transposing LDS read is free to do - and m,
// l and the rescaling of O are one value per lane.  O is only rescaled when a row's maximum grows by more than 2^8:
// probabilities stay below 2^8, which neither bf16, fp16 nor the fp32 sums mind.  A row that sees keys, but none with a score
// above -inf, is NaN, as its softmax is.
//
// Keys and values are copied from their pages straight into LDS.  16-byte chunk c of key r lies in slot c ^ f(r), with an
// f of its own for K (sixteen neighbouring keys, one chunk: sixteen bank groups) and for V (four keys, four chunks).
//
// A cache in 8 bits holds e4m3 codes and a power of two for each key and head: code times power is a value of the element type
// (widen.h), so its keys go through registers on their way to LDS, where they arrive in 16 bits, and
// everything behind that is the same.
//
// The kernels are templates: paged_attention.hip has those of plain 16-bit calls (MODE 0), attention_{bf16,f16,bf16_fp8,f16_fp8}.hip the others.
#pragma once

#include "fp8_device.h"
#include "layer_kernels.h"
#include "widen.h"

namespace phyai {
namespace {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef __attribute__((address_space(3))) uint32_t lds_u32;   // (through a generic pointer an access would count as one to memory too)
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8hf __attribute__((ext_vector_type(8)));

// What a kernel can do beside plain attention over 16-bit pages.
enum Mode : int {
    MODE_MORE = 1,   // prompts that causal rows see the whole of, shared leading keys
    MODE_FP8 = 2,    // pages in 8 bits
    MODE_CAP = 4,    // scores capped by a tanh
    MODE_WIDE = 8,   // the same with a cap that scores may be far below (above 256)
};

constexpr int ROWS = 32;               // rows of a wavefront's tile
constexpr float kNone = -__builtin_huge_valf();
constexpr float kLowest = -3.40282347e38f;   // maximum of a row part whose keys all have a score of -inf, where kNone is one that sees no key
constexpr float kRescaleAt = 8.0f;     // log2 of how far a row's maximum may grow before O is rescaled

// Sixteen bytes of zeros and of NaNs: where copies of keys that do not exist and of pages that do not exist come from.
__device__ __align__(16) const uint32_t kFill[2][2][4] = {{{0, 0, 0, 0}, {0, 0, 0, 0}},
                                                          {{0x7FC07FC0, 0x7FC07FC0, 0x7FC07FC0, 0x7FC07FC0}, {0x7E007E00, 0x7E007E00, 0x7E007E00, 0x7E007E00}}};

template <int TYPE>
__device__ __forceinline__ v16f mfma(v4i a, v4i b, v16f c) {
    if constexpr (TYPE == HEAD_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8hf, a), __builtin_bit_cast(v8hf, b), c, 0, 0, 0);
}
template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (TYPE == HEAD_BF16) return pack_bf16x2(a, b);
    else {   // (both at once: no instruction that writes half a register)
        typedef float two __attribute__((ext_vector_type(2)));
        typedef _Float16 pair __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(two{a, b}, pair));
    }
}
template <int TYPE>
__device__ __forceinline__ float to_f32(uint32_t h) {
    if constexpr (TYPE == HEAD_BF16) return __uint_as_float(h << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
// sum + both halves of w, one instruction
template <int TYPE>
__device__ __forceinline__ float add_pair(uint32_t w, float sum) {
    if constexpr (TYPE == HEAD_BF16) {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, w), __builtin_bit_cast(pair, 0x3F803F80u), sum, false);
    } else {
        typedef _Float16 pair __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(pair, w), __builtin_bit_cast(pair, 0x3C003C00u), sum, false);
    }
}
// the value of the lane 32 away, and this lane's: both orders are fine for max and sum
__device__ __forceinline__ float other_half_max(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float other_half_sum(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ int clamp_i(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

using Division = AttentionDivision;
using Plan = AttentionPlan;

// j / d for 0 <= j < 2^31 and a d known on the host: one high product (magic 0: d = 1).
__device__ __forceinline__ int divide(int j, Division d) { return d.magic == 0 ? j : (int)(__umulhi((uint32_t)j, d.magic) >> d.shift); }

// The sum over the lanes up to this one: four steps inside a row of sixteen lanes, two across rows.
template <int CTRL, int ROWS_OF = 0xF>
__device__ __forceinline__ int dpp_or_zero(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS_OF, 0xF, true); }
__device__ __forceinline__ int sum_up_to_lane(int v) {
    v += dpp_or_zero<0x111>(v);
    v += dpp_or_zero<0x112>(v);
    v += dpp_or_zero<0x114>(v);
    v += dpp_or_zero<0x118>(v);
    v += dpp_or_zero<0x142, 0xA>(v);   // lane 15's to the next row, 47's likewise
    v += dpp_or_zero<0x143, 0xC>(v);   // lane 31's to the upper half
    return v;
}

// Where a tile of `rows_per_tile` packed rows lies: the tiles of the sequences are numbered one sequence after another.
// Every wavefront finds it by itself, 64 sequences at a time.
struct Tile {
    int b, row0, rows, q_begin, q_len;
    int length, kv_len;   // keys as stated, which is where the tokens stand, and those of them that the table has room for
    int prompt;           // keys that every row sees of those that exist
};
template <int MODE>
__device__ __forceinline__ bool locate(const PagedAttention& p, int group, int rows_per_tile, int tile, Tile& o) {   // (rows_per_tile: a power of two)
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < p.B; base += 64) {
        const int b = base + lane;
        int q0 = 0, q1 = 0, kv = 0;
        if (b < p.B) {
            kv = p.kv_lens[b];
            q0 = clamp_i(p.q_offsets[b], 0, p.T);
            q1 = clamp_i(p.q_offsets[b + 1], q0, p.T);
        }
        const int tiles = ((q1 - q0) * group + rows_per_tile - 1) / rows_per_tile;
        const int upto = sum_up_to_lane(tiles);
        const uint64_t hit = __ballot(before + upto > tile);
        if (hit != 0) {
            const int l = __builtin_ctzll(hit);
            o.b = base + l;
            o.q_begin = __builtin_amdgcn_readlane(q0, l);
            o.q_len = __builtin_amdgcn_readlane(q1, l) - o.q_begin;
            o.rows = o.q_len * group;
            o.row0 = (tile - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(tiles, l))) * rows_per_tile;
            const int64_t most = (int64_t)p.table_width * p.page_size;
            kv = __builtin_amdgcn_readlane(kv, l);
            o.length = kv < 0 ? 0 : kv;
            o.kv_len = o.length > most ? (int)most : o.length;
            o.prompt = (MODE & MODE_MORE) && p.prefix_lens != nullptr ? clamp_i(p.prefix_lens[o.b], 0, o.kv_len) : 0;
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// ---- keys and values into LDS --------------------------------------------------------------------------------------
template <int DP>
struct Shape {
    static constexpr int ROW = 2 * DP;                 // bytes of a key in LDS
    static constexpr int CHUNKS = ROW / 16;            // 16-byte chunks of a key
    static constexpr int PER_COPY = 64 / CHUNKS;       // keys that one copy instruction brings
};
template <int DP>
__device__ __forceinline__ uint32_t k_swizzle(uint32_t r) { return DP == 64 ? (r >> 1) & 7u : r & 15u; }
template <int DP>
__device__ __forceinline__ uint32_t v_swizzle(uint32_t r) { return DP == 64 ? ((r >> 1) & 1u) * 4 : (r & 3u) * 4 | ((r >> 2) & 3u); }

__device__ __forceinline__ void copy16_from(const uint8_t* at, uint32_t lds_wave_base) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(at), "s"(lds_wave_base) : "memory", "m0");
}

// Where keys come from, for one sequence and key head.
struct Pool {
    const uint8_t *k, *v;              // the key head's first element in page 0
    const uint8_t *zero, *nan;
    const int32_t* table;              // the sequence's pages
    int64_t page_bytes, token_bytes;
    int n_pages, page_size, kv_len;
    Division by_page;
    int d_chunks;                      // 16-byte chunks of a key that exist
    bool neat;                         // runs of eight keys are neighbours in a page, and a key fills a row of LDS
    const uint8_t *k_scale, *v_scale;  // pages in 8 bits: the key head's first scale in page 0
    int64_t scale_page, scale_token;
};

// A wavefront's part of bringing blocks `begin`, begin + 1, ... of STEP keys into LDS: N keys of each, from key `row` of the
// block on.  Its lanes look the places of 64 such keys up at once, those of 64 / N blocks - page number, 64-bit offset,
// whether it is there at all - so that a block's copies cost little more than themselves (looked up for every block:
// 1000 cycles where the block's arithmetic takes 1500).  Page numbers go through LDS like the keys, asked for a turn ahead:
// a load of the compiler's own would wait for all copies in flight.
template <int DP, int STEP, int N>
struct Feeder {
    static constexpr int BLOCKS = 64 / N, PER_COPY = Shape<DP>::PER_COPY, COPIES = N / PER_COPY, ROW = Shape<DP>::ROW;
    static constexpr int RUN = 8;      // keys, neighbours in a page, that copies share an address for
    const Pool& s;
    const int begin, row;
    lds_u32* const ids;                // two times 64 words of LDS, this wavefront's
    int lo, hi, gone;                  // of the lane's key: its offset; its page does not exist
    uint64_t odd;                      // lanes whose key is gone
    uint32_t k_at, v_at;               // the lane's part of an address: of K and V, copy 0

    __device__ __forceinline__ Feeder(const Pool& pool, int first, int first_row, uint32_t* words)
        : s(pool), begin(first), row(first_row), ids((lds_u32*)words), lo(0), hi(0), gone(0), odd(0) {
        const uint32_t lane = threadIdx.x & 63, lr = lane / Shape<DP>::CHUNKS, lc = lane % Shape<DP>::CHUNKS;
        k_at = (lc ^ k_swizzle<DP>((uint32_t)row + lr)) << 4;
        v_at = (lc ^ v_swizzle<DP>((uint32_t)row + lr)) << 4;
    }
    // The lane's key.  In the place of one beyond the last, the first of the last key's run: no row sees what is copied
    // there, it only has to be in the cache, like all keys of that run (filled with zeros instead, by lanes that each have an
    // address of their own, a block took 3 us longer at 256 dims).
    __device__ __forceinline__ int key(int turn) const {
        const int lane = threadIdx.x & 63, j = (begin + turn * BLOCKS + lane / N) * STEP + row + lane % N;
        return j < s.kv_len ? j : (s.kv_len - 1) & ~(RUN - 1);
    }
    // The page numbers of a turn of BLOCKS blocks; to be waited for before look().
    __device__ __forceinline__ void ask(int turn) {
        const int page = divide(key(turn), s.by_page);
        copy4_to_lds<kBaseSettles>(reinterpret_cast<const uint8_t*>(s.table), (uint32_t)page * 4u,
                                   __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(ids + (turn & 1) * 64)));
    }
    __device__ __forceinline__ void look(int turn) {
        const int page = (int)((volatile lds_u32*)ids)[(turn & 1) * 64 + (threadIdx.x & 63)];
        const int j = key(turn);
        gone = page < 0 || page >= s.n_pages;
        const int64_t off = (int64_t)page * s.page_bytes + (int64_t)(j - divide(j, s.by_page) * s.page_size) * s.token_bytes;
        lo = (int)(uint32_t)off;
        hi = (int)(off >> 32);
        odd = __ballot(gone);
    }
    // Block `blk`, whose turn has been looked up, to the buffers at k_lds and v_lds: 2 COPIES copies.
    __device__ __forceinline__ void copy(int blk, uint32_t k_lds, uint32_t v_lds) {
        const int from = ((blk - begin) % BLOCKS) * N;   // the block's first lane
        if (s.neat && ((odd >> from) & (N == 64 ? ~0ull : (1ull << (N & 63)) - 1)) == 0) {
            const uint32_t token = (uint32_t)s.token_bytes, lr = (threadIdx.x & 63) / Shape<DP>::CHUNKS;
#pragma unroll
            for (int r = 0; r < N; r += RUN) {
                const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(lo, from + r) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, from + r) << 32;
                const uint8_t *k = s.k + at, *v = s.v + at;
#pragma unroll
                for (int i = 0; i < RUN; i += PER_COPY) {
                    const uint32_t to = (uint32_t)(row + r + i) * ROW, key = (lr + i) * token;
                    // (the swizzles of these keys are those of the first with the bits of r + i flipped)
                    copy16_to_lds<kBaseSettles>(k, (k_at ^ k_swizzle<DP>(r + i) << 4) + key, __builtin_amdgcn_readfirstlane(k_lds + to));
                    copy16_to_lds<kBaseSettles>(v, (v_at ^ v_swizzle<DP>(r + i) << 4) + key, __builtin_amdgcn_readfirstlane(v_lds + to));
                }
            }
            return;
        }
#pragma unroll 1   // (code that a cold instruction cache does not have to bring: most calls come here once)
        for (int t = 0; t < COPIES; ++t) {
            const int lane = from + t * PER_COPY + (int)(threadIdx.x & 63) / Shape<DP>::CHUNKS;
            const int64_t at = (int64_t)(uint32_t)__shfl(lo, lane) | (int64_t)__shfl(hi, lane) << 32;
            const int none = __shfl(gone, lane);
            const uint32_t kc = k_at ^ k_swizzle<DP>(t * PER_COPY) << 4, vc = v_at ^ v_swizzle<DP>(t * PER_COPY) << 4;
            const uint8_t* ka = (int)(kc >> 4) >= s.d_chunks ? s.zero : none ? s.nan : s.k + at + kc;
            const uint8_t* va = (int)(vc >> 4) >= s.d_chunks ? s.zero : none ? s.nan : s.v + at + vc;
            const uint32_t to = (uint32_t)(row + t * PER_COPY) * ROW;
            copy16_from(ka, __builtin_amdgcn_readfirstlane(k_lds + to));
            copy16_from(va, __builtin_amdgcn_readfirstlane(v_lds + to));
        }
    }
};

// The same part of a block for pages in 8 bits, through registers: what was asked for while a block was worked on is widened and
// put into LDS at its end (32 keys of 128 dims: 32 registers a lane).  The places of 64 keys are looked up at once, as above,
// their scales with them: 64 sequences of up to 8192 keys of 8 heads of 128 in 165 us, 4.3 TB/s, where the same keys in 16 bits take 267 at 5.3: what is left is the
// chain of a wavefront (codes, LDS, products) with eight of them a CU.  Widening costs the many-row kernel, in which each workgroup does it again, what it saves in bytes and
// more: 2048 tokens over 8192 keys 310 us for 255.
template <int DP, int TYPE, int STEP, int N>
struct Widener {
    static constexpr int LANES = DP / 16, PER = 64 / LANES, LOADS = N / PER, BLOCKS = 64 / N, ROW = Shape<DP>::ROW;   // lanes of a key, keys of a load
    static constexpr int RUN = 8;
    const Pool& s;
    const int begin, end, row;
    int page, lo, hi;                  // of the lane's key: its page in the turn to come; its offset
    uint32_t k_power, v_power, powers; // its scales as they were asked for; both, of the turn being stored
    uint32_t both[LOADS];              // the scales of the block being stored
    bool unknown;                      // a scale of the turn is a NaN
    uint64_t odd;                      // lanes whose key's page does not exist
    uint32_t at;                       // the lane's part of an address: its key of a load, its chunk
    uint32_t k_to, v_to;               // where its first chunk of load 0 goes in a buffer
    v4i k[LOADS], v[LOADS];            // of the block to come

    __device__ __forceinline__ Widener(const Pool& pool, int first, int last, int first_row)
        : s(pool), begin(first), end(last), row(first_row), page(0), lo(0), hi(0), k_power(0), v_power(0), powers(0), unknown(false), odd(0) {
        const uint32_t lane = threadIdx.x & 63, r = (uint32_t)row + lane / LANES, chunk = 2 * (lane % LANES) + turned();
        at = lane / LANES * (uint32_t)s.token_bytes + lane % LANES * 16;
        k_to = r * ROW + ((chunk ^ k_swizzle<DP>(r)) << 4);
        v_to = r * ROW + ((chunk ^ v_swizzle<DP>(r)) << 4);
    }
    // Of eight lanes, which LDS takes at once, four write their first eight values first and four the others: all in different banks.
    __device__ __forceinline__ static uint32_t turned() { return (threadIdx.x >> 2) & 1; }
    __device__ __forceinline__ int key(int turn) const {
        const int lane = threadIdx.x & 63, j = (begin + turn * BLOCKS + lane / N) * STEP + row + lane % N;
        return j < s.kv_len ? j : (s.kv_len - 1) & ~(RUN - 1);
    }
    __device__ __forceinline__ void ask(int turn) { page = s.table[divide(key(turn), s.by_page)]; }
    __device__ __forceinline__ void look(int turn) {
        const int j = key(turn), at = j - divide(j, s.by_page) * s.page_size;
        const bool gone = page < 0 || page >= s.n_pages;
        const int64_t off = (int64_t)page * s.page_bytes + (int64_t)at * s.token_bytes;
        lo = (int)(uint32_t)off;
        hi = (int)(off >> 32);
        odd = __ballot(gone);
        k_power = v_power = 127;
        if (!gone) {
            const int64_t scale = (int64_t)page * s.scale_page + (int64_t)at * s.scale_token;
            k_power = s.k_scale[scale];
            v_power = s.v_scale[scale];
        }
    }
    // Asks for block `blk` (below end; the blocks one after another, block `begin` after ask(0)).
    __device__ __forceinline__ void load(int blk) {
        const int nth = blk - begin, first = nth % BLOCKS * N;
        if (nth % BLOCKS == 0) {
            look(nth / BLOCKS);
            if (blk + BLOCKS < end) ask(nth / BLOCKS + 1);
        }
        if (s.neat && ((odd >> first) & (N == 64 ? ~0ull : (1ull << (N & 63)) - 1)) == 0) {
            // runs of eight keys share a base
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int from = first + i * PER / RUN * RUN, run = PER > RUN ? (int)((threadIdx.x & 63) / LANES) / RUN * RUN : 0;
                if constexpr (PER > RUN) {   // (two runs a load: each lane its own)
                    const int64_t off = (int64_t)(uint32_t)__shfl(lo, from + run) | (int64_t)__shfl(hi, from + run) << 32;
                    const int64_t to = off + at - (int64_t)run * s.token_bytes;
                    k[i] = *reinterpret_cast<const v4i*>(s.k + to);
                    v[i] = *reinterpret_cast<const v4i*>(s.v + to);
                } else {
                    const int64_t off = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(lo, from) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, from) << 32) +
                                        (int64_t)(i * PER % RUN) * s.token_bytes;
                    k[i] = *reinterpret_cast<const v4i*>(s.k + off + at);
                    v[i] = *reinterpret_cast<const v4i*>(s.v + off + at);
                }
            }
            return;
        }
        const int lane = threadIdx.x & 63, chunk = lane % LANES;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int from = first + i * PER + lane / LANES;
            const int64_t off = (int64_t)(uint32_t)__shfl(lo, from) | (int64_t)__shfl(hi, from) << 32;
            const int fill = chunk < s.d_chunks && ((odd >> from) & 1) ? (int)kNanCodes : 0;
            v4i a = {fill, fill, fill, fill}, b = a;
            if (chunk < s.d_chunks && !((odd >> from) & 1)) {
                a = *reinterpret_cast<const v4i*>(s.k + off + chunk * 16);
                b = *reinterpret_cast<const v4i*>(s.v + off + chunk * 16);
            }
            k[i] = a;
            v[i] = b;
        }
    }
    __device__ __forceinline__ void put(uint8_t* lds, uint32_t to, uint32_t power, const v4i& codes) const {
        v4i w[2];
        widen16<TYPE>(turned() ? v4i{codes[2], codes[3], codes[0], codes[1]} : codes, power, w);
        *reinterpret_cast<v4i*>(lds + to) = w[0];
        *reinterpret_cast<v4i*>(lds + (to ^ 16u)) = w[1];
    }
    // The block asked for last, which is `blk`, into the buffers, piece by piece of 2 LOADS (work to be done beside matrix
    // products); its scales first.  Codes of a scale that is a NaN become NaNs.
    static constexpr int PIECES = 2 * LOADS;
    __device__ __forceinline__ void scales(int blk) {
        if ((blk - begin) % BLOCKS == 0) {
            powers = k_power | v_power << 8;
            unknown = __any(k_power == 255 || v_power == 255);
        }
        const int from = (blk - begin) % BLOCKS * N + (int)(threadIdx.x & 63) / LANES;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) both[i] = (uint32_t)__builtin_amdgcn_ds_bpermute((from + i * PER) * 4, (int)powers);
        if (unknown) {   // (apart, so that the pieces are without a branch)
            constexpr int NANS = (int)kNanCodes;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                if ((both[i] & 255u) == 255u) k[i] = v4i{NANS, NANS, NANS, NANS};
                if ((both[i] >> 8) == 255u) v[i] = v4i{NANS, NANS, NANS, NANS};
            }
        }
    }
    __device__ __forceinline__ void piece(int p, uint8_t* k_lds, uint8_t* v_lds) const {
        const int i = p >> 1;
        // (the swizzles of these keys are those of load 0's with the bits of i PER flipped)
        if ((p & 1) == 0) put(k_lds, (k_to ^ k_swizzle<DP>(i * PER) << 4) + i * PER * ROW, both[i] & 255u, k[i]);
        else put(v_lds, (v_to ^ v_swizzle<DP>(i * PER) << 4) + i * PER * ROW, both[i] >> 8, v[i]);
    }
    __device__ __forceinline__ void store(int blk, uint8_t* k_lds, uint8_t* v_lds) {
        asm volatile("" ::: "memory");
        scales(blk);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) piece(p, k_lds, v_lds);
        asm volatile("" ::: "memory");
    }
};

// A row of the tile: which token and head it is and which keys it sees.
struct Row {
    int token, head, lo, hi;
    bool valid;
};

// ---- one block of 32 keys against 32 rows ----------------------------------------------------------------------------
template <int DP>
struct State {
    v16f o[DP / 32];   // O^T: value dim 32 b + 8 (i / 4) + 4 (lane / 32) + i % 4 of row lane % 32
    float m, l;        // running maximum (scaled, base 2) and this lane's half of the sum
};

template <int TYPE>
__device__ __forceinline__ bool any_special(uint32_t w) {
    constexpr uint32_t E = TYPE == HEAD_BF16 ? 0x7F80u : 0x7C00u;
    return (w & E) == E || (w & (E << 16)) == (E << 16);
}
template <int TYPE>
__device__ __forceinline__ uint32_t without_special(uint32_t w) {
    constexpr uint32_t E = TYPE == HEAD_BF16 ? 0x7F80u : 0x7C00u;
    if ((w & E) == E) w &= 0xFFFF0000u;
    if ((w & (E << 16)) == (E << 16)) w &= 0xFFFFu;
    return w;
}
// A probability of zero times an infinity or a NaN is a NaN.  In a tile that some rows see only part of, such values are
// taken out of V as it lands (each wavefront looks through the `keys` keys it has copied itself and whatever lies behind them;
// true if there were any among the keys), and add_specials gives them to the rows that see their key after the last tile.
template <int DP, int TYPE, int N>
__device__ __forceinline__ bool clean_values(uint8_t* v, int keys) {
    bool special = false;
    constexpr int PER = N * Shape<DP>::ROW / 1024, AT_ONCE = PER < 4 ? PER : 4;   // 16 bytes of a lane: in all, read together
#pragma unroll 1
    for (int x = (threadIdx.x & 63) * 16; x < N * Shape<DP>::ROW; x += AT_ONCE * 1024) {
        v4i f[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) f[k] = *reinterpret_cast<const v4i*>(v + x + k * 1024);
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            bool any = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) any |= any_special<TYPE>((uint32_t)f[k][i]);
            if (any) {
#pragma unroll
                for (int i = 0; i < 4; ++i) f[k][i] = (int)without_special<TYPE>((uint32_t)f[k][i]);
                *reinterpret_cast<v4i*>(v + x + k * 1024) = f[k];
            }
            special |= any && (x + k * 1024) / Shape<DP>::ROW < keys;
        }
    }
    return __any(special);
}
// Infinities and NaNs of keys first .. last - 1, from their pages: add(q, e, value) is for value dim 8 q + 4 (lane / 32) + e of the lane's row.
// (A page that does not exist has made its scores NaN already.)
template <int DP, int TYPE, int MODE, typename Add>
__device__ __forceinline__ void special_values(const Pool& s, int first, int last, int d_end, int lo, int hi, Add add) {
    const int half = (threadIdx.x & 63) >> 5;
    constexpr int AT_ONCE = DP == 64 || (MODE & MODE_FP8) ? 8 : 16;   // loads on their way together (16 of 8 bits: masks spilled at 128 dims)
    last = last < s.kv_len ? last : s.kv_len;
#pragma unroll 1
    for (int j = first; j < last; ++j) {
        const int at = divide(j, s.by_page), page = s.table[at];
        if (page < 0 || page >= s.n_pages || j < lo || j >= hi) continue;
        const uint8_t* v = s.v + (int64_t)page * s.page_bytes + (int64_t)(j - at * s.page_size) * s.token_bytes;
        uint32_t power = 0;
        if constexpr (MODE & MODE_FP8) power = s.v_scale[(int64_t)page * s.scale_page + (int64_t)(j - at * s.page_size) * s.scale_token];
#pragma unroll 1
        for (int q0 = 0; q0 < DP / 8; q0 += AT_ONCE) {
            uint2 w[AT_ONCE];
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) {
                const int d = 8 * (q0 + q) + 4 * half;
                w[q] = make_uint2(0, 0);
                if (d < d_end) {
                    if constexpr (MODE & MODE_FP8) w[q].x = *reinterpret_cast<const uint32_t*>(v + d);
                    else w[q] = *reinterpret_cast<const uint2*>(v + 2 * d);
                }
            }
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) {
                if constexpr (MODE & MODE_FP8) {
                    const uint32_t codes = power == 255 && 8 * (q0 + q) + 4 * half < d_end ? kNanCodes : w[q].x;
                    w[q] = make_uint2(widen2<TYPE>(codes, __uint_as_float(power << 23), false), widen2<TYPE>(codes, __uint_as_float(power << 23), true));
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t h = ((e & 2 ? w[q].y : w[q].x) >> (16 * (e & 1))) & 0xFFFFu;
                    if (any_special<TYPE>(h)) add(q0 + q, e, to_f32<TYPE>(h));
                }
            }
        }
    }
}
// O in LDS: a row of it for each of a wavefront's rows, OLD floats apart.
template <int DP>
constexpr int OLD = DP + 4;
template <int DP>
__device__ __forceinline__ float* row_of_sums(float* sums) { return sums + (threadIdx.x & 31) * OLD<DP> + 4 * ((threadIdx.x & 63) >> 5); }
template <int DP>
__device__ __forceinline__ void put_sums(const State<DP>& st, float* row) {
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v4f v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = st.o[b][4 * i + e];
            *reinterpret_cast<v4f*>(row + 32 * b + 8 * i) = v;
        }
}
template <int DP>
__device__ __forceinline__ void get_sums(State<DP>& st, const float* row) {
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const v4f v = *reinterpret_cast<const v4f*>(row + 32 * b + 8 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[b][4 * i + e] = v[e];
        }
}
// Those of the blocks of STEP keys from begin up to end that some rows see only part of.  O goes through LDS meanwhile (`sums`: the wavefront's, which nobody
// reads any more): in registers, an element of O each in the code, their masks spilled up to 270 scalars into vector registers that the loop over
// the keys wants, and 8 to 24 bytes of scratch in the kernels of 8 bits and 128 dims (at 256, up to 556 with selects for the branches).  16 x 816 tokens
// of 256 dims in half precision 68.5 to 67.6 us, 2048 over 8192 keys of 128 dims 257 to 252.  64 dims have the registers, and 30.5 us for 29.6 by way of LDS.
// Where there is a NaN in every page: 16 x 816 causal tokens of 256 dims 767 to 635 us, but 2048 over 8192 keys of 128 dims 357 to 389
// and 64 of up to 8192 keys 296 to 319.
template <int DP, int TYPE, int MODE, int STEP>
__device__ __forceinline__ void add_specials(State<DP>& st, float* sums, const Pool& s, int begin, int end, int all_lo, int all_hi, int d_end, int lo, int hi) {
    auto blocks = [&](auto add) {
#pragma unroll 1
        for (int blk = begin; blk < end; ++blk)
            if (blk * STEP < all_lo || blk * STEP + STEP > all_hi) special_values<DP, TYPE, MODE>(s, blk * STEP, blk * STEP + STEP, d_end, lo, hi, add);
    };
    if constexpr (DP == 64) {
        blocks([&](int q, int e, float v) { st.o[(q >> 2) & 1][4 * (q & 3) + e] += v; });
    } else {
        float* row = row_of_sums<DP>(sums);
        put_sums<DP>(st, row);
        blocks([&](int q, int e, float v) { row[8 * q + e] += v; });
        get_sums<DP>(st, row);
    }
}

// The pieces of a block's work; kbuf, vbuf: the tile's buffers, row: the block's first key in them.
// Operand K: chunks 2 kk + half of key lane % 32, an xor with a constant below 256 bytes, an offset above.
template <int DP>
__device__ __forceinline__ v4i read_k(const uint8_t* kbuf, int row, int kk) {
    using S = Shape<DP>;
    const int lane = threadIdx.x & 63;
    const uint32_t r = (uint32_t)(lane & 31), a0 = r * S::ROW + (((uint32_t)(lane >> 5) ^ k_swizzle<DP>(r)) << 4);
    return *reinterpret_cast<const v4i*>(kbuf + row * S::ROW + (a0 ^ ((uint32_t)(kk & 7) << 5)) + (kk >> 3) * 256);
}
// Operand V^T, value dims 32 b .. and keys 16 e ..: lane (16 g + t) asks for key 4 half + t / 4 of a run of eight and dims 16 (g & 1)
// + 4 (t & 3) .. and gets four keys of one dim.
template <int DP>
__device__ __forceinline__ v4i read_v(const uint8_t* vbuf, int row, int b, int e) {
    using S = Shape<DP>;
    const int lane = threadIdx.x & 63;
    const uint32_t key0 = (uint32_t)(4 * (lane >> 5) + ((lane & 15) >> 2)), chunk0 = (uint32_t)((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    const uint32_t v0 = key0 * S::ROW + ((chunk0 ^ v_swizzle<DP>(key0)) << 4) + (lane & 1) * 8;
    const uint8_t* vr = vbuf + row * S::ROW;
    union { v4s h[2]; v4i v; } f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        // eight keys further the swizzle has bit 1 of the chunk flipped (two chunks of four bits at DP = 64: none)
        const uint32_t flip = ((uint32_t)(b & 3) << 6) ^ (DP != 64 && x ? 32u : 0u);
        f.h[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(vr + (v0 ^ flip) + (16 * e + 8 * x) * S::ROW + (b >> 2) * 256));
    }
    return f.v;
}
__device__ __forceinline__ void mask_scores(v16f& s, int j0, int lo, int hi) {
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int j = j0 + 8 * (i >> 2) + 4 * half + (i & 3);
        s[i] = j >= lo && j < hi ? s[i] : kNone;
    }
}
template <int NB>
__device__ __forceinline__ float max_score(const v16f (&s)[NB]) {
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 16 * NB; ++i) mx = __builtin_fmaxf(mx, s[i / 16][i % 16]);
    return other_half_max(mx);
}
// The row's maximum may have become `mx` (scaled): does any row of the wavefront need its O rescaled, and that.
__device__ __forceinline__ bool maximum_rises(float m, float mx) { return __any(mx > m + kRescaleAt); }
template <int DP>
__device__ __forceinline__ void raise_maximum(State<DP>& st, float mx) {
    const float m = __builtin_fmaxf(st.m, mx);
    const float a = m == kNone ? 1.0f : __builtin_amdgcn_exp2f(st.m - m);   // (0 the first time, when O and l are zero)
    st.l *= a;
    if (!__all(st.m == kNone)) {   // (the first keys of all find only zeros there)
#pragma unroll
        for (int b = 0; b < DP / 32; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) st.o[b][i] *= a;
    }
    st.m = m;
}
// A score s to cap tanh(s / cap) in base 2: with e = 2^(s by), by = 2 log2(e) scale / cap, tanh = 1 - 2 / (e + 1), exact where the
// power over- or underflows.  Kept is -1 / (e + 1), from which the score (less a maximum) is one multiply-add: times 2 cap log2(e), and cap log2(e)
// left out, which all scores have in common.  Off by some 2^-22 of cap in all, which is what the score's own rounding is.
// Four instructions a score, two of them at half the rate, and not hidden behind the products: 2048 tokens of 32 heads of 128 over 8192
// keys 354 us for 255, 16 x 816 of 8 heads of 256 98 for 76.
struct Cap {
    float by, most;
};
template <int N>
__device__ __forceinline__ void cap_some(v16f& s, int first, Cap c) {
#pragma unroll
    for (int i = first; i < first + N; ++i) s[i] = -__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[i] * c.by) + 1.0f);
}
// That rounding is 2^-22 of the cap also for scores far below it, which large caps are there to leave alone.  So for those: with y = s by,
// by = scale / cap, s times the first terms of tanh(y) / y = 1 - y^2 / 3 + ..., the one left out 6e-8 of it at the border, and beyond
// cap / scale times 1 - 2 / (e^2y + 1).  The result is a score as it was.  Three times the instructions: only in kernels of its own,
// and only in those for few rows: 64 sequences of up to 8192 keys in 8 bits 210 us where a cap of 50 takes 170, but 2048 tokens over 8192 keys 770 for 396 (16 bits 634 for
// 354), 16 x 816 of 256 dims 160 for 98, 64 tokens behind 8192 shared keys 94 for 39 without a cap.
__device__ __forceinline__ void cap_wide(v16f& s, Cap c) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float y = s[i] * c.by, u = y * y;
        float f = __builtin_fmaf(u, -1382.0f / 155925, 62.0f / 2835);
        f = __builtin_fmaf(u, f, -17.0f / 315);
        f = __builtin_fmaf(u, f, 2.0f / 15);
        f = __builtin_fmaf(u, f, -1.0f / 3);
        const float small = __builtin_fmaf(s[i] * u, f, s[i]);
        const float t = 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(__builtin_fabsf(y) * 2.8853900817779268f) + 1.0f);
        s[i] = __builtin_fabsf(y) > 0.4f ? __builtin_copysignf(t * c.most, s[i]) : small;
    }
}
// Scores to probabilities, as the second product's operand.  The sum is of the rounded ones, those that the product uses:
// their common error cancels.
template <int TYPE>
__device__ __forceinline__ float probabilities(v16f& s, v4i (&pf)[2], float m, float c) {
    const float base = m == kNone ? 0.f : m;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -base));
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = pack2<TYPE>(s[8 * e + 2 * i], s[8 * e + 2 * i + 1]);
            pf[e][i] = (int)w;
            sum[e] = add_pair<TYPE>(w, sum[e]);
        }
    return sum[0] + sum[1];
}

// The keys from 32 NB blk on, NB blocks of 32 a step.  top(step) makes a step's keys available and says where they are (null:
// no row of the wavefront sees any of it); all rows see whole_lo .. whole_hi.  The loop inside touches O by matrix products
// alone; a step that raises a maximum leaves it, is finished outside, and the loop goes on behind it.  (With the rescaling
// inside, 256 dims' O moved from the accumulation registers and back for every block: 256 instructions beside 32 products.)
// beside: work of a step that has nothing to do with its keys, done between the products with its values, a piece at a time, and all at
// once where the maximum rises.  (No step is left out then, also where a wavefront's rows see nothing of it: a way round the products
// made the compiler keep O in memory.)
struct Nothing {
    static constexpr int PIECES = 0;
    __device__ __forceinline__ void start(int) const {}
    __device__ __forceinline__ void piece(int) const {}
};
template <typename Beside>
__device__ __forceinline__ void all_pieces(const Beside& beside, int step) {
    if constexpr (Beside::PIECES > 0) {
        beside.start(step);
#pragma unroll
        for (int p = 0; p < Beside::PIECES; ++p) beside.piece(p);
    }
}
template <int DP, int TYPE, int NB, int MODE, typename Top, typename Beside>
__device__ __forceinline__ void attend_steps(State<DP>& st, const v4i* qf, int step, int end, const Row& row, int whole_lo, int whole_hi, float c, Cap cap, Top top,
                                             const Beside& beside) {
    using S = Shape<DP>;
    // V is read while the scores are turned into probabilities; as much of it as there are registers for
    constexpr int EARLY = DP == 64 || (DP == 128 && (MODE & MODE_FP8) && (MODE & MODE_CAP)) ? 2 : NB == 1 || DP == 256 ? 4 : 2;
    while (step < end) {
        v16f s[NB];
        float mx = kNone;
        const uint8_t *k = nullptr, *v = nullptr;
        bool rises = false;
#pragma unroll 1
        for (; step < end; ++step) {
            k = top(step);
            if constexpr (Beside::PIECES == 0) {
                if (k == nullptr) continue;
            }
            v = k + NB * 32 * S::ROW;
            v4i kf[DP / 16], vf[EARLY][2], pf[NB][2];
            // a block's reads all together, during the products of the one before: left to itself the compiler reads two,
            // waits, multiplies, and waits again
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) kf[kk] = read_k<DP>(k, 0, kk);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[n][i] = 0.f;
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {
                    s[n] = mfma<TYPE>(kf[kk], qf[kk], s[n]);
                    if constexpr ((MODE & MODE_CAP) != 0) {   // the scores of the block before, meanwhile
                        if (n > 0) cap_some<256 / DP>(s[n > 0 ? n - 1 : 0], kk * (256 / DP), cap);
                    }
                    if (n + 1 < NB) kf[kk] = read_k<DP>(k, 32 * (n + 1), kk);
                }
                if (n + 1 == NB) {
#pragma unroll
                    for (int b = 0; b < EARLY; ++b)
#pragma unroll
                        for (int e = 0; e < 2; ++e) vf[b][e] = read_v<DP>(v, 0, b, e);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (MODE & MODE_CAP) cap_some<16>(s[NB - 1], 0, cap);
            if constexpr ((MODE & MODE_WIDE) != 0) {
#pragma unroll
                for (int n = 0; n < NB; ++n) cap_wide(s[n], cap);
            }
            const int j0 = step * (32 * NB);
            if (j0 < whole_lo || j0 + 32 * NB > whole_hi) {
#pragma unroll
                for (int n = 0; n < NB; ++n) mask_scores(s[n], j0 + 32 * n, row.lo, row.hi);
            }
            mx = max_score<NB>(s) * c;
            rises = maximum_rises(st.m, mx);
            if (rises) break;
            if constexpr (Beside::PIECES > 0) beside.start(step);
#pragma unroll
            for (int n = 0; n < NB; ++n) st.l += probabilities<TYPE>(s[n], pf[n], st.m, c);
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        st.o[b] = mfma<TYPE>(n == 0 && b < EARLY ? vf[b % EARLY][e] : read_v<DP>(v, 32 * n, b, e), pf[n][e], st.o[b]);
                        if constexpr (Beside::PIECES > 0) {
                            constexpr int EACH = NB * (DP / 16) / Beside::PIECES;
                            const int at = (n * (DP / 32) + b) * 2 + e;
                            if (at % EACH == 0) beside.piece(at / EACH);
                        }
                    }
        }
        if (!rises) break;
        all_pieces(beside, step);
        raise_maximum<DP>(st, mx);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            v4i pf[2];
            st.l += probabilities<TYPE>(s[n], pf, st.m, c);
#pragma unroll
            for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e) st.o[b] = mfma<TYPE>(read_v<DP>(v, 32 * n, b, e), pf[e], st.o[b]);
        }
        ++step;
    }
}

template <int MODE>
__device__ __forceinline__ Row row_of(const PagedAttention& p, const Tile& t, const Plan& g, int kv_head, int row) {
    Row r;
    r.valid = row < t.rows;
    const int i = r.valid ? divide(row, g.group) : 0;
    r.token = t.q_begin + i;
    r.head = kv_head * g.group_size + (r.valid ? row - i * g.group_size : 0);
    const int position = t.length - t.q_len + i;
    r.hi = !r.valid ? 0 : p.causal ? clamp_i(position + 1, 0, t.kv_len) : t.kv_len;
    r.lo = p.window > 0 && position >= p.window ? position - p.window + 1 : 0;
    if constexpr (MODE & MODE_MORE) {
        if (r.valid && r.hi < t.prompt) r.hi = t.prompt;
        r.lo = r.lo > g.shared ? r.lo : g.shared;
    }
    return r;
}
// First and last + 1 key that any of the rows row0 .. row1 sees, and that all of them see.
template <int MODE>
__device__ __forceinline__ void span_of(const PagedAttention& p, const Tile& t, const Plan& g, int row0, int row1, int& lo, int& hi, int& all_lo, int& all_hi) {
    const int i0 = divide(row0, g.group), i1 = divide(row1, g.group);
    const int position0 = t.length - t.q_len + i0, position1 = t.length - t.q_len + i1;
    lo = p.window > 0 && position0 >= p.window ? position0 - p.window + 1 : 0;
    hi = p.causal ? clamp_i(position1 + 1, 0, t.kv_len) : t.kv_len;
    all_lo = p.window > 0 && position1 >= p.window ? position1 - p.window + 1 : 0;
    all_hi = p.causal ? clamp_i(position0 + 1, 0, t.kv_len) : t.kv_len;
    if constexpr (MODE & MODE_MORE) {
        hi = hi > t.prompt ? hi : t.prompt;
        all_hi = all_hi > t.prompt ? all_hi : t.prompt;
        lo = lo > g.shared ? lo : g.shared;
        all_lo = all_lo > g.shared ? all_lo : g.shared;
        if (lo >= hi) lo = hi = 0;
    } else lo = lo < hi ? lo : hi;
}

template <int DP>
__device__ __forceinline__ void load_q(const PagedAttention& p, const Row& r, v4i* qf) {
    const int half = (threadIdx.x & 63) >> 5;
    const uint16_t* q = p.q + (int64_t)r.token * p.q_token + (int64_t)r.head * p.q_head;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
        const int d = 16 * kk + 8 * half;
        v4i v = {0, 0, 0, 0};
        if (r.valid && d < p.D) v = *reinterpret_cast<const v4i*>(q + d);
        qf[kk] = v;
    }
}

template <int DP, int TYPE, int MODE>
__device__ __forceinline__ Pool make_pool(const PagedAttention& p, const Tile& t, int kv_head, const Plan& g) {
    Pool s;
    constexpr int SIZE = MODE & MODE_FP8 ? 1 : 2;
    s.k = static_cast<const uint8_t*>(p.k_pages) + kv_head * p.kv_stride[2] * SIZE;
    s.v = static_cast<const uint8_t*>(p.v_pages) + kv_head * p.kv_stride[2] * SIZE;
    s.zero = reinterpret_cast<const uint8_t*>(kFill[0][0]);
    s.nan = reinterpret_cast<const uint8_t*>(kFill[1][TYPE]);
    s.page_bytes = p.kv_stride[0] * SIZE;
    s.token_bytes = p.kv_stride[1] * SIZE;
    s.n_pages = (int)p.n_pages;
    s.page_size = p.page_size;
    s.kv_len = t.kv_len;
    s.by_page = g.page;
    s.table = p.table + (int64_t)t.b * p.table_ld;
    s.d_chunks = p.D * SIZE / 16;
    s.neat = p.D == DP && p.page_size % 8 == 0;
    if constexpr (MODE & MODE_FP8) {
        s.k_scale = p.k_scales + kv_head * p.scale_stride[2];
        s.v_scale = p.v_scales + kv_head * p.scale_stride[2];
        s.scale_page = p.scale_stride[0];
        s.scale_token = p.scale_stride[1];
    }
    return s;
}

// ---- few rows: the wavefronts of a workgroup, and several workgroups, share the keys of 32 rows --------------------------
// Each wavefront has 32 keys in LDS to itself and waits for nobody until the end: it copies a block, waits, multiplies,
// copies the next; the others' copies are under way meanwhile (twice as many wavefronts beat two stages for each).  Then the
// workgroup's states meet in LDS; with more than one workgroup per tile they leave unnormalised sums for
// attend_join_kernel.  Many sequences: bound by memory, 64 x 8192 keys of 8 heads of 128 in 253 us, 5.1 TB/s.  Few: by the chain of
// sequence, page numbers, keys (64 bytes a cycle into a CU), products, sums: 50 tokens over 866 keys of 256 dims 14.4 us, 3 to 4 of them the join.
template <int DP, int WAVES_OF>
struct SplitShape {
    static constexpr int WAVES = WAVES_OF;
    static constexpr int STAGE = 2 * 32 * Shape<DP>::ROW;
    static constexpr int WAVE_BYTES = STAGE > 32 * OLD<DP> * 4 ? STAGE : 32 * OLD<DP> * 4;
    static constexpr int LDS = WAVES * (WAVE_BYTES + 512 + 256 + 128);   // and page numbers, maxima and sums, shares
};
template <int DP>
constexpr int SPLIT_WAVES = DP == 256 ? 4 : 8;   // of a workgroup that has a CU to itself (64 dims: two fit)
// What a row's O is divided by, inverted: a sum of zero is a row's that sees nothing, or only scores of -inf.
__device__ __forceinline__ float one_over(float sum, bool sees) { return sum != 0.f ? 1.0f / sum : sees ? __builtin_nanf("") : 0.f; }
// How much of a state with maximum m belongs into one with the larger maximum `all` (m = -inf: it has seen nothing, or NaN).
__device__ __forceinline__ float share(float m, float l, float all) { return m == kNone ? (l != l ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(m - all); }

// The rows of all sequences against the shared leading keys, which the first sequence's pages hold.
__device__ __forceinline__ bool locate_shared(const PagedAttention& p, const Plan& g, int rows_per_tile, int tile, Tile& o) {
    const int q0 = clamp_i(p.q_offsets[0], 0, p.T), q1 = clamp_i(p.q_offsets[p.B], q0, p.T);
    o.b = 0;
    o.q_begin = q0;
    o.q_len = q1 - q0;
    o.rows = o.q_len * g.group_size;
    o.row0 = tile * rows_per_tile;
    o.length = o.kv_len = g.shared;
    o.prompt = 0;
    return o.row0 < o.rows;
}
// A wavefront's row of such a tile, whose sequence tells which keys it sees, and the spans of all of them.
__device__ __forceinline__ Row row_of_shared(const PagedAttention& p, const Tile& t, const Plan& g, int kv_head, int first, int& lo, int& hi, int& all_lo, int& all_hi) {
    const int lane = threadIdx.x & 63, row = first + (lane & 31);
    Row r;
    r.valid = row < t.rows;
    const int i = r.valid ? divide(row, g.group) : 0;
    r.token = t.q_begin + i;
    r.head = kv_head * g.group_size + (r.valid ? row - i * g.group_size : 0);
    // how many sequences end at or before the row's token, 64 of them and a token at a time
    const int last = first + ROWS < t.rows ? first + ROWS - 1 : t.rows - 1;
    const int i0 = divide(first < t.rows ? first : 0, g.group), i1 = first < t.rows ? divide(last, g.group) : -1;   // (none: no row is there)
    int b = 0;
    for (int base = 0; base < p.B; base += 64) {
        const int end = base + lane < p.B ? p.q_offsets[base + lane + 1] : 0x7FFFFFFF;
        int seen = 0;
        for (int x = i0; x <= i1; ++x) {
            seen = __popcll(__ballot(end <= t.q_begin + x));
            if (i == x) b += seen;
        }
        if (seen < 64) break;   // (the last token's sequence is among these)
    }
    b = b < p.B ? b : p.B - 1;
    const int q0 = clamp_i(p.q_offsets[b], 0, p.T), q1 = clamp_i(p.q_offsets[b + 1], q0, p.T);
    const int length = p.kv_lens[b] < 0 ? 0 : p.kv_lens[b], prompt = p.prefix_lens != nullptr ? p.prefix_lens[b] : 0;
    const int position = length - (q1 - q0) + (r.token - q0);
    int end = p.causal ? clamp_i(position + 1, 0, length) : length;
    end = end > prompt ? end : prompt < length ? prompt : length;
    r.hi = !r.valid ? 0 : end < t.kv_len ? end : t.kv_len;
    r.lo = p.window > 0 && position >= p.window ? position - p.window + 1 : 0;
    // (a row that is not there widens nothing)
    const bool sees = r.lo < r.hi;
    lo = sees ? r.lo : 0x7FFFFFFF;
    hi = sees ? r.hi : 0;
    all_lo = r.valid ? r.lo : 0;
    all_hi = r.valid ? r.hi : 0x7FFFFFFF;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        lo = min(lo, __shfl_xor(lo, x));
        hi = max(hi, __shfl_xor(hi, x));
        all_lo = max(all_lo, __shfl_xor(all_lo, x));
        all_hi = min(all_hi, __shfl_xor(all_hi, x));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    return r;
}

template <int DP, int TYPE, int MODE, int WAVES_OF>
__device__ __forceinline__ void attend_split(const PagedAttention& p, const Plan& g, float* __restrict__ part, uint8_t* lds, int tile, int kv_head, int z) {
    using S = Shape<DP>;
    using X = SplitShape<DP, WAVES_OF>;
    auto ids = reinterpret_cast<uint32_t (*)[2][64]>(lds + X::WAVES * X::WAVE_BYTES);
    auto ml = reinterpret_cast<float (*)[32][2]>(lds + X::WAVES * (X::WAVE_BYTES + 512));
    auto weight = reinterpret_cast<float (*)[32]>(lds + X::WAVES * (X::WAVE_BYTES + 512 + 256));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (the shared keys' splits come first)
    const bool shared = (MODE & MODE_MORE) != 0 && z < g.shared_splits;
    Tile t;
    Row row;
    int lo, hi, all_lo, all_hi;
    if (shared) {   // (here and below: the same for the whole workgroup)
        if (tile >= g.shared_tiles || !locate_shared(p, g, ROWS, tile, t)) return;
        row = row_of_shared(p, t, g, kv_head, t.row0, lo, hi, all_lo, all_hi);
        if (lo >= hi) lo = hi = 0;
    } else {
        if (!locate<MODE>(p, g.group_size, ROWS, tile, t)) return;
        row = row_of<MODE>(p, t, g, kv_head, t.row0 + (lane & 31));
        span_of<MODE>(p, t, g, t.row0, t.row0 + ROWS < t.rows ? t.row0 + ROWS - 1 : t.rows - 1, lo, hi, all_lo, all_hi);
    }
    const int b0 = lo / 32, n = (hi + 31) / 32 - b0;   // blocks of 32 keys (none: hi = lo = 0)
    // even shares, the first ones a block larger
    const int of = MODE & MODE_MORE ? (shared ? g.shared_splits : g.splits - g.shared_splits) : g.splits;
    const int me = (z - (shared || !(MODE & MODE_MORE) ? 0 : g.shared_splits)) * X::WAVES + wave;
    const int each = shared ? divide(n, g.shared_workers) : divide(n, g.workers), rest = n - each * of * X::WAVES;
    const int begin = b0 + me * each + (me < rest ? me : rest), end = begin + each + (me < rest ? 1 : 0);
    const Pool pool = make_pool<DP, TYPE, MODE>(p, t, kv_head, g);
    const float c = MODE & MODE_CAP ? 2.0f * p.cap : p.scale * 1.4426950408889634f;
    const Cap cap = {p.cap_by, p.cap_most};

    State<DP> st;
    st.m = kNone;
    st.l = 0.f;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[b][i] = 0.f;
    uint8_t* mine = lds + wave * X::WAVE_BYTES;
    bool special = false;
    if constexpr (MODE & MODE_FP8) {
        if (begin < end) {
            Widener<DP, TYPE, 32, 32> feed(pool, begin, end, 0);
            feed.ask(0);
            v4i qf[DP / 16];
            load_q<DP>(p, row, qf);
            feed.load(begin);
            attend_steps<DP, TYPE, 1, MODE>(st, qf, begin, end, row, all_lo, all_hi, c, cap, [&](int blk) -> const uint8_t* {
                feed.store(blk, mine, mine + 32 * S::ROW);
                if (blk + 1 < end) feed.load(blk + 1);
                if (blk * 32 < all_lo || blk * 32 + 32 > all_hi) special |= clean_values<DP, TYPE, 32>(mine + 32 * S::ROW, t.kv_len - blk * 32);
                return mine;
            }, Nothing());
        }
    } else if (begin < end) {
        const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)mine);
        Feeder<DP, 32, 32> feed(pool, begin, 0, ids[wave][0]);
        constexpr int TURN = Feeder<DP, 32, 32>::BLOCKS;
        feed.ask(0);
        v4i qf[DP / 16];
        load_q<DP>(p, row, qf);
        attend_steps<DP, TYPE, 1, MODE>(st, qf, begin, end, row, all_lo, all_hi, c, cap, [&](int blk) -> const uint8_t* {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // the page numbers are there, the block before has been read
            const int turn = (blk - begin) / TURN;
            if ((blk - begin) % TURN == 0) feed.look(turn);
            feed.copy(blk, base, base + 32 * S::ROW);
            if ((blk - begin) % TURN == 0 && blk + TURN < end) feed.ask(turn + 1);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (blk * 32 < all_lo || blk * 32 + 32 > all_hi) special |= clean_values<DP, TYPE, 32>(mine + 32 * S::ROW, t.kv_len - blk * 32);
            return mine;
        }, Nothing());
    }
    if (special) add_specials<DP, TYPE, MODE, 32>(st, reinterpret_cast<float*>(mine), pool, begin, end, all_lo, all_hi, p.D, row.lo, row.hi);
    // the wavefronts' states meet
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    const float l = other_half_sum(st.l);
    put_sums<DP>(st, row_of_sums<DP>(reinterpret_cast<float*>(mine)));
    if (lane < 32) {
        const int from = row.lo > begin * 32 ? row.lo : begin * 32, to = row.hi < end * 32 ? row.hi : end * 32;
        ml[wave][lane][0] = st.m == kNone && l == 0.f && from < to ? kLowest : st.m;
        ml[wave][lane][1] = l;
    }
    __syncthreads();
    // split z's sums of row i of out: DP floats at part + (z * T * H + i) * DP; their maximum and weight: behind all sums
    const int64_t all = (int64_t)p.T * p.H, first = (int64_t)z * all;
    if (threadIdx.x < 32) {
        // every wavefront's share of a row; divided by the row's sum where nothing else is to be added
        float m = kNone, sum = 0.f, a[X::WAVES];
#pragma unroll
        for (int w = 0; w < X::WAVES; ++w) m = __builtin_fmaxf(m, ml[w][lane][0]);
#pragma unroll
        for (int w = 0; w < X::WAVES; ++w) {
            a[w] = share(ml[w][lane][0], ml[w][lane][1], m);
            sum = __builtin_fmaf(ml[w][lane][1], a[w], sum);
        }
        const float by = g.splits > 1 ? 1.0f : one_over(sum, m != kNone);
#pragma unroll
        for (int w = 0; w < X::WAVES; ++w) weight[w][lane] = a[w] * by;
        if (g.splits > 1 && row.valid)
            *reinterpret_cast<float2*>(part + g.splits * all * DP + (first + (int64_t)row.token * p.H + row.head) * 2) = make_float2(m, sum);
    }
    __syncthreads();
    const int rows = t.rows - t.row0 < ROWS ? t.rows - t.row0 : ROWS;
    for (int x = threadIdx.x; x < rows * (DP / 4); x += X::WAVES * 64) {
        const int r = x / (DP / 4), d = x % (DP / 4) * 4;
        if (d >= p.D) continue;
        v4f v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < X::WAVES; ++w) {
            const float a = weight[w][r];
            const v4f ow = *reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(lds + w * X::WAVE_BYTES) + r * OLD<DP> + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(ow[e], a, v[e]);
        }
        const int token = divide(t.row0 + r, g.group);
        const int64_t i = (int64_t)(t.q_begin + token) * p.H + kv_head * g.group_size + (t.row0 + r - token * g.group_size);
        if (g.splits > 1) *reinterpret_cast<v4f*>(part + (first + i) * DP + d) = v;
        else *reinterpret_cast<uint2*>(p.out + i * p.D + d) = make_uint2(pack2<TYPE>(v[0], v[1]), pack2<TYPE>(v[2], v[3]));
    }
}

template <int DP, int TYPE, int MODE, int WAVES_OF>
__global__ __launch_bounds__(WAVES_OF * 64, SPLIT_WAVES<DP> / WAVES_OF) void attend_split_kernel(const PagedAttention p, const Plan g, float* __restrict__ part) {
    __shared__ __align__(16) uint8_t lds[SplitShape<DP, WAVES_OF>::LDS];
    attend_split<DP, TYPE, MODE, WAVES_OF>(p, g, part, lds, blockIdx.x, blockIdx.y, blockIdx.z);
}

// The workgroups' sums of a row joined, in the order of the splits; DP / 4 lanes a row, four value dims each.  Rows lie as in
// out, so that nothing has to be looked up before the loads: the first splits' sums, all maxima and weights and the ends of
// the sequences come in one turn of memory's latency (found by its tile, a row took three).
constexpr int MAX_SPLITS = 64;
template <int DP, int TYPE>
__global__ __launch_bounds__(256) void attend_join_kernel(const PagedAttention p, const Plan g, const float* __restrict__ part) {
    constexpr int QUADS = DP / 4, PER = 256 / QUADS, EACH = MAX_SPLITS / QUADS;   // lanes and rows; splits whose share a lane works out
    __shared__ float weight[PER][MAX_SPLITS];
    const int64_t all = (int64_t)p.T * p.H;
    const int mine = threadIdx.x / QUADS, at = threadIdx.x % QUADS, d = at * 4;
    const int64_t i = (int64_t)blockIdx.x * PER + mine, r = i < all ? i : all - 1;
    const float* one = part + r * DP + d;
    const float* ml = part + g.splits * all * DP + r * 2;
    constexpr int AHEAD = 8;
    v4f o[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) o[k] = *reinterpret_cast<const v4f*>(one + (k < g.splits ? k : 0) * all * DP);
    float m = kNone, sm[EACH], sl[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int z = k * QUADS + at;
        const float2 v = *reinterpret_cast<const float2*>(ml + (z < g.splits ? z : 0) * all * 2);
        sm[k] = z < g.splits ? v.x : kNone;
        sl[k] = z < g.splits ? v.y : 0.f;
    }
    const int begin = p.q_offsets[0], end = p.q_offsets[p.B];
#pragma unroll
    for (int k = 0; k < EACH; ++k) m = __builtin_fmaxf(m, sm[k]);
#pragma unroll
    for (int x = 1; x < QUADS; x <<= 1) m = __builtin_fmaxf(m, __shfl_xor(m, x));
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const float a = share(sm[k], sl[k], m);
        weight[mine][k * QUADS + at] = a;
        sum = __builtin_fmaf(sl[k], a, sum);
    }
#pragma unroll
    for (int x = 1; x < QUADS; x <<= 1) sum += __shfl_xor(sum, x);
    __syncthreads();
    const float inv = one_over(sum, m != kNone);
    v4f v = {0, 0, 0, 0};
    for (int z = 0; z < g.splits; z += AHEAD) {
        if (z > 0) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) o[k] = *reinterpret_cast<const v4f*>(one + (z + k < g.splits ? z + k : z) * all * DP);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const float a = z + k < g.splits ? weight[mine][z + k] : 0.f;
            if (a != 0.f) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(o[k][e], a, v[e]);
            }
        }
    }
    const int token = (int)(r / p.H);
    if (i >= all || d >= p.D || token < begin || token >= end) return;
    *reinterpret_cast<uint2*>(p.out + r * p.D + d) = make_uint2(pack2<TYPE>(v[0] * inv, v[1] * inv), pack2<TYPE>(v[2] * inv, v[3] * inv));
}

// ---- many rows: four wavefronts of 32 rows each go through the same keys ----------------------------------------------
// A step of 64 keys at a time, the next one on its way to LDS meanwhile; a wait for the wavefront's own copies and a barrier a
// step.  Bound by the issue of instructions: two wavefronts a SIMD, of which each has 130 vector and 86 scalar ones beside 16
// products for 32 keys when it takes those at a time (four such steps in LDS: 316 us for 2048 tokens of 32 heads of 128
// dims over 8192 keys, 84 us for 16 x 816 of 8 heads of 256 over 816), and far fewer for 64 (then 270 and 77, now 255 and 67).
template <int DP>
struct ManyShape {
    static constexpr int WAVES = 4, STEP = 64, MINE = STEP / WAVES, STAGE = 2 * STEP * Shape<DP>::ROW;
    static constexpr int LDS = 2 * STAGE + WAVES * 512 + 128;   // and page numbers, words between wavefronts
};

// Which tile and key head a workgroup has.  Key heads change fastest: workgroups go round the eight chiplets, so each of those has few heads'
// keys in its cache.  Causal rows see the more keys the later they are: the last ones first, and where two workgroups share a CU and
// all run at once, the second half the other way round, so that a long one has a short one beside it.
template <int DP>
__device__ __forceinline__ bool place(const PagedAttention& p, int at, int tiles, int& tile, int& kv_head) {
    const int all = tiles * p.KV;
    if (at >= all) return false;
    if (p.causal && DP != 256 && all <= 512 && at >= 256) at = all - 1 - (at - 256);
    tile = at / p.KV;
    kv_head = at - tile * p.KV;
    if (p.causal) tile = tiles - 1 - tile;
    return true;
}

// The step behind the one that is worked on, widened beside its products into the buffers at `next` (V: V_AT bytes further).
template <typename W, int V_AT>
struct Widening {
    static constexpr int PIECES = W::PIECES;
    W& wide;
    uint8_t*& next;
    const int end;
    __device__ __forceinline__ void start(int step) const {
        if (step + 1 < end) wide.scales(step + 1);
    }
    __device__ __forceinline__ void piece(int p) const { wide.piece(p, next, next + V_AT); }
};

template <int DP, int TYPE, int MODE>
__device__ __forceinline__ void attend_many(const PagedAttention& p, const Plan& g, float* __restrict__ part, uint8_t* lds, int at, int z) {
    using S = Shape<DP>;
    using X = ManyShape<DP>;
    auto ids = reinterpret_cast<uint32_t (*)[2][64]>(lds + 2 * X::STAGE);
    auto specials = reinterpret_cast<int*>(lds + 2 * X::STAGE + X::WAVES * 512);
    auto spans = reinterpret_cast<int (*)[4]>(lds + 2 * X::STAGE + X::WAVES * 512 + 64);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool shared = (MODE & MODE_MORE) != 0 && z < g.shared_splits;
    int tile, kv_head;
    Tile t;
    if (!place<DP>(p, at, shared ? g.shared_tiles : g.tiles, tile, kv_head)) return;   // (here and below: the same for the whole workgroup)
    if (shared ? !locate_shared(p, g, ROWS * X::WAVES, tile, t) : !locate<MODE>(p, g.group_size, ROWS * X::WAVES, tile, t)) return;
    const int row0 = t.row0 + wave * ROWS, row_last = t.rows - 1;
    Row row;
    int lo, hi, all_lo, all_hi;                             // of the workgroup
    int my_lo = 0, my_hi = 0, whole_lo = 0, whole_hi = 0;   // of the wavefront
    if (shared) {
        row = row_of_shared(p, t, g, kv_head, row0, my_lo, my_hi, whole_lo, whole_hi);
        if (lane == 0) {
            spans[wave][0] = my_lo;
            spans[wave][1] = my_hi;
            spans[wave][2] = whole_lo;
            spans[wave][3] = whole_hi;
        }
        __syncthreads();
        lo = min(min(spans[0][0], spans[1][0]), min(spans[2][0], spans[3][0]));
        hi = max(max(spans[0][1], spans[1][1]), max(spans[2][1], spans[3][1]));
        all_lo = max(max(spans[0][2], spans[1][2]), max(spans[2][2], spans[3][2]));
        all_hi = min(min(spans[0][3], spans[1][3]), min(spans[2][3], spans[3][3]));
        lo = __builtin_amdgcn_readfirstlane(lo < hi ? lo : 0);
        hi = __builtin_amdgcn_readfirstlane(lo < hi ? hi : 0);
        all_lo = __builtin_amdgcn_readfirstlane(all_lo);
        all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    } else {
        row = row_of<MODE>(p, t, g, kv_head, row0 + (lane & 31));
        span_of<MODE>(p, t, g, t.row0, t.row0 + ROWS * X::WAVES - 1 < row_last ? t.row0 + ROWS * X::WAVES - 1 : row_last, lo, hi, all_lo, all_hi);
        if (row0 <= row_last) span_of<MODE>(p, t, g, row0, row0 + ROWS - 1 < row_last ? row0 + ROWS - 1 : row_last, my_lo, my_hi, whole_lo, whole_hi);
    }
    int begin = lo / X::STEP, end = (hi + X::STEP - 1) / X::STEP;
    if constexpr (MODE & MODE_MORE) {   // the split's part of them, the first ones a step larger
        const int of = shared ? g.shared_splits : g.splits - g.shared_splits, me = z - (shared ? 0 : g.shared_splits);
        const int n = end - begin, each = shared ? divide(n, g.shared_workers) : divide(n, g.workers), rest = n - each * of;
        begin += me * each + (me < rest ? me : rest);
        end = begin + each + (me < rest ? 1 : 0);
    }
    const Pool pool = make_pool<DP, TYPE, MODE>(p, t, kv_head, g);
    const float c = MODE & MODE_CAP ? 2.0f * p.cap : p.scale * 1.4426950408889634f;
    const Cap cap = {p.cap_by, p.cap_most};
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    using Feed = Feeder<DP, X::STEP, X::MINE>;
    Feed feed(pool, begin, wave * X::MINE, ids[wave][0]);
    Widener<DP, TYPE, X::STEP, X::MINE> wide(pool, begin, end, wave * X::MINE);
    auto copy = [&](int step) {
        const int at = step - begin;
        if (at % Feed::BLOCKS == 0) {
            feed.look(at / Feed::BLOCKS);
            if (step + Feed::BLOCKS < end) feed.ask(at / Feed::BLOCKS + 1);
        }
        const uint32_t to = base + (uint32_t)(at & 1) * X::STAGE;
        feed.copy(step, to, to + X::STEP * S::ROW);
    };
    v4i qf[DP / 16];
    load_q<DP>(p, row, qf);
    bool special = false;
    if (begin < end) {
        if constexpr (MODE & MODE_FP8) {
            wide.ask(0);
            wide.load(begin);
            wide.store(begin, lds, lds + X::STEP * S::ROW);
            if (DP == 128 && begin + 1 < end) wide.load(begin + 1);
        } else {
            feed.ask(0);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            copy(begin);
        }
    }
    State<DP> st;
    st.m = kNone;
    st.l = 0.f;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[b][i] = 0.f;
    // Pages in 8 bits: the step to come is asked for at the top of this one and widened beside its products.  (In the last step
    // what is there is stored once more, where nobody reads it.)  At 128 dims, where two wavefronts share a SIMD and their registers
    // do not reach for that, it is widened at the top and the one behind it asked for.
    constexpr bool BESIDE = (MODE & MODE_FP8) != 0 && DP != 128;
    uint8_t* next = lds;
    auto top = [&](int step) -> const uint8_t* {
        if constexpr (!(MODE & MODE_FP8)) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this step has landed; behind the barrier everybody has read the one before it
        uint8_t* k = lds + (uint32_t)((step - begin) & 1) * X::STAGE;
        const int j0 = step * X::STEP;
        if (j0 < all_lo || j0 + X::STEP > all_hi) special |= clean_values<DP, TYPE, X::MINE>(k + (X::STEP + wave * X::MINE) * S::ROW, t.kv_len - j0 - wave * X::MINE);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if constexpr (MODE & MODE_FP8) {
            next = lds + (uint32_t)((step + 1 - begin) & 1) * X::STAGE;
            if constexpr (BESIDE) {
                if (step + 1 < end) wide.load(step + 1);
            } else if (step + 1 < end) {
                wide.store(step + 1, next, next + X::STEP * S::ROW);
                if (step + 2 < end) wide.load(step + 2);
            }
        } else if (step + 1 < end) copy(step + 1);
        return !BESIDE && (j0 >= my_hi || j0 + X::STEP <= my_lo) ? nullptr : k;
    };
    if constexpr (BESIDE) attend_steps<DP, TYPE, X::STEP / 32, MODE>(st, qf, begin, end, row, whole_lo, whole_hi, c, cap, top, Widening<decltype(wide), X::STEP * S::ROW>{wide, next, end});
    else attend_steps<DP, TYPE, X::STEP / 32, MODE>(st, qf, begin, end, row, whole_lo, whole_hi, c, cap, top, Nothing());
    if (lane == 0) specials[wave] = special ? 1 : 0;
    __syncthreads();
    if ((specials[0] | specials[1] | specials[2] | specials[3]) != 0) {
        // (the wavefronts' sums lie in all of LDS but these words)
        static_assert(X::WAVES * 32 * OLD<DP> * 4 <= 2 * X::STAGE + X::WAVES * 512, "sums reach into the words between wavefronts");
        add_specials<DP, TYPE, MODE, X::STEP>(st, reinterpret_cast<float*>(lds) + wave * 32 * OLD<DP>, pool, begin, end, all_lo, all_hi, p.D, row.lo, row.hi);
    }
    const float l = other_half_sum(st.l);
    if constexpr (MODE & MODE_MORE) {
        if (g.splits > 1) {   // as attend_split_kernel leaves them
            if (!row.valid) return;
            const int64_t all = (int64_t)p.T * p.H, i = z * all + (int64_t)row.token * p.H + row.head;
            const int from = row.lo > begin * X::STEP ? row.lo : begin * X::STEP, to = row.hi < end * X::STEP ? row.hi : end * X::STEP;
            if (lane < 32)
                *reinterpret_cast<float2*>(part + g.splits * all * DP + i * 2) = make_float2(st.m == kNone && l == 0.f && from < to ? kLowest : st.m, l);
            float* o = part + i * DP + 4 * (lane >> 5);
#pragma unroll
            for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v4f v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = st.o[b][4 * k + e];
                    if (32 * b + 8 * k + 4 * (lane >> 5) < p.D) *reinterpret_cast<v4f*>(o + 32 * b + 8 * k) = v;
                }
            return;
        }
    }
    const float inv = one_over(l, row.lo < row.hi);
    if (!row.valid) return;
    uint16_t* out = p.out + ((int64_t)row.token * p.H + row.head) * p.D;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 32 * b + 8 * i + 4 * (lane >> 5);
            if (d < p.D)
                *reinterpret_cast<uint2*>(out + d) = make_uint2(pack2<TYPE>(st.o[b][4 * i] * inv, st.o[b][4 * i + 1] * inv),
                                                                pack2<TYPE>(st.o[b][4 * i + 2] * inv, st.o[b][4 * i + 3] * inv));
        }
}

template <int DP, int TYPE, int MODE>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attend_many_kernel(const PagedAttention p, const Plan g, float* __restrict__ part) {
    __shared__ __align__(16) uint8_t lds[ManyShape<DP>::LDS];
    attend_many<DP, TYPE, MODE>(p, g, part, lds, blockIdx.y * gridDim.x + blockIdx.x, blockIdx.z);
}

// The shared keys for many rows a workgroup, bound by arithmetic, and the sequences' own for few, bound by memory, in one launch: first
// come the workgroups of the shared ones.  64 single tokens of 32 heads on 8 of 128 dims behind 8192 shared keys, up to 512 of their own: 33 us
// and 5 for the join, where few rows for both take 64 in all, and 110 without sharing.
template <int DP, int TYPE, int MODE>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attend_both_kernel(const PagedAttention p, const Plan g, float* __restrict__ part) {
    using X = SplitShape<DP, 4>;
    __shared__ __align__(16) uint8_t lds[X::LDS > ManyShape<DP>::LDS ? X::LDS : ManyShape<DP>::LDS];
    const int once = g.shared_tiles * p.KV, before = once * g.shared_splits;
    int at = blockIdx.x;
    if (at < before) {
        const int z = at / once;
        attend_many<DP, TYPE, MODE>(p, g, part, lds, at - z * once, z);
    } else {
        at -= before;
        const int z = at / (g.tiles * p.KV), rest = at - z * (g.tiles * p.KV), kv_head = rest / g.tiles;
        attend_split<DP, TYPE, MODE, 4>(p, g, part, lds, rest - kv_head * g.tiles, kv_head, g.shared_splits + z);
    }
}

// ---- launches --------------------------------------------------------------------------------------------------------
template <int DP, int TYPE, int MODE>
hipError_t launch(const PagedAttention& p, const Plan& plan, hipStream_t stream) {
    float* part = static_cast<float*>(p.workspace);
    constexpr int WAVES = SPLIT_WAVES<DP>;
    const dim3 grid(plan.tiles > plan.shared_tiles ? plan.tiles : plan.shared_tiles, p.KV, plan.splits);
    hipError_t e = hipSuccess;
    bool done = false;
    if constexpr ((MODE & MODE_MORE) != 0 && (MODE & MODE_WIDE) == 0) {
        done = true;
        if (plan.shared > 0 && plan.shared_many && !plan.many) {
            const int64_t all = ((int64_t)plan.shared_tiles * plan.shared_splits + (int64_t)plan.tiles * (plan.splits - plan.shared_splits)) * p.KV;
            e = enqueue(attend_both_kernel<DP, TYPE, MODE>, dim3((uint32_t)all), dim3(256), stream, p, plan, part);
        } else if (!plan.many && plan.small) e = enqueue(attend_split_kernel<DP, TYPE, MODE, WAVES / 2>, grid, dim3(WAVES * 32), stream, p, plan, part);
        else done = false;
    }
    if constexpr (MODE & MODE_WIDE) e = enqueue(attend_split_kernel<DP, TYPE, MODE, WAVES>, grid, dim3(WAVES * 64), stream, p, plan, part);
    else if (!done) {
        e = plan.many ? enqueue(attend_many_kernel<DP, TYPE, MODE>, grid, dim3(256), stream, p, plan, part)
                      : enqueue(attend_split_kernel<DP, TYPE, MODE, WAVES>, grid, dim3(WAVES * 64), stream, p, plan, part);
    }
    if (e != hipSuccess || plan.splits == 1) return e;
    return enqueue(attend_join_kernel<DP, TYPE>, dim3((unsigned)(((int64_t)p.T * p.H + 1024 / DP - 1) / (1024 / DP))), dim3(256), stream, p, plan, (const float*)part);
}
inline int padded_dim(int64_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
template <int TYPE, int MODE>
hipError_t launch_d(const PagedAttention& p, const Plan& plan, hipStream_t stream) {
    switch (padded_dim(p.D)) {
        case 64: return launch<64, TYPE, MODE>(p, plan, stream);
        case 128: return launch<128, TYPE, MODE>(p, plan, stream);
        default: return launch<256, TYPE, MODE>(p, plan, stream);
    }
}

}  // namespace

// The kernels of one element type and kind of cache, for calls that are more than plain attention over 16-bit pages; one
// source each, since they take long to compile.
hipError_t launch_attention_bf16(const PagedAttention& p, const AttentionPlan& plan, hipStream_t stream);
hipError_t launch_attention_f16(const PagedAttention& p, const AttentionPlan& plan, hipStream_t stream);
hipError_t launch_attention_bf16_fp8(const PagedAttention& p, const AttentionPlan& plan, hipStream_t stream);
hipError_t launch_attention_f16_fp8(const PagedAttention& p, const AttentionPlan& plan, hipStream_t stream);

}  // namespace phyai
