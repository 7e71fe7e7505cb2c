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
#include "fp8_device.h"
#include "layer_kernels.h"
#include "tuning.h"

namespace phyai {
namespace {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef __attribute__((address_space(3))) uint32_t lds_u32;   // (through a generic pointer an access would count as one to memory too)
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8hf __attribute__((ext_vector_type(8)));

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

// j / d for 0 <= j < 2^31 and a d known on the host: one high product (magic 0: d = 1).
struct Division {
    uint32_t magic, shift;
};
__device__ __forceinline__ int divide(int j, Division d) { return d.magic == 0 ? j : (int)(__umulhi((uint32_t)j, d.magic) >> d.shift); }

// What the host works out once per call.
struct Plan {
    Division page, group, workers;
    int group_size, tiles, splits, many;
};

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
};
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
// true if there were any among the keys), and add_special gives them to the rows that see their key after the last tile.
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
// Keys first .. last - 1, from their pages.  (A page that does not exist has made its scores NaN already.)
template <int DP, int TYPE>
__device__ __forceinline__ void add_special(State<DP>& st, const Pool& s, int first, int last, int d_end, int lo, int hi) {
    const int half = (threadIdx.x & 63) >> 5;
    last = last < s.kv_len ? last : s.kv_len;
#pragma unroll 1
    for (int j = first; j < last; ++j) {
        const int at = divide(j, s.by_page), page = s.table[at];
        if (page < 0 || page >= s.n_pages) continue;
        const uint8_t* v = s.v + (int64_t)page * s.page_bytes + (int64_t)(j - at * s.page_size) * s.token_bytes;
        const bool sees = j >= lo && j < hi;
#pragma unroll
        for (int b = 0; b < DP / 32; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 32 * b + 8 * i + 4 * half;
                uint2 w = make_uint2(0, 0);
                if (d < d_end && sees) w = *reinterpret_cast<const uint2*>(v + 2 * d);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t h = ((e & 2 ? w.y : w.x) >> (16 * (e & 1))) & 0xFFFFu;
                    if (any_special<TYPE>(h)) st.o[b][4 * i + e] += to_f32<TYPE>(h);
                }
            }
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
template <int DP, int TYPE, int NB, typename Top>
__device__ __forceinline__ void attend_steps(State<DP>& st, const v4i* qf, int step, int end, const Row& row, int whole_lo, int whole_hi, float c, Top top) {
    using S = Shape<DP>;
    // V is read while the scores are turned into probabilities; as much of it as there are registers for
    constexpr int EARLY = DP == 64 ? 2 : NB == 1 || DP == 256 ? 4 : 2;
    while (step < end) {
        v16f s[NB];
        float mx = kNone;
        const uint8_t *k = nullptr, *v = nullptr;
        bool rises = false;
#pragma unroll 1
        for (; step < end; ++step) {
            k = top(step);
            if (k == nullptr) continue;
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
            const int j0 = step * (32 * NB);
            if (j0 < whole_lo || j0 + 32 * NB > whole_hi) {
#pragma unroll
                for (int n = 0; n < NB; ++n) mask_scores(s[n], j0 + 32 * n, row.lo, row.hi);
            }
            mx = max_score<NB>(s) * c;
            rises = maximum_rises(st.m, mx);
            if (rises) break;
#pragma unroll
            for (int n = 0; n < NB; ++n) st.l += probabilities<TYPE>(s[n], pf[n], st.m, c);
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) st.o[b] = mfma<TYPE>(n == 0 && b < EARLY ? vf[b % EARLY][e] : read_v<DP>(v, 32 * n, b, e), pf[n][e], st.o[b]);
        }
        if (!rises) break;
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

__device__ __forceinline__ Row row_of(const PagedAttention& p, const Tile& t, const Plan& g, int kv_head, int row) {
    Row r;
    r.valid = row < t.rows;
    const int i = r.valid ? divide(row, g.group) : 0;
    r.token = t.q_begin + i;
    r.head = kv_head * g.group_size + (r.valid ? row - i * g.group_size : 0);
    const int position = t.length - t.q_len + i;
    r.hi = !r.valid ? 0 : p.causal ? clamp_i(position + 1, 0, t.kv_len) : t.kv_len;
    r.lo = p.window > 0 && position >= p.window ? position - p.window + 1 : 0;
    return r;
}
// First and last + 1 key that any of the rows row0 .. row1 sees, and that all of them see.
__device__ __forceinline__ void span_of(const PagedAttention& p, const Tile& t, const Plan& g, int row0, int row1, int& lo, int& hi, int& all_lo, int& all_hi) {
    const int i0 = divide(row0, g.group), i1 = divide(row1, g.group);
    const int position0 = t.length - t.q_len + i0, position1 = t.length - t.q_len + i1;
    lo = p.window > 0 && position0 >= p.window ? position0 - p.window + 1 : 0;
    hi = p.causal ? clamp_i(position1 + 1, 0, t.kv_len) : t.kv_len;
    lo = lo < hi ? lo : hi;
    all_lo = p.window > 0 && position1 >= p.window ? position1 - p.window + 1 : 0;
    all_hi = p.causal ? clamp_i(position0 + 1, 0, t.kv_len) : t.kv_len;
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

template <int DP, int TYPE>
__device__ __forceinline__ Pool make_pool(const PagedAttention& p, const Tile& t, int kv_head, const Plan& g) {
    Pool s;
    s.k = reinterpret_cast<const uint8_t*>(p.k_pages + kv_head * p.kv_stride[2]);
    s.v = reinterpret_cast<const uint8_t*>(p.v_pages + kv_head * p.kv_stride[2]);
    s.zero = reinterpret_cast<const uint8_t*>(kFill[0][0]);
    s.nan = reinterpret_cast<const uint8_t*>(kFill[1][TYPE]);
    s.page_bytes = p.kv_stride[0] * 2;
    s.token_bytes = p.kv_stride[1] * 2;
    s.n_pages = (int)p.n_pages;
    s.page_size = p.page_size;
    s.kv_len = t.kv_len;
    s.by_page = g.page;
    s.table = p.table + (int64_t)t.b * p.table_ld;
    s.d_chunks = p.D / 8;
    s.neat = p.D == DP && p.page_size % 8 == 0;
    return s;
}

// ---- few rows: the wavefronts of a workgroup, and several workgroups, share the keys of 32 rows --------------------------
// Each wavefront has 32 keys in LDS to itself and waits for nobody until the end: it copies a block, waits, multiplies,
// copies the next; the others' copies are under way meanwhile (twice as many wavefronts beat two stages for each).  Then the
// workgroup's states meet in LDS; with more than one workgroup per tile they leave unnormalised sums for
// attend_join_kernel.  Many sequences: bound by memory, 64 x 8192 keys of 8 heads of 128 in 254 us, 5.1 TB/s.  Few: by the chain of
// sequence, page numbers, keys (64 bytes a cycle into a CU), products, sums: 50 tokens over 866 keys of 256 dims 15.3 us, 3 to 4 of them the join.
template <int DP>
struct SplitShape {
    static constexpr int WAVES = DP == 256 ? 4 : 8;
    static constexpr int STAGE = 2 * 32 * Shape<DP>::ROW;
    static constexpr int OLD = DP + 4;                            // floats of a row of O in LDS
    static constexpr int WAVE_BYTES = STAGE > 32 * OLD * 4 ? STAGE : 32 * OLD * 4;
};
// What a row's O is divided by, inverted: a sum of zero is a row's that sees nothing, or only scores of -inf.
__device__ __forceinline__ float one_over(float sum, bool sees) { return sum != 0.f ? 1.0f / sum : sees ? __builtin_nanf("") : 0.f; }
// How much of a state with maximum m belongs into one with the larger maximum `all` (m = -inf: it has seen nothing, or NaN).
__device__ __forceinline__ float share(float m, float l, float all) { return m == kNone ? (l != l ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(m - all); }

template <int DP, int TYPE>
__global__ __launch_bounds__(SplitShape<DP>::WAVES * 64, 1) void attend_split_kernel(const PagedAttention p, const Plan g, float* __restrict__ part) {
    using S = Shape<DP>;
    using X = SplitShape<DP>;
    __shared__ __align__(16) uint8_t lds[X::WAVES * X::WAVE_BYTES];
    __shared__ uint32_t ids[X::WAVES][2][64];
    __shared__ float ml[X::WAVES][32][2], weight[X::WAVES][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = blockIdx.x, kv_head = blockIdx.y, z = blockIdx.z;
    Tile t;
    if (!locate(p, g.group_size, ROWS, tile, t)) return;   // (the same for the whole workgroup)
    const Row row = row_of(p, t, g, kv_head, t.row0 + (lane & 31));
    int lo, hi, all_lo, all_hi;
    span_of(p, t, g, t.row0, t.row0 + ROWS < t.rows ? t.row0 + ROWS - 1 : t.rows - 1, lo, hi, all_lo, all_hi);
    const int b0 = lo / 32, n = (hi + 31) / 32 - b0;   // blocks of 32 keys (none: hi = lo = 0)
    // even shares, the first ones a block larger
    const int me = z * X::WAVES + wave, each = divide(n, g.workers), rest = n - each * g.splits * X::WAVES;
    const int begin = b0 + me * each + (me < rest ? me : rest), end = begin + each + (me < rest ? 1 : 0);
    const Pool pool = make_pool<DP, TYPE>(p, t, kv_head, g);
    const float c = p.scale * 1.4426950408889634f;

    State<DP> st;
    st.m = kNone;
    st.l = 0.f;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[b][i] = 0.f;
    uint8_t* mine = lds + wave * X::WAVE_BYTES;
    bool special = false;
    if (begin < end) {
        const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)mine);
        Feeder<DP, 32, 32> feed(pool, begin, 0, ids[wave][0]);
        constexpr int TURN = Feeder<DP, 32, 32>::BLOCKS;
        feed.ask(0);
        v4i qf[DP / 16];
        load_q<DP>(p, row, qf);
        attend_steps<DP, TYPE, 1>(st, qf, begin, end, row, all_lo, all_hi, c, [&](int blk) -> const uint8_t* {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // the page numbers are there, the block before has been read
            const int turn = (blk - begin) / TURN;
            if ((blk - begin) % TURN == 0) feed.look(turn);
            feed.copy(blk, base, base + 32 * S::ROW);
            if ((blk - begin) % TURN == 0 && blk + TURN < end) feed.ask(turn + 1);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (blk * 32 < all_lo || blk * 32 + 32 > all_hi) special |= clean_values<DP, TYPE, 32>(mine + 32 * S::ROW, t.kv_len - blk * 32);
            return mine;
        });
    }
    if (special) {
#pragma unroll 1
        for (int blk = begin; blk < end; ++blk)
            if (blk * 32 < all_lo || blk * 32 + 32 > all_hi) add_special<DP, TYPE>(st, pool, blk * 32, blk * 32 + 32, p.D, row.lo, row.hi);
    }
    // the wavefronts' states meet
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    const float l = other_half_sum(st.l);
    float* o = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v4f v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = st.o[b][4 * i + e];
            *reinterpret_cast<v4f*>(o + (lane & 31) * X::OLD + 32 * b + 8 * i + 4 * (lane >> 5)) = v;
        }
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
            const v4f ow = *reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(lds + w * X::WAVE_BYTES) + r * X::OLD + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(ow[e], a, v[e]);
        }
        const Row w = row_of(p, t, g, kv_head, t.row0 + r);
        const int64_t i = (int64_t)w.token * p.H + w.head;
        if (g.splits > 1) *reinterpret_cast<v4f*>(part + (first + i) * DP + d) = v;
        else *reinterpret_cast<uint2*>(p.out + i * p.D + d) = make_uint2(pack2<TYPE>(v[0], v[1]), pack2<TYPE>(v[2], v[3]));
    }
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
// dims over 8192 keys, 84 us for 16 x 816 of 8 heads of 256 over 816), and far fewer for 64 (then 270 and 77, now 260 and 68).
template <int DP>
struct ManyShape {
    static constexpr int WAVES = 4, STEP = 64, MINE = STEP / WAVES, STAGE = 2 * STEP * Shape<DP>::ROW;
};

template <int DP, int TYPE>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attend_many_kernel(const PagedAttention p, const Plan g) {
    using S = Shape<DP>;
    using X = ManyShape<DP>;
    __shared__ __align__(16) uint8_t lds[2 * X::STAGE];
    __shared__ uint32_t ids[X::WAVES][2][64];
    __shared__ int specials[X::WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv_head = blockIdx.y;
    Tile t;
    if (!locate(p, g.group_size, ROWS * X::WAVES, blockIdx.x, t)) return;
    const int row0 = t.row0 + wave * ROWS, row_last = t.rows - 1;
    const Row row = row_of(p, t, g, kv_head, row0 + (lane & 31));
    int lo, hi, all_lo, all_hi;          // of the workgroup
    span_of(p, t, g, t.row0, t.row0 + ROWS * X::WAVES - 1 < row_last ? t.row0 + ROWS * X::WAVES - 1 : row_last, lo, hi, all_lo, all_hi);
    int my_lo = 0, my_hi = 0, whole_lo = 0, whole_hi = 0;   // of the wavefront
    if (row0 <= row_last) span_of(p, t, g, row0, row0 + ROWS - 1 < row_last ? row0 + ROWS - 1 : row_last, my_lo, my_hi, whole_lo, whole_hi);
    const int begin = lo / X::STEP, end = (hi + X::STEP - 1) / X::STEP;
    const Pool pool = make_pool<DP, TYPE>(p, t, kv_head, g);
    const float c = p.scale * 1.4426950408889634f;
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    using Feed = Feeder<DP, X::STEP, X::MINE>;
    Feed feed(pool, begin, wave * X::MINE, ids[wave][0]);
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
        feed.ask(0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        copy(begin);
    }
    State<DP> st;
    st.m = kNone;
    st.l = 0.f;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[b][i] = 0.f;
    attend_steps<DP, TYPE, X::STEP / 32>(st, qf, begin, end, row, whole_lo, whole_hi, c, [&](int step) -> const uint8_t* {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this step has landed; behind the barrier everybody has read the one before it
        uint8_t* k = lds + (uint32_t)((step - begin) & 1) * X::STAGE;
        const int j0 = step * X::STEP;
        if (j0 < all_lo || j0 + X::STEP > all_hi) special |= clean_values<DP, TYPE, X::MINE>(k + (X::STEP + wave * X::MINE) * S::ROW, t.kv_len - j0 - wave * X::MINE);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (step + 1 < end) copy(step + 1);
        return j0 >= my_hi || j0 + X::STEP <= my_lo ? nullptr : k;
    });
    if (lane == 0) specials[wave] = special ? 1 : 0;
    __syncthreads();
    if ((specials[0] | specials[1] | specials[2] | specials[3]) != 0) {
#pragma unroll 1
        for (int step = begin; step < end; ++step) {
            const int j0 = step * X::STEP;
            if (j0 < all_lo || j0 + X::STEP > all_hi) add_special<DP, TYPE>(st, pool, j0, j0 + X::STEP, p.D, row.lo, row.hi);
        }
    }
    const float l = other_half_sum(st.l);
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

// magic = ceil(2^(31 + l) / d), l = ceil(log2 d)
Division division(uint32_t d) {
    if (d == 1) return {0, 0};
    uint32_t l = 1;
    while ((1ull << l) < d) ++l;
    return {(uint32_t)(((1ull << (31 + l)) + d - 1) / d), l - 1};
}

int padded_dim(int64_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
int64_t tiles_bound(int64_t T, int64_t B, int64_t group, int64_t rows) {
    return T * group / rows + (B < T ? B : T);   // every sequence with tokens adds less than one tile of its own
}
Plan make_plan(int64_t T, int64_t B, int64_t H, int64_t KV, int64_t D, int64_t max_kv, int64_t page_size) {
    Plan r;
    const int64_t group = H / KV;
    r.group_size = (int)group;
    r.page = division((uint32_t)page_size);
    r.group = division((uint32_t)group);
    // Many rows a workgroup once there are workgroups for most of the chip and rows enough to fill them.  Measured, many
    // against few: 104 workgroups of 256 dims 40 and 36 us, 208 of them 44 and 61 (156: 43 and 49); 136 of 128 dims 112 and 73, 264
    // of them 111 and 126; 288 of 64 dims (two to four fit a CU) 28 and 25, 576 of them 37 and 42.
    const int DP = padded_dim(D), waves = DP == 256 ? 4 : 8;
    const int64_t many = tiles_bound(T, B, group, 128) * KV;
    const char* forced = tuning_env("PHYAI_LAYER_ATTEND");   // 0: many rows; n: few rows, n splits
    r.many = forced != nullptr ? atoi(forced) == 0 : many >= (DP == 64 ? 512 : 192) && T * group >= 64 * B;
    r.tiles = (int)tiles_bound(T, B, group, r.many ? 128 : ROWS);
    r.splits = 1;
    if (!r.many) {
        // As many splits as workgroups run at once, and no more than give every wavefront a block: 32 tiles of 4096 keys 34 us
        // in one split, 18.5 in seven; 200 tiles of 816 keys 27.6 in one, 46 in two.
        const int64_t most = (max_kv + 32 * waves - 1) / (32 * waves), tiles = r.tiles * KV, at_once = DP == 64 ? 512 : 256;
        int64_t s = at_once / tiles;
        s = s < most ? s : most;
        if (forced != nullptr) s = atoi(forced);
        r.splits = (int)(s < 1 ? 1 : s < MAX_SPLITS ? s : MAX_SPLITS);
    }
    r.workers = division((uint32_t)(r.splits * waves));
    return r;
}

template <int DP, int TYPE>
hipError_t launch(const PagedAttention& p, const Plan& plan, hipStream_t stream) {
    if (plan.many) return enqueue(attend_many_kernel<DP, TYPE>, dim3(plan.tiles, p.KV), dim3(256), stream, p, plan);
    float* part = static_cast<float*>(p.workspace);
    const hipError_t e = enqueue(attend_split_kernel<DP, TYPE>, dim3(plan.tiles, p.KV, plan.splits), dim3(SplitShape<DP>::WAVES * 64), stream, p, plan, part);
    if (e != hipSuccess || plan.splits == 1) return e;
    return enqueue(attend_join_kernel<DP, TYPE>, dim3((unsigned)(((int64_t)p.T * p.H + 1024 / DP - 1) / (1024 / DP))), dim3(256), stream, p, plan, (const float*)part);
}
template <int TYPE>
hipError_t launch_d(const PagedAttention& p, const Plan& plan, hipStream_t stream) {
    switch (padded_dim(p.D)) {
        case 64: return launch<64, TYPE>(p, plan, stream);
        case 128: return launch<128, TYPE>(p, plan, stream);
        default: return launch<256, TYPE>(p, plan, stream);
    }
}

}  // namespace

size_t paged_attention_workspace_bytes(int64_t T, int64_t B, int64_t H, int64_t KV, int64_t D, int64_t max_kv) {
    if (T <= 0 || B <= 0) return 0;
    const Plan plan = make_plan(T, B, H, KV, D, max_kv, 1);
    if (plan.many || plan.splits == 1) return 0;
    return (size_t)plan.splits * T * H * (padded_dim(D) + 2) * sizeof(float);
}

hipError_t launch_paged_attention(const PagedAttention& p, hipStream_t stream) {
    const Plan plan = make_plan(p.T, p.B, p.H, p.KV, p.D, (int64_t)p.table_width * p.page_size, p.page_size);
    return p.type == HEAD_BF16 ? launch_d<HEAD_BF16>(p, plan, stream) : launch_d<HEAD_F16>(p, plan, stream);
}

}  // namespace phyai
