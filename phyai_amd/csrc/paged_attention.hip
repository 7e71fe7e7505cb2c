// Attention of each sequence's new tokens over its pages (gfx950).  Row (i, g) of sequence b and key head h - new token i,
// query head h G + g, position kv_b - q_b + i - sees the keys j with lo <= j < hi (causal: hi = position + 1, window: lo =
// position - window + 1) and gets sum_j softmax_j(scale q.k_j) v_j, zero where it sees nothing.
//
// One pass over the keys with a running maximum m and sum l per row, in the base-2 domain.  Both products are computed
// transposed: S^T = K Q^T by v_mfma_f32_32x32x16, so a lane holds 16 of the 32 keys' scores of ONE row (the other 16 are in
// the lane 32 further) and the softmax needs a single exchange; P^T then lies in the registers exactly as the B operand of
// O^T = V^T P^T wants it, if V's keys are taken in the same order - which the transposing LDS read is free to do - and m,
// l and the rescaling of O are one value per lane.  O is only rescaled when a row's maximum grows by more than 2^8:
// probabilities stay below 2^8, which neither bf16, fp16 nor the fp32 sums mind.
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
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8hf __attribute__((ext_vector_type(8)));

constexpr int ROWS = 32;               // rows of a wavefront's tile
constexpr float kNone = -__builtin_huge_valf();
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
    else return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
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

// Where a tile of `rows_per_tile` packed rows lies: the tiles of the sequences are numbered one sequence after another.
// Every wavefront finds it by itself, 64 sequences at a time.
struct Tile {
    int b, row0, rows, q_begin, q_len, kv_len;
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
        int upto = tiles;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int v = __shfl_up(upto, s);
            if (lane >= s) upto += v;
        }
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
            o.kv_len = kv < 0 ? 0 : kv > most ? (int)most : kv;
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

// What a wavefront needs to bring N keys of a tile (its share): the place of key `row` + lane % N in the pool.
struct Pool {
    const uint8_t *k, *v;              // the key head's first element in page 0
    const uint8_t *zero, *nan;
    int64_t page_bytes, token_bytes;
    int n_pages, page_size, kv_len;
    Division by_page;
    int d_chunks;                      // 16-byte chunks of a key that exist
    bool neat;                         // whole keys of a copy instruction are neighbours in a page
};
__device__ __forceinline__ int page_of(const Pool& s, int j) { return divide(j, s.by_page); }

// The page number of key j for every lane, into `slot` (256 bytes of LDS): issued with the copies and counted with them.
__device__ __forceinline__ void copy_page_id(const Pool& s, const int32_t* table_row, int width, int j, uint32_t slot) {
    int page = page_of(s, j);
    page = page < width ? page : width - 1;
    copy4_to_lds<kBaseSettles>(reinterpret_cast<const uint8_t*>(table_row), (uint32_t)page * 4u, slot);
}

// Copies keys j0 .. j0 + N - 1 of K and V to rows `row` .. of the tile's buffers; `page` is the number of the page that
// key j0 + lane % N lies in.
template <int DP, int N>
__device__ __forceinline__ void copy_keys(const Pool& s, int page, int j0, int row, uint32_t k_lds, uint32_t v_lds) {
    using S = Shape<DP>;
    constexpr int COPIES = N / S::PER_COPY;
    const int lane = threadIdx.x & 63;
    const int j = j0 + (lane & (N - 1));
    const int first = page_of(s, j) * s.page_size;
    const bool there = j < s.kv_len, good = page >= 0 && page < s.n_pages;
    const int64_t off = (int64_t)page * s.page_bytes + (int64_t)(j - first) * s.token_bytes;
    const uint32_t lr = (uint32_t)lane / S::CHUNKS, lc = (uint32_t)lane % S::CHUNKS;
    if (s.neat && __all(there && good)) {
        // the swizzles of copy t are those of copy 0 with the bits of t's first key flipped
        const uint32_t run = lr * (uint32_t)s.token_bytes, kc = (lc ^ k_swizzle<DP>((uint32_t)row + lr)) << 4, vc = (lc ^ v_swizzle<DP>((uint32_t)row + lr)) << 4;
#pragma unroll
        for (int t = 0; t < COPIES; ++t) {
            const uint32_t to = (uint32_t)(row + t * S::PER_COPY) * S::ROW;
            const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)off, t * S::PER_COPY) |
                                (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(off >> 32), t * S::PER_COPY) << 32;
            copy16_to_lds<kBaseSettles>(s.k + at, (kc ^ k_swizzle<DP>(t * S::PER_COPY) << 4) + run, __builtin_amdgcn_readfirstlane(k_lds + to));
            copy16_to_lds<kBaseSettles>(s.v + at, (vc ^ v_swizzle<DP>(t * S::PER_COPY) << 4) + run, __builtin_amdgcn_readfirstlane(v_lds + to));
        }
        return;
    }
    const int lo = (int)(uint32_t)off, hi = (int)(off >> 32), kind = !there ? 1 : !good ? 2 : 0;
#pragma unroll 1   // (code that a cold instruction cache does not have to bring: most calls come here once)
    for (int t = 0; t < COPIES; ++t) {
        const int from = t * S::PER_COPY + (int)lr;
        const uint32_t r = (uint32_t)(row + from);
        const int64_t at = (int64_t)(uint32_t)__shfl(lo, from) | (int64_t)__shfl(hi, from) << 32;
        const int what = __shfl(kind, from);
        const uint32_t kc = lc ^ k_swizzle<DP>(r), vc = lc ^ v_swizzle<DP>(r);
        const uint8_t* fill = what == 2 ? s.nan : s.zero;
        const uint8_t* ka = what != 0 ? fill : (int)kc < s.d_chunks ? s.k + at + kc * 16 : s.zero;
        const uint8_t* va = what != 0 ? fill : (int)vc < s.d_chunks ? s.v + at + vc * 16 : s.zero;
        const uint32_t to = (uint32_t)(row + t * S::PER_COPY) * S::ROW;
        copy16_from(ka, __builtin_amdgcn_readfirstlane(k_lds + to));
        copy16_from(va, __builtin_amdgcn_readfirstlane(v_lds + to));
    }
}

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
// taken out of V as it lands (each wavefront looks through the keys it has copied itself; true if there were any), and
// add_special gives them to the rows that see their key after the last tile.
template <int DP, int TYPE, int N>
__device__ __forceinline__ bool clean_values(uint8_t* v) {
    bool special = false;
#pragma unroll 1
    for (int x = (threadIdx.x & 63) * 16; x < N * Shape<DP>::ROW; x += 1024) {
        v4i f = *reinterpret_cast<const v4i*>(v + x);
        bool any = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            any |= any_special<TYPE>((uint32_t)f[i]);
            f[i] = (int)without_special<TYPE>((uint32_t)f[i]);
        }
        if (any) *reinterpret_cast<v4i*>(v + x) = f;
        special |= any;
    }
    return __any(special);
}
// Keys first .. last - 1, from their pages.  (A page that does not exist has made its scores NaN already.)
template <int DP, int TYPE>
__device__ __forceinline__ void add_special(State<DP>& st, const Pool& s, const int32_t* table, int first, int last, int d_end, int lo, int hi) {
    const int half = (threadIdx.x & 63) >> 5;
    last = last < s.kv_len ? last : s.kv_len;
#pragma unroll 1
    for (int j = first; j < last; ++j) {
        const int at = page_of(s, j), page = table[at];
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

// kbuf, vbuf: the tile's buffers; row: the block's first key in them; j0: that key's number; the row sees [lo, hi).
// masked (uniform): some row of the wavefront does not see the whole block.
template <int DP, int TYPE>
__device__ __forceinline__ void attend_block(State<DP>& st, const v4i* qf, const uint8_t* kbuf, const uint8_t* vbuf, int row, int j0, int lo, int hi, float c,
                                             bool masked) {
    using S = Shape<DP>;
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
    v16f s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
    {
        // chunk 2 kk + half of the lane's key: an xor with a constant below 256 bytes, an offset above
        const uint32_t r = (uint32_t)l32, a0 = r * S::ROW + (((uint32_t)half ^ k_swizzle<DP>(r)) << 4);
        const uint8_t* kr = kbuf + row * S::ROW;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
            const v4i a = *reinterpret_cast<const v4i*>(kr + (a0 ^ ((uint32_t)(kk & 7) << 5)) + (kk >> 3) * 256);
            s = mfma<TYPE>(a, qf[kk], s);
        }
    }
    if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int j = j0 + 8 * (i >> 2) + 4 * half + (i & 3);
            s[i] = j >= lo && j < hi ? s[i] : kNone;
        }
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = __builtin_fmaxf(mx, s[i]);
    mx = other_half_max(mx) * c;
    if (__any(mx > st.m + kRescaleAt)) {
        const float m = __builtin_fmaxf(st.m, mx);
        const float a = m == kNone ? 1.0f : __builtin_amdgcn_exp2f(st.m - m);
        if (__any(st.m != kNone)) {   // (else O and l are zero)
            st.l *= a;
#pragma unroll
            for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) st.o[b][i] *= a;
        }
        st.m = m;
    }
    const float base = st.m == kNone ? 0.f : st.m;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -base));
    // the sum is of the rounded probabilities, those that the second product uses: their common error cancels
    v4i pf[2];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = pack2<TYPE>(s[8 * e + 2 * i], s[8 * e + 2 * i + 1]);
            pf[e][i] = (int)w;
            sum[e] = add_pair<TYPE>(w, sum[e]);
        }
    st.l += sum[0] + sum[1];
    // V^T: lane (16 g + t) asks for key 4 half + t / 4 of a run of eight and dims 16 (g & 1) + 4 (t & 3) .. of a block of 32
    const uint32_t key0 = (uint32_t)(4 * half + ((lane & 15) >> 2)), chunk0 = (uint32_t)((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    const uint32_t v0 = key0 * S::ROW + ((chunk0 ^ v_swizzle<DP>(key0)) << 4) + (lane & 1) * 8;
    const uint8_t* vr = vbuf + row * S::ROW;
    auto read_v = [&](int b, int e) -> v4i {
        union { v4s h[2]; v4i v; } f;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            // eight keys further the swizzle has bit 1 of the chunk flipped (two chunks of four bits at DP = 64: none)
            const uint32_t flip = ((uint32_t)(b & 3) << 6) ^ (DP != 64 && x ? 32u : 0u);
            f.h[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(vr + (v0 ^ flip) + (16 * e + 8 * x) * S::ROW + (b >> 2) * 256));
        }
        return f.v;
    };
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) st.o[b] = mfma<TYPE>(read_v(b, e), pf[e], st.o[b]);
}

// A row of the tile: which token and head it is and which keys it sees.
struct Row {
    int token, head, lo, hi;
    bool valid;
};
__device__ __forceinline__ Row row_of(const PagedAttention& p, const Tile& t, const Plan& g, int kv_head, int row) {
    Row r;
    r.valid = row < t.rows;
    const int i = r.valid ? divide(row, g.group) : 0;
    r.token = t.q_begin + i;
    r.head = kv_head * g.group_size + (r.valid ? row - i * g.group_size : 0);
    const int position = t.kv_len - t.q_len + i;
    r.hi = !r.valid ? 0 : p.causal ? clamp_i(position + 1, 0, t.kv_len) : t.kv_len;
    r.lo = p.window > 0 && position >= p.window ? position - p.window + 1 : 0;
    return r;
}
// First and last + 1 key that any of the rows row0 .. row1 sees, and that all of them see.
__device__ __forceinline__ void span_of(const PagedAttention& p, const Tile& t, const Plan& g, int row0, int row1, int& lo, int& hi, int& all_lo, int& all_hi) {
    const int i0 = divide(row0, g.group), i1 = divide(row1, g.group);
    const int position0 = t.kv_len - t.q_len + i0, position1 = t.kv_len - t.q_len + i1;
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
    s.d_chunks = p.D / 8;
    s.neat = p.D == DP && p.page_size % Shape<DP>::PER_COPY == 0;
    return s;
}

// ---- few rows: the wavefronts of a workgroup, and several workgroups, share the keys of 32 rows --------------------------
// Each wavefront has 32 keys in LDS to itself and waits for nobody until the end: it copies a block, waits, multiplies,
// copies the next; the others' copies are under way meanwhile (twice as many wavefronts beat two stages for each).  Then the
// workgroup's states meet in LDS; with more than one workgroup per tile they leave unnormalised sums for
// attend_join_kernel.
template <int DP>
struct SplitShape {
    static constexpr int WAVES = DP == 256 ? 4 : 8;
    static constexpr int STAGE = 2 * 32 * Shape<DP>::ROW;
    static constexpr int OLD = DP + 4;                            // floats of a row of O in LDS
    static constexpr int WAVE_BYTES = STAGE > 32 * OLD * 4 ? STAGE : 32 * OLD * 4;
};
// How much of a state with maximum m belongs into one with the larger maximum `all` (m = -inf: it has seen nothing, or NaN).
__device__ __forceinline__ float share(float m, float l, float all) { return m == kNone ? (l != l ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(m - all); }

template <int DP, int TYPE>
__global__ __launch_bounds__(SplitShape<DP>::WAVES * 64, 1) void attend_split_kernel(const PagedAttention p, const Plan g, float* __restrict__ part) {
    using S = Shape<DP>;
    using X = SplitShape<DP>;
    __shared__ __align__(16) uint8_t lds[X::WAVES * X::WAVE_BYTES];
    __shared__ uint32_t ids[X::WAVES][64];
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
    const int32_t* table = p.table + (int64_t)t.b * p.table_ld;
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
        const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)mine), idp = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)ids[wave]);
        volatile uint32_t* my_id = &ids[wave][lane];
        copy_page_id(pool, table, p.table_width, begin * 32 + (lane & 31), idp);
        v4i qf[DP / 16];
        load_q<DP>(p, row, qf);
#pragma unroll 1
        for (int blk = begin; blk < end; ++blk) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // the page numbers are there, the block before has been read
            const int page = (int)*my_id;
            copy_keys<DP, 32>(pool, page, blk * 32, 0, base, base + 32 * S::ROW);
            if (blk + 1 < end) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                copy_page_id(pool, table, p.table_width, (blk + 1) * 32 + (lane & 31), idp);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            const int j0 = blk * 32;
            if (j0 < all_lo || j0 + 32 > all_hi) special |= clean_values<DP, TYPE, 32>(mine + 32 * S::ROW);
            const bool whole = !row.valid || (j0 >= row.lo && j0 + 32 <= row.hi);
            attend_block<DP, TYPE>(st, qf, mine, mine + 32 * S::ROW, 0, j0, row.lo, row.hi, c, !__all(whole));
        }
    }
    if (special) {
#pragma unroll 1
        for (int blk = begin; blk < end; ++blk)
            if (blk * 32 < all_lo || blk * 32 + 32 > all_hi) add_special<DP, TYPE>(st, pool, table, blk * 32, blk * 32 + 32, p.D, row.lo, row.hi);
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
        ml[wave][lane][0] = st.m;
        ml[wave][lane][1] = l;
    }
    __syncthreads();
    float* part_o = part + (((int64_t)z * gridDim.y + kv_head) * g.tiles + tile) * (ROWS * (DP + 2));
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
        const float by = g.splits > 1 ? 1.0f : sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
        for (int w = 0; w < X::WAVES; ++w) weight[w][lane] = a[w] * by;
        if (g.splits > 1) {
            part_o[ROWS * DP + 2 * lane] = m;
            part_o[ROWS * DP + 2 * lane + 1] = sum;
        }
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
        if (g.splits > 1) {
            *reinterpret_cast<v4f*>(part_o + r * DP + d) = v;
        } else {
            const Row w = row_of(p, t, g, kv_head, t.row0 + r);
            *reinterpret_cast<uint2*>(p.out + ((int64_t)w.token * p.H + w.head) * p.D + d) = make_uint2(pack2<TYPE>(v[0], v[1]), pack2<TYPE>(v[2], v[3]));
        }
    }
}

// The workgroups' sums of a tile's rows joined, in the order of the splits.  One lane per four value dims of a row; what each
// split's share is, the lanes of a wavefront work out one split each.
constexpr int MAX_SPLITS = 64;
template <int DP, int TYPE>
__global__ __launch_bounds__(256) void attend_join_kernel(const PagedAttention p, const Plan g, const float* __restrict__ part) {
    constexpr int QUADS = DP / 4, PER = 256 / QUADS;   // rows of a workgroup
    __shared__ float weight[PER][MAX_SPLITS];
    const int tile = blockIdx.x, kv_head = blockIdx.y;
    Tile t;
    if (!locate(p, g.group_size, ROWS, tile, t)) return;
    const int r0 = blockIdx.z * PER, rows = t.rows - t.row0;
    if (r0 >= rows) return;   // (the whole workgroup)
    const float* all = part + ((int64_t)kv_head * g.tiles + tile) * (ROWS * (DP + 2));
    const int64_t step = (int64_t)p.KV * g.tiles * (ROWS * (DP + 2));
    const int lane = threadIdx.x & 63;
    for (int i = threadIdx.x >> 6; i < PER; i += 4) {
        float m = kNone, l = 0.f;
        if (lane < g.splits && r0 + i < rows) {
            const float* one = all + lane * step + ROWS * DP + 2 * (r0 + i);
            m = one[0];
            l = one[1];
        }
        float top = m;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, s));
        const float a = share(m, l, top);
        float sum = wave_sum_f32(l * a);
        weight[i][lane] = a * (sum == 0.f ? 0.f : 1.0f / sum);
    }
    __syncthreads();
    const int i = threadIdx.x / QUADS, r = r0 + i, d = (threadIdx.x % QUADS) * 4;
    if (r >= rows || d >= p.D) return;
    v4f v = {0, 0, 0, 0};
    const float* one = all + r * DP + d;
    for (int z = 0; z < g.splits; z += 8) {
        v4f o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = *reinterpret_cast<const v4f*>(one + (z + k < g.splits ? z + k : z) * step);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float a = z + k < g.splits ? weight[i][z + k] : 0.f;
            if (a != 0.f) {   // (a split that has seen nothing may have left anything)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(o[k][e], a, v[e]);
            }
        }
    }
    const Row w = row_of(p, t, g, kv_head, t.row0 + r);
    *reinterpret_cast<uint2*>(p.out + ((int64_t)w.token * p.H + w.head) * p.D + d) = make_uint2(pack2<TYPE>(v[0], v[1]), pack2<TYPE>(v[2], v[3]));
}

// ---- many rows: four wavefronts of 32 rows each go through the same keys ----------------------------------------------
template <int DP>
struct ManyShape {
    static constexpr int WAVES = 4, KEYS = DP == 256 ? 32 : 64;
    static constexpr int STAGE = 2 * KEYS * Shape<DP>::ROW;
};

template <int DP, int TYPE>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attend_many_kernel(const PagedAttention p, const Plan g) {
    using S = Shape<DP>;
    using X = ManyShape<DP>;
    constexpr int MINE = X::KEYS / X::WAVES;
    __shared__ __align__(16) uint8_t lds[2 * X::STAGE];
    __shared__ uint32_t ids[X::WAVES][64];
    __shared__ int specials[X::WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv_head = blockIdx.y;
    Tile t;
    if (!locate(p, g.group_size, ROWS * X::WAVES, blockIdx.x, t)) return;
    const Row row = row_of(p, t, g, kv_head, t.row0 + wave * ROWS + (lane & 31));
    int lo, hi, all_lo, all_hi;
    span_of(p, t, g, t.row0, t.row0 + ROWS * X::WAVES < t.rows ? t.row0 + ROWS * X::WAVES - 1 : t.rows - 1, lo, hi, all_lo, all_hi);
    const int begin = lo / X::KEYS, end = (hi + X::KEYS - 1) / X::KEYS;
    const Pool pool = make_pool<DP, TYPE>(p, t, kv_head, g);
    const int32_t* table = p.table + (int64_t)t.b * p.table_ld;
    const float c = p.scale * 1.4426950408889634f;
    State<DP> st;
    st.m = kNone;
    st.l = 0.f;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[b][i] = 0.f;
    v4i qf[DP / 16];
    load_q<DP>(p, row, qf);
    const uint32_t base = (uint32_t)(uintptr_t)lds, idp = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)ids[wave]);
    volatile uint32_t* my_id = &ids[wave][lane];
    const int ahead = wave * MINE + (lane & (MINE - 1));   // the key of a tile whose page this lane looks up
    if (begin < end) copy_page_id(pool, table, p.table_width, begin * X::KEYS + ahead, idp);
    bool special = false;
    for (int blk = begin - 1; blk < end; ++blk) {
        const int cur = (blk - begin) & 1;
        // this tile and the next one's page numbers have landed; behind the barrier the other stage has been read
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (blk >= begin && (blk * X::KEYS < all_lo || (blk + 1) * X::KEYS > all_hi))
            special |= clean_values<DP, TYPE, MINE>(lds + cur * X::STAGE + (X::KEYS + wave * MINE) * S::ROW);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (blk + 1 < end) {
            const int page = (int)*my_id;
            const uint32_t to = base + (cur ^ 1) * X::STAGE;
            copy_keys<DP, MINE>(pool, page, (blk + 1) * X::KEYS + wave * MINE, wave * MINE, to, to + X::KEYS * S::ROW);
            if (blk + 2 < end) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                copy_page_id(pool, table, p.table_width, (blk + 2) * X::KEYS + ahead, idp);
            }
        }
        if (blk < begin) continue;
        const uint8_t* k = lds + cur * X::STAGE;
#pragma unroll
        for (int x = 0; x < X::KEYS / 32; ++x) {
            const int j0 = blk * X::KEYS + x * 32;
            const bool whole = !row.valid || (j0 >= row.lo && j0 + 32 <= row.hi), none = j0 >= row.hi || j0 + 32 <= row.lo;
            if (__all(none)) continue;
            attend_block<DP, TYPE>(st, qf, k, k + X::KEYS * S::ROW, x * 32, j0, row.lo, row.hi, c, !__all(whole));
        }
    }
    if (lane == 0) specials[wave] = special ? 1 : 0;
    __syncthreads();
    if ((specials[0] | specials[1] | specials[2] | specials[3]) != 0) {
#pragma unroll 1
        for (int blk = begin; blk < end; ++blk)
            if (blk * X::KEYS < all_lo || (blk + 1) * X::KEYS > all_hi)
                add_special<DP, TYPE>(st, pool, table, blk * X::KEYS, (blk + 1) * X::KEYS, p.D, row.lo, row.hi);
    }
    const float l = other_half_sum(st.l);
    const float inv = l == 0.f ? 0.f : 1.0f / l;
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
    const int64_t many = tiles_bound(T, B, group, 128) * KV;
    const char* forced = tuning_env("PHYAI_LAYER_ATTEND");   // 0: many rows; n: few rows, n splits
    r.many = forced != nullptr ? atoi(forced) == 0 : many >= 256 && T * group >= 64 * B;
    r.tiles = (int)tiles_bound(T, B, group, r.many ? 128 : ROWS);
    r.splits = 1;
    const int waves = padded_dim(D) == 256 ? 4 : 8;
    if (!r.many) {
        const int64_t most = (max_kv + 32 * waves - 1) / (32 * waves);
        int64_t s = (512 + r.tiles * KV - 1) / (r.tiles * KV);
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
    return enqueue(attend_join_kernel<DP, TYPE>, dim3(plan.tiles, p.KV, ROWS / (256 / (DP / 4))), dim3(256), stream, p, plan, (const float*)part);
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
    return (size_t)plan.splits * KV * plan.tiles * (ROWS * (padded_dim(D) + 2)) * sizeof(float);
}

hipError_t launch_paged_attention(const PagedAttention& p, hipStream_t stream) {
    const Plan plan = make_plan(p.T, p.B, p.H, p.KV, p.D, (int64_t)p.table_width * p.page_size, p.page_size);
    return p.type == HEAD_BF16 ? launch_d<HEAD_BF16>(p, plan, stream) : launch_d<HEAD_F16>(p, plan, stream);
}

}  // namespace phyai
