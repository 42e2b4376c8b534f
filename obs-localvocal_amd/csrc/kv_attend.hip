// kv_attend.hip — attention of each sequence's new tokens over its paged keys and values.
//
//   out[t][h] = sum_j softmax_j(scale q[t][h] . k_j) v_j,   j <= p(t),  and with a window j > p(t) - window or j < sinks
//
// One pass over the keys with the running maximum m and sum l of the softmax; base-2 exponents (scale log2(e) is folded
// into the scores).  Everything is computed transposed, so that no operand changes lanes:
//   S^T[key][row] = K . Q^T    A = K (lane: key l & 15, 8 dims), B = Q (lane: row l & 15, 8 dims; registers)
//                              -> lane (row = l & 15, g = l >> 4) holds keys 4g .. 4g + 3 of a 16-key tile
//   O^T[dim][row] += V^T . P^T B = P^T: the 4 + 4 probabilities a lane has of two key tiles ARE its fragment if the contraction
//                              index of 32 keys is ordered (g, tile, r); A = V^T in that order is what two transposing LDS
//                              reads (ds_read_tr16_b64) give from V rows as they lie in the cache
// A "row" is one (token, query head) pair; the query heads that share a key / value head are rows of one tile, so each
// cached row is read once for all of them.
//
// 8-bit caches: the codes become bf16 exactly (e4m3 has 4 significant bits, int8 codes 8) and go through the same products;
// a key's scale multiplies its scores, a value's scale its probabilities, both in fp32.
#include "decoder_ops.hpp"

#include <type_traits>

namespace mw {

namespace {

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x2 = __attribute__((ext_vector_type(2))) float;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
using u32x2 = __attribute__((ext_vector_type(2))) unsigned;
using u16x2 = __attribute__((ext_vector_type(2))) unsigned short;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using lds_s16x4 = __attribute__((address_space(3))) s16x4;

constexpr int BF16 = MW_ELEM_BF16, E4M3 = MW_ELEM_E4M3, INT8 = MW_ELEM_INT8;

struct AttendP {
    KvView V;
    int n_heads, group;  // query heads per key / value head
    const bf16_t *q;
    int64_t q_row, q_head;
    bf16_t *out;
    int64_t o_row, o_head;
    float c;  // scale log2(e)
    int window, sinks, splits, split_steps, tiles;
    float *ws_o, *ws_ml;  // [splits][n_rows][n_heads][head_dim], [splits][n_rows][n_heads][2]
};

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

// signed byte B of w as a float, in one instruction (from C every other one came with a v_bfe_i32 of its own)
template <int B> __device__ __forceinline__ float byte_of(unsigned w) {
    float f;
    if constexpr (B == 0) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(f) : "v"(w));
    else if constexpr (B == 1) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f) : "v"(w));
    else if constexpr (B == 2) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f) : "v"(w));
    else asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f) : "v"(w));
    return f;
}
// 8 cache elements -> 8 bf16
template <int KIND> struct Raw { using type = u32x2; };
template <> struct Raw<BF16> { using type = u32x4; };
template <int KIND> __device__ __forceinline__ u32x4 to_bf16(typename Raw<KIND>::type r) {
    if constexpr (KIND == BF16) {
        return r;
    } else if constexpr (KIND == E4M3) {
        return u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x, 1.0f, false)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x, 1.0f, true)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.y, 1.0f, false)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.y, 1.0f, true))};
    } else {
        return u32x4{pack_bf16(byte_of<0>(r.x), byte_of<1>(r.x)), pack_bf16(byte_of<2>(r.x), byte_of<3>(r.x)),
                     pack_bf16(byte_of<0>(r.y), byte_of<1>(r.y)), pack_bf16(byte_of<2>(r.y), byte_of<3>(r.y))};
    }
}
// fragment f (8 elements) of 16 bytes of a row: all of it in bf16, one of two in 8 bits.  The order in which a lane has the dims
// is free as long as the queries' fragments have the same: 16 bytes a lane are 64 adjacent bytes of a row (with 8, an 8-bit
// cache was read in pieces of 32 and twice as many loads).
template <int KIND> __device__ __forceinline__ u32x4 fragment(u32x4 x, int f) {
    if constexpr (KIND == BF16) return x;
    else return to_bf16<KIND>(f ? u32x2{x.z, x.w} : u32x2{x.x, x.y});
}
// what the rounding of 8 probabilities to bf16 (hi) left, itself in bf16
__device__ __forceinline__ u32x4 low_part(const float *e, u32x4 hi) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        o[i] = pack_bf16(e[2 * i] - __uint_as_float(hi[i] << 16), e[2 * i + 1] - __uint_as_float(hi[i] & 0xffff0000u));
    return o;
}
// the n lowest of 32 bits (none below 0, all from 32 on)
__device__ __forceinline__ unsigned low_bits(int64_t n) {
    const int c = (int)min(max(n, (int64_t)0), (int64_t)32);
    return c == 0 ? 0u : ~0u >> (32 - c);
}
__device__ __forceinline__ bool has_nonfinite(u32x4 x) {  // of 8 bf16
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[i] & 0x7fff7fffu));
    return max(m.x, m.y) >= 0x7f80;
}

// A value that is the same in all lanes, for the compiler to know: what follows from it (a step's keys, the loops' ends) then stays
// in scalar registers.
__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The tile of `tile_rows` rows (token, head of the group) a workgroup has.  Sequences are cut into tiles one after the other; every
// wave looks through 64 sequences at a time, and each lane loads all that is to be known of its own: one trip to memory.
struct Tile {
    int seq, first;  // sequence, first row inside it
    int row0, nq;    // the sequence's first row in q, its tokens
    int kv_len;
};
__device__ __forceinline__ bool find_tile(const KvView &V, int group, int tile_rows, int tile, Tile &T) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int s0 = 0; s0 < V.n_seqs; s0 += 64) {
        const int b = s0 + lane;
        int n = 0, start = 0, end = 0, len = 0;
        if (b < V.n_seqs) {
            start = kv_cu(V, b);
            end = kv_cu(V, b + 1);
            len = V.kv_len[b];
            const int64_t rows = (int64_t)max(0, end - start) * group;
            n = (int)((rows + tile_rows - 1) / tile_rows);
        }
        int incl = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(incl, o);
            if (lane >= o) incl += u;
        }
        const int all = scalar(__shfl(incl, 63));
        if (tile - base < all) {
            const unsigned long long m = __ballot(base + incl > tile);
            const int l = __ffsll((unsigned long long)m) - 1;
            T.seq = scalar(s0 + l);
            T.first = scalar((tile - base - __shfl(incl - n, l)) * tile_rows);
            T.row0 = scalar(__shfl(start, l));
            T.nq = scalar(__shfl(end, l)) - T.row0;
            T.kv_len = scalar(__shfl(len, l));
            return true;
        }
        base += all;
    }
    return false;
}

// The keys a tile of rows at positions p_lo .. p_hi needs, in steps of KS keys: first the sinks below the window, then the
// window (without one: everything from 0).
struct KeySteps {
    int64_t lo, hi;  // main stretch (lo a multiple of KS), hi: one behind the last visible key
    int n_sink, n;   // steps of the sinks, steps in all
};
template <int KS> __device__ __forceinline__ KeySteps key_steps(const KvView &V, int window, int sinks, int64_t p_lo, int64_t p_hi) {
    KeySteps s;
    s.hi = min(p_hi + 1, (int64_t)V.table_cols << V.shift);
    const int64_t first = window > 0 ? max((int64_t)0, p_lo - window + 1) : 0;
    s.lo = first / KS * KS;
    const int64_t sink_end = window > 0 ? min(min((int64_t)sinks, s.lo), s.hi) : 0;
    s.n_sink = (int)((max(sink_end, (int64_t)0) + KS - 1) / KS);
    s.n = s.n_sink + (int)(max((int64_t)0, s.hi - s.lo + KS - 1) / KS);
    return s;
}
template <int KS> __device__ __forceinline__ int64_t step_key(const KeySteps &s, int i) { return i < s.n_sink ? (int64_t)i * KS : s.lo + (int64_t)(i - s.n_sink) * KS; }

// The steps of a split: all splits but a sequence's last have the same number, so that long and short sequences of a batch give
// workgroups of one size; the last split takes what the expected lengths did not foresee.
struct KeyRange {
    int begin, end;
};
__device__ __forceinline__ KeyRange split_steps(int n, int split, const AttendP &A) {
    const int64_t b = (int64_t)split * A.split_steps, e = b + A.split_steps;
    return {(int)min(b, (int64_t)n), split == A.splits - 1 ? n : (int)min(e, (int64_t)n)};
}

// The table's entry for key j (anything below 2^62; a table has at least one column where there are keys).  No branch: it is loaded
// in any case, from a column that exists, and looked at only when the key's rows are loaded, a step later: a check beside the load
// waited for it, and with it for every row on its way.
__device__ __forceinline__ int page_entry(const KvView &V, int seq, int64_t j) {
    const int64_t col = min(max(j, (int64_t)0) >> V.shift, (int64_t)V.table_cols - 1);
    return V.table[seq * V.table_stride + col];
}

// ------------------------------------------------------------------------------------------------------------------------
// Tiles of 16 rows: four waves take every fourth step of 32 keys; no wave waits for another before the end.  The next step's
// rows are on their way while one is computed, their table entries were loaded a step before (a key per lane).
//
// Bound: HBM bytes of the keys and values, once the workgroups fill the card.  A lane loads 16 bytes (8-bit caches: two fragments'
// worth, the dims permuted alike in q), 8 such loads in flight; rows go to LDS only for the transposing reads of V.  The step is one
// body for whole and masked steps (two of them took 240 registers and a third of the waves), values that are not finite are left
// to the end.  e4m3, 64 streams of 100 - 1500 keys, 20 heads of 64: 32.5 us, 4.3 TB/s (a copy reaches 4.7); int8, 8 streams of 9 - 33 k
// keys, 32 heads on 8 of 128: 87 us, 4.1 TB/s, and 5 us for joining the splits; one stream of 224 keys: 6.5 us, launch and four
// trips to memory one after the other (lengths, table, rows, result).
// ------------------------------------------------------------------------------------------------------------------------
constexpr int RS = 32;      // keys per step
constexpr int RW = 4;       // waves
constexpr int VPAD = 16;    // V rows in LDS: 16 elements of padding put 8 consecutive rows on different banks for the transposing reads

template <int KIND, int DH>
__global__ __launch_bounds__(64 * RW, DH == 64 ? 4 : 3) void attend_rows_kernel(AttendP A) {
    constexpr int NS = DH / 32;        // 32-dim slices of the score product
    constexpr int ND = DH / 16;        // 16-dim tiles of the output
    constexpr int VLD = DH + VPAD;
    constexpr int EB = KIND == BF16 ? 2 : 1;
    constexpr int NL = DH * EB / 64;   // 16-byte loads of a lane per row
    constexpr int FL = NS / NL;        // fragments (8 elements) in each
    __shared__ __attribute__((aligned(16))) union {
        bf16_t vt[RW][RS * VLD];
        float part[RW][16][DH + 4];
    } U;
    __shared__ float sc[RW][2 * RS], pw[RW][KIND == INT8 ? 1 : RS * 16];
    __shared__ float ml[RW][16][2];
    const KvView &V = A.V;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, g = lane >> 4;
    const int split = blockIdx.x % A.splits;
    const int hk = (blockIdx.x / A.splits) % V.n_kv_heads, tile = blockIdx.x / A.splits / V.n_kv_heads;
    Tile T;
    if (!find_tile(V, A.group, 16, tile, T)) return;
    const int seq = T.seq, first = T.first, row0 = T.row0, nq = T.nq;
    const int64_t p_base = (int64_t)T.kv_len - nq;  // position of the sequence's first row
    const int n_tile = min(16, nq * A.group - first);
    // this lane's row; lanes behind the tile's end repeat its last row and store nothing
    const int row = first + min(fr, n_tile - 1);
    const int tok = row / A.group, head = hk * A.group + row % A.group;
    const int64_t p = p_base + tok;
    const int64_t p_lo = p_base + first / A.group, p_hi = p_base + (first + n_tile - 1) / A.group;
    u32x4 qf[NS];
    {
        const bf16_t *qp = A.q + (row0 + tok) * A.q_row + head * A.q_head + 8 * FL * g;
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = *(const u32x4 *)(qp + s / FL * 32 * FL + 8 * (s % FL));
    }
    const KeySteps ks = key_steps<RS>(V, A.window, A.sinks, p_lo, p_hi);
    const KeyRange range = split_steps(ks.n, split, A);
    const int i0 = range.begin + wave, i1 = range.end;
    f32x4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    const char *kbase = V.k + hk * V.head_stride * EB + 16 * g, *vbase = V.v + hk * V.head_stride * EB + 16 * g;
    const float *sbase = (lane < RS ? V.ks : V.vs) + hk * V.s_head;
    struct Step {
        u32x4 k[2][NL], v[2][NL];
        float scale;
        unsigned dead;  // keys that no row sees, a bit each
    };
    // key lane & 31 of step i: its table entry, and from that its page, -1 when no row of the tile can see it
    auto entry_of = [&](int i) { return page_entry(V, seq, step_key<RS>(ks, i) + (lane & 31)); };
    auto page_of = [&](int i, int entry) -> int {
        const int64_t j = step_key<RS>(ks, i) + (lane & 31);
        const bool seen = (j < ks.hi) & !((A.window > 0) & (j <= p_lo - A.window) & (j >= A.sinks));
        return (seen & ((unsigned)entry < (unsigned)V.n_pages)) ? entry : -1;
    };
    // (rows that are not there come from page 0 and are dropped later)
    auto load = [&](Step &x, int i, int page) {
        const int64_t j = step_key<RS>(ks, i) + (lane & 31);
        const int pg = max(page, 0), r = (int)j & V.mask;
        const int64_t off = (pg * V.page_stride + r * V.row_stride) * EB;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int64_t at = __shfl(off, 16 * t + fr);
#pragma unroll
            for (int s = 0; s < NL; ++s) {
                x.k[t][s] = *(const u32x4 *)(kbase + at + 64 * s);
                x.v[t][s] = *(const u32x4 *)(vbase + at + 64 * s);
            }
        }
        if constexpr (KIND != BF16) x.scale = sbase[pg * V.s_page + r * V.s_row];  // lanes 0 .. 31 the keys', the others the values'
        x.dead = (unsigned)__ballot(page < 0);
    };
    // V rows (and scales) of a step -> LDS, keys that no row sees as zeros; whether one that some rows may not see is not finite
    auto put = [&](const Step &x, bool whole) {
        bool bad = false;
        if constexpr (KIND != BF16) sc[wave][lane] = x.scale;
        auto row = [&](int t, int c) { return (u32x4 *)&U.vt[wave][(16 * t + fr) * VLD + c / FL * 32 * FL + 8 * FL * g + 8 * (c % FL)]; };
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int c = 0; c < NS; ++c) *row(t, c) = fragment<KIND>(x.v[t][c / FL], c % FL);
        if (!whole) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if ((x.dead >> (16 * t + fr)) & 1) {
#pragma unroll
                    for (int c = 0; c < NS; ++c) *row(t, c) = u32x4{0, 0, 0, 0};
                }
            }
        }
        // (of a step that every row sees whole, too, where infinities can be: an infinity times a probability's residue is no number)
        if (KIND == BF16 || (KIND == E4M3 && !whole)) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                bool odd = false;
#pragma unroll
                for (int c = 0; c < NS; ++c) odd |= has_nonfinite(fragment<KIND>(x.v[t][c / FL], c % FL));
                bad |= odd & !((x.dead >> (16 * t + fr)) & 1);
            }
        }
        __builtin_amdgcn_wave_barrier();  // what other lanes of the wave read below is written above (LDS keeps a wave's order)
        return KIND != INT8 && __ballot(bad) != 0;
    };
    // scores (taken out of the result vectors at once: an element set under a branch there was compiled wrongly)
    auto scores = [&](const Step &x, float (&s)[2][4]) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < NS; ++c)
                a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fragment<KIND>(x.k[t][c / FL], c % FL)),
                                                            __builtin_bit_cast(bf16x8, qf[c]), a, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][r] = a[r] * (KIND == BF16 ? A.c : sc[wave][16 * t + 4 * g + r] * A.c);
        }
    };
    // the 32 keys this lane's row sees, a bit each
    auto visible = [&](unsigned dead, int64_t key0) {
        unsigned vis = ~dead & low_bits(p - key0 + 1);
        if (A.window > 0) vis &= ~low_bits(p - A.window - key0 + 1) | low_bits((int64_t)A.sinks - key0);
        return vis;
    };
    // running maximum and sum; s becomes the values' weights
    auto softmax = [&](float (&s)[2][4], unsigned vis) {
        const unsigned mine = vis >> (4 * g);  // bit 16 t + r: the lane's key r of tile t
        float mx = m;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[t][r] = mine & (1u << (16 * t + r)) ? s[t][r] : -INFINITY;
                mx = fmaxf(mx, s[t][r]);
            }
        mx = xor_max<32>(xor_max<16>(mx));
        const float ref = mx == -INFINITY ? 0.0f : mx;  // nothing seen so far: exp2(-inf - 0) = 0
        const float corr = __builtin_amdgcn_exp2f(m - ref);
        m = mx;
        float ps = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = __builtin_amdgcn_exp2f(s[t][r] - ref);
                ps += e;
                // (the scale of a value that is not seen may be anything)
                if constexpr (KIND == BF16) s[t][r] = e;
                else s[t][r] = mine & (1u << (16 * t + r)) ? e * sc[wave][RS + 16 * t + 4 * g + r] : 0.0f;
            }
        l = l * corr + ps;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] *= corr;
    };
    // one step; whole: every row sees every key of it.  x takes the next step's rows as soon as this one's are used.
    int entry = 0;  // of the step after next
    bool left = false;  // steps with values that are not finite and that some rows do not see: done at the end
    auto step = [&](Step &x, bool whole, int64_t key0, int next) {
        unsigned dead = x.dead;
        float s[2][4];
        if (put(x, whole)) {
            left = true;
            whole = false;
            dead = ~0u;  // (as if no row saw it)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int c = 0; c < NS; ++c)
                    *(u32x4 *)&U.vt[wave][(16 * t + fr) * VLD + c / FL * 32 * FL + 8 * FL * g + 8 * (c % FL)] = u32x4{0, 0, 0, 0};
            __builtin_amdgcn_wave_barrier();
        }
        scores(x, s);
        const int at = min(next, i1 - 1);
        load(x, at, page_of(at, entry));
        entry = entry_of(next + RW);
        softmax(s, whole ? ~0u : visible(dead, key0));
        // the residue of the probabilities' rounding goes through a second product: these kernels wait for memory, not for the MFMAs
        const u32x4 pb = {pack_bf16(s[0][0], s[0][1]), pack_bf16(s[0][2], s[0][3]), pack_bf16(s[1][0], s[1][1]), pack_bf16(s[1][2], s[1][3])};
        const u32x4 pl = low_part(&s[0][0], pb);
        const bf16_t *vb = &U.vt[wave][(4 * g + (fr >> 2)) * VLD + (fr & 3) * 4];
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const u32x2 a0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vb + 16 * d)));
            const u32x2 a1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vb + 16 * VLD + 16 * d)));
            const u32x4 a = {a0.x, a0.y, a1.x, a1.y};
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, pb), o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, pl), o[d], 0, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();  // the next step's rows come after this one's reads
    };
    if (i0 < i1) {
        Step x;
        load(x, i0, page_of(i0, entry_of(i0)));
        entry = entry_of(i0 + RW);
        auto whole = [&](int64_t key0) {
            return x.dead == 0 && key0 + RS - 1 <= p_lo && (A.window <= 0 || key0 > p_hi - A.window || key0 + RS <= A.sinks);
        };
        for (int i = i0; i < i1; i += RW) {
            const int64_t key0 = step_key<RS>(ks, i);
            step(x, whole(key0), key0, i + RW);
        }
        if (KIND != INT8 && left) {
            // 0 x inf = NaN in a product over rows that do and rows that do not see a value: key by key, rows that see it only
#pragma unroll 1
            for (int i = i0; i < i1; i += RW) {
                const int64_t key0 = step_key<RS>(ks, i);
                load(x, i, page_of(i, entry_of(i)));
                if (!put(x, whole(key0))) continue;
                const unsigned vis = visible(x.dead, key0);
                float s[2][4];
                scores(x, s);
                softmax(s, vis);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) pw[wave][(16 * t + 4 * g + r) * 16 + fr] = s[t][r];
                __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                for (int k = 0; k < RS; ++k) {
                    const float pk = pw[wave][k * 16 + fr];
                    const bf16_t *vrow = &U.vt[wave][k * VLD + 4 * g];
                    const bool ok = (vis >> k) & 1;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float y = fmaf(pk, __uint_as_float((unsigned)vrow[16 * d + e] << 16), o[d][e]);
                            o[d][e] = ok ? y : o[d][e];
                        }
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
    }
    l = xor_sum<32>(xor_sum<16>(l));
    // join the four waves
    if (g == 0) {
        ml[wave][fr][0] = m;
        ml[wave][fr][1] = l;
    }
    __syncthreads();
    float M = ml[0][fr][0];
#pragma unroll
    for (int w = 1; w < RW; ++w) M = fmaxf(M, ml[w][fr][0]);
    const float ref = M == -INFINITY ? 0.0f : M;
    const float f = __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
    for (int d = 0; d < ND; ++d) *(f32x4 *)&U.part[wave][fr][16 * d + 4 * g] = o[d] * f;
    __syncthreads();
    // 256 threads: row threadIdx / 16, DH / 16 dims each
    constexpr int E = DH / 16;
    const int r = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * E;
    if (r >= n_tile) return;
    float Mr = ml[0][r][0];
#pragma unroll
    for (int w = 1; w < RW; ++w) Mr = fmaxf(Mr, ml[w][r][0]);
    const float rr = Mr == -INFINITY ? 0.0f : Mr;
    float L = 0.0f, acc[E] = {};
#pragma unroll
    for (int w = 0; w < RW; ++w) {
        L += ml[w][r][1] * __builtin_amdgcn_exp2f(ml[w][r][0] - rr);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += U.part[w][r][d0 + e];
    }
    const int rw = first + r, tk = rw / A.group, hd = hk * A.group + rw % A.group;
    if (A.splits == 1) {
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        bf16_t *op = A.out + (row0 + tk) * A.o_row + hd * A.o_head + d0;
#pragma unroll
        for (int e = 0; e < E; e += 2) *(unsigned *)(op + e) = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
    } else {
        const int64_t at = ((int64_t)split * V.n_rows + row0 + tk) * A.n_heads + hd;
#pragma unroll
        for (int e = 0; e < E; e += 4) *(f32x4 *)(A.ws_o + at * DH + d0 + e) = f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
        if ((threadIdx.x & 15) == 0) *(f32x2 *)(A.ws_ml + at * 2) = f32x2{Mr, L};
    }
}

// ------------------------------------------------------------------------------------------------------------------------
// Tiles of 128 rows for chunks: four waves of 32 rows share steps of 64 keys, double-buffered in LDS.  KW = 2: tiles of 64 rows, two
// waves for the same 32, each with half of a step's keys; their results are joined at the end as splits are.
//
// 32 x 32 x 16 products: lane (row = l & 31, h = l >> 5) holds of a block of 32 keys the scores of keys 8 b + 4 h + r (b, r = 0 .. 3),
// so a row's maximum and sum are completed by one exchange with lane ^ 32, and the probabilities of 16 keys are a fragment
// of P^T if the contraction index is ordered (h, b, r) — the order two transposing reads give V^T in.
// The next step's rows are on their way while one is computed: bf16 rows directly to LDS, 8-bit ones through registers (their codes
// become bf16 there); their table entries are loaded one step earlier still, a key per lane.
//
// Bound: the issue of the softmax's 5 operations a score beside the matrix products (which alone keep a wave busy for 40 % of a
// step), so two or three workgroups a compute unit, one's softmax under another's products.  2048 tokens behind 14336, 32 heads on
// 8 of 128, bf16: 555 - 585 us from card to card, 0.9 PFLOP/s (a plain product of 8192 cubed reaches 1.38; calls back to back: traced
// launches take 586 - 764); with rows through registers and pages looked up beside their loads it was 640 where it is 555 now.  8-bit
// caches, whose codes each tile converts for itself: e4m3 688 us, int8 889 (a second product with the values) where bf16 takes 572.  One half's exponents under the other's products took more registers than there are.  8 prompts
// of 17 - 448 tokens, 20 heads of 64: 32 us (64-row tiles), the longest tile's 23 steps.
// ------------------------------------------------------------------------------------------------------------------------
constexpr int CR = 128, CK = 64;  // rows, keys per step
using gptr_t = const __attribute__((address_space(1))) void *;
using lptr_t = __attribute__((address_space(3))) void *;
// Asks the scheduler for an order of a block's LDS reads and products: AHEAD products' reads first (READS each), then a product and the
// reads of the one AHEAD of it.  Left alone it reads a fragment, waits the whole LDS latency and multiplies.
template <int PRODUCTS, int READS, int AHEAD> __device__ __forceinline__ void pipeline_reads() {
    __builtin_amdgcn_sched_group_barrier(0x100, READS * AHEAD, 0);
#pragma unroll
    for (int i = 0; i < PRODUCTS - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}
using f32x16 = __attribute__((ext_vector_type(16))) float;

template <int KIND, int DH, int KW>
__global__ __launch_bounds__(256, DH == 64 && KIND == BF16 ? 3 : 2) void attend_chunk_kernel(AttendP A) {
    // Row strides in LDS.  8-bit rows pass through registers (their codes become bf16) and are padded; bf16 rows go to LDS
    // directly, 1 KB a wave and load, which leaves no room for padding: the 16-byte pieces of a row are permuted instead.
    constexpr bool DIRECT = KIND == BF16;
    constexpr int KLD = DIRECT ? DH : DH + 8, VLD = DIRECT ? DH : DH + 16;
    constexpr int ROWS = CR / KW, NT = 2 / KW;  // rows of the tile, blocks of 32 keys a wave has of a step
    constexpr int ND = DH / 32;
    constexpr int EB = KIND == BF16 ? 2 : 1;
    constexpr int LPR = DH / 8, RPP = 256 / LPR, NP = CK / RPP;  // lanes per row, rows per pass, passes
    using raw_t = typename Raw<KIND>::type;
    // (one object: the compiler waits for loads on their way to one shared array before it reads any other)
    __shared__ __attribute__((aligned(1024))) struct {
        bf16_t kt[2][CK * KLD], vt[2][CK * VLD];
        float sc[2][2][CK];
        int odd[2];  // the step whose values in a buffer are not all finite
    } L;
    auto &kt = L.kt;
    auto &vt = L.vt;
    auto &sc = L.sc;
    auto &odd = L.odd;
    const KvView &V = A.V;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 31, h = lane >> 5;
    const int wr = KW == 1 ? wave : wave & 1, mine0 = KW == 1 ? 0 : (wave >> 1) * 32;  // the wave's rows (32 of them), its first key of a step
    // tiles with the most keys first: in a chunk the later ones
    const int hk = blockIdx.x % V.n_kv_heads, rest = blockIdx.x / V.n_kv_heads;
    const int split = rest % A.splits, tile = A.tiles - 1 - rest / A.splits;
    Tile T;
    if (!find_tile(V, A.group, ROWS, tile, T)) return;
    const int seq = T.seq, first = T.first, row0 = T.row0, nq = T.nq;
    const int64_t p_base = (int64_t)T.kv_len - nq;
    const int n_tile = min(ROWS, nq * A.group - first);
    const int row = first + min(wr * 32 + fr, n_tile - 1);
    const int tok = row / A.group, head = hk * A.group + row % A.group;
    const int64_t p = p_base + tok;
    const int64_t p_lo = p_base + first / A.group, p_hi = p_base + (first + n_tile - 1) / A.group;
    u32x4 qf[DH / 16];
    {
        const bf16_t *qp = A.q + (row0 + tok) * A.q_row + head * A.q_head + 8 * h;
#pragma unroll
        for (int s = 0; s < DH / 16; ++s) qf[s] = *(const u32x4 *)(qp + 16 * s);
    }
    const KeySteps ks = key_steps<CK>(V, A.window, A.sinks, p_lo, p_hi);
    const KeyRange range = split_steps(ks.n, split, A);
    const int i0 = range.begin, i1 = range.end;
    f32x16 o[DH / 32];
#pragma unroll
    for (int d = 0; d < DH / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    const int srow = tid / LPR, sub = tid % LPR;
    const bool busy = wr * 32 < n_tile;  // a wave without rows only loads
    // key `lane` of step i: its table entry, and from that its page, -1 when no row of the tile can see it
    auto entry_of = [&](int i) { return page_entry(V, seq, step_key<CK>(ks, i) + lane); };
    auto page_of = [&](int i, int entry) -> int {
        const int64_t j = step_key<CK>(ks, i) + lane;
        const bool seen = (j < ks.hi) & !((A.window > 0) & (j <= p_lo - A.window) & (j >= A.sinks));
        return (seen & ((unsigned)entry < (unsigned)V.n_pages)) ? entry : -1;
    };
    // whether every row of the tile sees every key of the step at key0 (pages apart)
    auto all_see = [&](int64_t key0) { return key0 + CK - 1 <= p_lo && (A.window <= 0 || key0 > p_hi - A.window || key0 + CK <= A.sinks); };
    // The piece (16 bytes) of row r that lies in slot s is s ^ turn(r): 16 rows' pieces of one dim lie on different banks (score
    // products), and so do the 4 pieces of 8 rows that a transposing read takes.
    auto turn = [](int r) { return DH == 128 ? (r & 3) << 2 | ((r >> 2) & 3) : ((r >> 1) & 1) << 2 | ((r >> 2) & 3); };
    raw_t rk[DIRECT ? 1 : NP], rv[DIRECT ? 1 : NP];
    float rs = 0.0f;
    const int piece = DIRECT ? (lane % LPR) ^ turn(wave * (64 / LPR) + lane / LPR) : sub;  // (the same in every pass: rows 16 or 32 apart)
    const char *kbase = V.k + (hk * V.head_stride + piece * 8) * EB, *vbase = V.v + (hk * V.head_stride + piece * 8) * EB;
    const float *sbase = (wave ? V.vs : V.ks) + hk * V.s_head;
    // rows of the step at key0 (those that are not there from page 0: they are dropped before they are used)
    auto load = [&](int64_t key0, int page, int buf) {
        const int pg = max(page, 0), j = (int)(key0 + lane) & V.mask;
        const int64_t off = (pg * V.page_stride + j * V.row_stride) * EB;
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            const int64_t at = __shfl(off, s * RPP + srow);
            if constexpr (DIRECT) {
                const int row1 = s * RPP + wave * (64 / LPR);  // the wave's first row
                __builtin_amdgcn_global_load_lds((gptr_t)(kbase + at), (lptr_t)&kt[buf][row1 * DH], 16, 0, 0);
                __builtin_amdgcn_global_load_lds((gptr_t)(vbase + at), (lptr_t)&vt[buf][row1 * DH], 16, 0, 0);
            } else {
                rk[s] = *(const raw_t *)(kbase + at);
                rv[s] = *(const raw_t *)(vbase + at);
            }
        }
        if constexpr (!DIRECT) {  // waves 0 and 1: the keys' and the values' scales, a key per lane
            if (wave < 2) rs = sbase[pg * V.s_page + j * V.s_row];
        }
    };
    // 8-bit rows: registers -> LDS, keys that no row sees as zeros; mark: the step, if some row may not see some key of it (the same
    // steps here and at the end: what one leaves out the other adds)
    auto store = [&](int buf, int mark, unsigned long long gone) {
        bool bad = false;
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            const int r = s * RPP + srow;
            *(u32x4 *)&kt[buf][r * KLD + sub * 8] = to_bf16<KIND>(rk[s]);
            u32x4 x = to_bf16<KIND>(rv[s]);
            if (gone != 0) {
                const bool out = (gone >> r) & 1;
#pragma unroll
                for (int q = 0; q < 4; ++q) x[q] = out ? 0 : x[q];
            }
            if (KIND != INT8 && mark >= 0) bad |= has_nonfinite(x);
            *(u32x4 *)&vt[buf][r * VLD + sub * 8] = x;
        }
        if (wave < 2) sc[buf][wave][lane] = rs;
        if (KIND != INT8 && bad) odd[buf] = mark;
    };
    // bf16 rows of a step that not every row sees whole: the same, done in LDS
    auto mend = [&](int buf, int mark, unsigned long long gone) {
        const int r = tid >> 2;
        bf16_t *vr = &vt[buf][r * DH + (tid & 3) * (DH / 4)];
        bool bad = false;
#pragma unroll
        for (int q = 0; q < DH / 32; ++q) {
            if ((gone >> r) & 1) *(u32x4 *)(vr + 8 * q) = u32x4{0, 0, 0, 0};
            else bad |= has_nonfinite(*(const u32x4 *)(vr + 8 * q));
        }
        if (bad) odd[buf] = mark;
    };
    // what is on its way to LDS is there, for every wave, and every wave is done with what it read before
    auto arrived = [&]() {
        if constexpr (DIRECT) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    if (tid < 2) odd[tid] = -1;
    int entry = 0;  // of the next step
    unsigned long long dead = 0, dead_n = 0;
    if (i0 < i1) {
        const int64_t key0 = step_key<CK>(ks, i0);
        const int page = page_of(i0, entry_of(i0));
        dead = __ballot(page < 0);
        load(key0, page, 0);
        entry = entry_of(i0 + 1);
        if constexpr (!DIRECT) {
            __syncthreads();
            store(0, dead == 0 && all_see(key0) ? -1 : i0, dead);
        }
    }
    arrived();
    // s: weights of the values of a step, with the running maximum and sum.  MASKED: some row may not see some key of it, vis gets
    // the keys this lane's row sees; hide: none does
    auto weights = [&](auto masked, int cur, int64_t key0, bool hide, float (&s)[NT][16], unsigned (&vis)[NT]) {
        constexpr bool MASKED = decltype(masked)::value;
        // byte of row fr's first fragment; piece 2 c + h of a direct row is at slot (2 c + h) ^ turn(fr): an exclusive or with 32 c
        const char *kb = (const char *)kt[cur] + (mine0 + fr) * KLD * 2;
        const int k0 = DIRECT ? (h ^ turn(fr)) * 16 : h * 16;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f32x16 a;
#pragma unroll
            for (int r = 0; r < 16; ++r) a[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < DH / 16; ++c) {
                const u32x4 kf = *(const u32x4 *)(kb + 32 * t * KLD * 2 + (DIRECT ? k0 ^ (32 * c) : k0 + 32 * c));
                a = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kf), __builtin_bit_cast(bf16x8, qf[c]), a, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[t][r] = a[r];
        }
        pipeline_reads<NT * (DH / 16), 1, 4>();
        if constexpr (KIND != BF16) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f32x4 f = *(const f32x4 *)&sc[cur][0][mine0 + 32 * t + 8 * b + 4 * h];
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[t][4 * b + r] *= f[r];
                }
        }
        if constexpr (MASKED) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int64_t k1 = key0 + mine0 + 32 * t;
                unsigned v = hide ? 0u : ~(unsigned)(dead >> (mine0 + 32 * t)) & low_bits(p - k1 + 1);
                if (A.window > 0) v &= ~low_bits(p - A.window - k1 + 1) | low_bits((int64_t)A.sinks - k1);
                vis[t] = v;
                const unsigned mine = v >> (4 * h);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[t][r] = mine & (1u << (8 * (r >> 2) + (r & 3))) ? s[t][r] : -INFINITY;
            }
        }
        // running maximum (of the unscaled scores; the scale rides in the exponent's fma)
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[t][r]);
        mx = xor_max<32>(mx);
        // the reference follows the maximum only when that has left it by more than 2^8 (probabilities stay below 256, their
        // relative roundings are the same): rescaling the result at every new maximum of one of 32 rows cost a quarter of a step
        if (__ballot((mx - m) * A.c > 8.0f || (m == -INFINITY && mx > m))) {
            const float nm = fmaxf(mx, m), base = nm == -INFINITY ? 0.0f : nm;
            const float corr = __builtin_amdgcn_exp2f((m - base) * A.c);
            m = nm;
            l *= corr;
#pragma unroll
            for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= corr;
        }
        const float ref = m == -INFINITY ? 0.0f : -m * A.c;
        float ps = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[t][r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], A.c, ref));
                ps += s[t][r];
            }
        l += ps;
        if constexpr (KIND != BF16) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f32x4 f = *(const f32x4 *)&sc[cur][1][mine0 + 32 * t + 8 * b + 4 * h];
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[t][4 * b + r] *= f[r];
                }
            if (MASKED) {  // (the scale of a value that is not seen may be anything)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[t][r] = (vis[t] >> (4 * h)) & (1u << (8 * (r >> 2) + (r & 3))) ? s[t][r] : 0.0f;
            }
        }
    };
    auto products = [&](int cur, const float (&s)[NT][16]) {
        const int gi = lane >> 4, ii = lane & 15, r0 = 4 * h + (ii >> 2), q0 = 2 * (gi & 1) + ((ii & 3) >> 1);
        // byte of dims 32 d + .. of row 16 c + 8 e + r0: e and d turn the slot of a direct row by 32 e and 64 d bytes
        const char *va = (const char *)vt[cur] + (mine0 + r0) * VLD * 2;
        const int v0 = (DIRECT ? (q0 ^ turn(r0)) : q0) * 16 + (ii & 1) * 8;
        auto fragments = [&](int c, u32x4 (&f)[ND]) {
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                u32x2 x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    x[e] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                         (lds_s16x4 *)(va + (16 * c + 8 * e) * VLD * 2 + (DIRECT ? v0 ^ (64 * d + 32 * e) : v0 + 64 * d))));
                f[d] = u32x4{x[0].x, x[0].y, x[1].x, x[1].y};
            }
        };
        // a wave that multiplies goes before one at its softmax, which fills the gaps (570 -> 555 us; the scores' products raised as
        // well, or the softmax instead: 565; for int8 the order it gives the code spills)
        if constexpr (KIND == BF16) __builtin_amdgcn_s_setprio(1);
        u32x4 f[2][ND];
        fragments(0, f[0]);
#pragma unroll
        for (int c = 0; c < 2 * NT; ++c) {
            if (c < 2 * NT - 1) fragments(c + 1, f[(c + 1) & 1]);
            const float *e = &s[c >> 1][8 * (c & 1)];
            const u32x4 pb = {pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]), pack_bf16(e[4], e[5]), pack_bf16(e[6], e[7])};
            // A probability rounded to bf16 is off by at most 2^-8 of itself, as the result is when it is rounded: against the formula in 64
            // bits the result is then off by 0.0020 - 0.0023 of its size, and by 0.0017 with the residue in a second product, which the
            // 16-row kernel, waiting for memory, has for nothing.  Here it takes the chunk above from 555 to 745 us,
            // the prompts from 30 to 33, chunks of 600 - 1777 rows under a window of 512 from 32 to 37.
            u32x4 pl = {0, 0, 0, 0};
            if constexpr (KIND == INT8) pl = low_part(e, pb);  // (a code's scale leaves the largest weight no power of two: its rounding would show)
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f[c & 1][d]), __builtin_bit_cast(bf16x8, pb), o[d], 0, 0, 0);
                if constexpr (KIND == INT8)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f[c & 1][d]), __builtin_bit_cast(bf16x8, pl), o[d], 0, 0, 0);
            }
        }
        pipeline_reads<2 * NT * ND, 2, ND>();
        if constexpr (KIND == BF16) __builtin_amdgcn_s_setprio(0);
    };
    bool left = false;  // steps with values that are not finite and that some rows do not see: done at the end
    int i = i0, cur = 0;
    // the next step's rows on their way to the other buffer (last read before the previous barrier), this step
    auto advance = [&](auto masked) {
        const int64_t key0 = step_key<CK>(ks, i);
        const bool more = i + 1 < i1;
        const int64_t key1 = step_key<CK>(ks, more ? i + 1 : i);
        if (more) {
            const int page = page_of(i + 1, entry);
            dead_n = __ballot(page < 0);
            load(key1, page, cur ^ 1);
            entry = entry_of(i + 2);
        }
        if constexpr (DIRECT && decltype(masked)::value) {
            mend(cur, i, dead);
            // (not __syncthreads, which would wait for the next step's rows as well)
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        const bool hide = KIND != INT8 && decltype(masked)::value && odd[cur] == i;
        left |= hide;  // (in every wave: all of them load at the end)
        if (busy) {
            float s[NT][16];
            unsigned vis[NT];
            weights(masked, cur, key0, hide, s, vis);
            if (!hide) products(cur, s);
        }
        if constexpr (!DIRECT) {
            if (more) store(cur ^ 1, dead_n == 0 && all_see(key1) ? -1 : i + 1, dead_n);
        }
        dead = dead_n;
        cur ^= 1;
        ++i;
        arrived();
    };
    // steps that every row sees whole run in a loop of their own: with the masks' code in it the compiler kept two copies of the
    // result and spilled
    while (i < i1) {
        while (i < i1 && dead == 0 && all_see(step_key<CK>(ks, i))) advance(std::false_type{});
        if (i < i1) advance(std::true_type{});
    }
    if (KIND != INT8 && left) {
        // 0 x inf = NaN in a product over rows that do and rows that do not see a value: key by key, rows that see it only
#pragma unroll 1
        for (i = i0; i < i1; ++i) {
            const int64_t key0 = step_key<CK>(ks, i);
            const int pg = page_of(i, entry_of(i));
            dead = __ballot(pg < 0);
            if (dead == 0 && all_see(key0)) continue;
            load(key0, pg, 0);
            arrived();
            if constexpr (DIRECT) mend(0, i, dead);
            else store(0, i, dead);
            __syncthreads();
            if (odd[0] == i) {
                float s[NT][16];
                unsigned vis[NT];
                weights(std::true_type{}, 0, key0, false, s, vis);
#pragma unroll 1
                for (int k = 0; k < 32 * NT; ++k) {
                    const int at = (k >> 5) * 16 + ((k >> 3) & 3) * 4 + (k & 3);  // the key among the wave's 16 NT of its half
                    float mine = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16 * NT; ++e) mine = at == e ? s[e >> 4][e & 15] : mine;
                    const float other = __shfl_xor(mine, 32), pk = ((k >> 2) & 1) == h ? mine : other;
                    const bool ok = (vis[NT == 1 ? 0 : k >> 5] >> (k & 31)) & 1;
                    const bf16_t *vrow = vt[0] + (mine0 + k) * VLD;
#pragma unroll
                    for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            const int dim = 32 * d + 8 * (q >> 2) + 4 * h + (q & 3);
                            const int at_dim = DIRECT ? ((dim >> 3) ^ turn(k)) * 8 + (dim & 7) : dim;
                            const float x = fmaf(pk, __uint_as_float((unsigned)vrow[at_dim] << 16), o[d][q]);
                            o[d][q] = ok ? x : o[d][q];
                        }
                }
            }
            __syncthreads();
        }
    }
    l += __shfl_xor(l, 32);
    if constexpr (KW == 2) {  // the two waves of the same rows: the second gives its part to the first (every wave is done with the rows in LDS)
        float *x = (float *)&L + wr * 64 * (DH / 2 + 2) + lane;
        if (mine0) {
#pragma unroll
            for (int e = 0; e < DH / 2; ++e) x[64 * e] = o[e >> 4][e & 15];
            x[64 * (DH / 2)] = m;
            x[64 * (DH / 2 + 1)] = l;
        }
        __syncthreads();
        if (mine0) return;
        const float m2 = x[64 * (DH / 2)], l2 = x[64 * (DH / 2 + 1)];
        const float nm = fmaxf(m, m2), base = nm == -INFINITY ? 0.0f : nm;
        const float f1 = __builtin_amdgcn_exp2f((m - base) * A.c), f2 = __builtin_amdgcn_exp2f((m2 - base) * A.c);
#pragma unroll
        for (int e = 0; e < DH / 2; ++e) o[e >> 4][e & 15] = o[e >> 4][e & 15] * f1 + x[64 * e] * f2;
        l = l * f1 + l2 * f2;
        m = nm;
    }
    if (wr * 32 + fr >= n_tile) return;
    const bool part = A.splits > 1;
    const float inv = part ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t at = ((int64_t)split * V.n_rows + row0 + tok) * A.n_heads + head;
    bf16_t *op = A.out + (row0 + tok) * A.o_row + head * A.o_head + 4 * h;
#pragma unroll
    for (int d = 0; d < DH / 32; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const f32x4 x = {o[d][4 * b] * inv, o[d][4 * b + 1] * inv, o[d][4 * b + 2] * inv, o[d][4 * b + 3] * inv};
            if (part) *(f32x4 *)(A.ws_o + at * DH + 32 * d + 8 * b + 4 * h) = x;
            else *(u32x2 *)(op + 32 * d + 8 * b) = u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
        }
    // (the join takes maxima in scaled units)
    if (part && h == 0) *(f32x2 *)(A.ws_ml + at * 2) = f32x2{m * A.c, l};
}

// Joins the splits of a row: one wave per (row, head).  Splits without keys have l = 0 and m = -inf.  Nothing here but latency
// counts (a few hundred KB): a lane has four dims of every second (fourth) split, the loads of four of them at once.
constexpr int MAX_SPLITS = 64;
template <int DH>
__global__ __launch_bounds__(64) void attend_join_kernel(AttendP A) {
    constexpr int LP = DH / 4, G = 64 / LP;  // lanes of a split's row, splits at a time
    const int lane = threadIdx.x, d = lane % LP * 4, g = lane / LP;
    const int t = blockIdx.x / A.n_heads, h = blockIdx.x % A.n_heads;
    const int64_t item = blockIdx.x, step = (int64_t)A.V.n_rows * A.n_heads;
    float m = -INFINITY, l = 0.0f;
    if (t < A.V.cu[0] || t >= A.V.cu[A.V.n_seqs]) return;  // a row of no sequence
    if (lane < A.splits) {
        const f32x2 x = *(const f32x2 *)(A.ws_ml + (item + lane * step) * 2);
        m = x.x;
        l = x.y;
    }
    const float M = wave_max_desc(m);
    const float f = __builtin_amdgcn_exp2f(m - (M == -INFINITY ? 0.0f : M));
    const float L = wave_sum_desc(l * f);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < A.splits; s0 += 4 * G) {
        f32x4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *(const f32x4 *)(A.ws_o + (item + min(s0 + i * G + g, A.splits - 1) * step) * DH + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = s0 + i * G + g;
            const float fs = __shfl(f, s & 63);
            const f32x4 y = acc + fs * x[i];
            if (s < A.splits) acc = y;
        }
    }
#pragma unroll
    for (int o = 32; o >= LP; o >>= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    if (g == 0) *(u32x2 *)(A.out + t * A.o_row + h * A.o_head + d) = u32x2{pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv)};
}

// How a call is cut up; the workspace and the launch agree because both ask here.
struct Plan {
    int rows;  // of a tile
    int64_t tiles;
    int splits, steps;  // splits of a tile's keys, steps of each
};
Plan plan(int n_cus, const mw_kv_cache &c, const mw_kv_batch &b, int n_heads, int window, int sinks) {
    Plan p;
    const int group = n_heads / c.n_kv_heads;
    const int longest = b.max_rows > 0 ? std::min(b.max_rows, b.n_rows) : ceil_div(b.n_rows, b.n_seqs);
    // Where several tiles of 16 rows, that read the keys again from L2, and one of 64 (bf16) or 128, mostly empty, meet.  bf16, us with
    // tiles of 16 / 64: 16 rows 22 / 21 and 42 / 43 (8 sequences of 1500 keys and 48 of 1000; 20 heads of 64), 32 rows 30 / 21 and
    // 75 / 43.  8 bits, whose codes a larger tile converts for itself, 16 / 128: 48 rows 26 / 32 and 58 / 82, 64 rows 30 / 33 and
    // 70 / 82, 96 rows 33 / 37 and 103 / 85 (e4m3); on 8 heads of 128 (int8) 48 rows 25 / 30 and 52 / 60, 64 rows 27 / 32 and 61 / 60,
    // 96 rows 35 / 34 and 86 / 62.
    const int64_t rows = (int64_t)longest * group;
    const bool chunk = rows > (c.dtype == BF16 ? 16 : 64);
    // workgroups of the tiles that hold rows when the sequences are as expected.  (Not fewer than the rows fill: with a max_rows that
    // is too small the splits, and the workspace, would grow with the rows.)
    auto expected = [&](int tile) {
        const int64_t seqs = std::min(b.n_seqs, b.n_rows), full = (int64_t)b.n_rows * group / tile;
        return std::max<int64_t>(1, std::max(full, std::min(full + seqs, seqs * ceil_div<int64_t>(rows, tile))) * c.n_kv_heads);
    };
    p.rows = chunk ? CR : 16;
    // Tiles of 64 rows: the two waves of the same rows share the keys of a step, the chain of steps is half as long and the keys are
    // read twice.  Where a tile of 128 is half empty anyway (64 rows, 48 sequences: 57 -> 47 us, on heads of 128 41 -> 36), and for heads
    // of 64 where all fit at once (8 prompts of 17 - 448 rows: 36 -> 32 us; three chunks of 600 - 1777 rows, that do not: 34 -> 37; heads
    // of 128, 96 and 128 rows: 26 -> 27, 29 -> 29; e4m3, whose codes are converted twice as well: 37 -> 43).
    if (chunk && c.dtype == BF16 && (rows <= CR / 2 || (c.head_dim == 64 && expected(CR / 2) <= 3 * (int64_t)n_cus))) p.rows = CR / 2;
    p.tiles = (int64_t)b.n_rows * group / p.rows + b.n_seqs;
    const int64_t wgs = expected(p.rows);
    int64_t keys = std::max(b.max_kv, 1);
    if (window > 0) keys = std::min<int64_t>(keys, (int64_t)window + sinks + std::min<int64_t>(longest, p.rows));
    const int64_t steps = ceil_div<int64_t>(keys, chunk ? CK : RS), least = chunk ? 8 : 4 * RW;
    // Workgroups a compute unit.  16-row tiles: three fit.  Under a window all have the same keys and one full round is best (32
    // streams, 8 heads, window 2048: 33 us with three, 37 with four or more); without one the lengths differ, and more and shorter
    // ones even out (8 streams of 9 - 33 k keys: 103 us with four, 94 with six, 93 with eight).  Chunks: two (8 prompts of 17 -
    // 448 rows in tiles of 128: 36 us with one to three, 42 with four: partial results cost more than shorter workgroups give).
    const int64_t per_cu = chunk ? 2 : window > 0 ? 3 : 6;
    const int64_t want = std::min<int64_t>(per_cu * n_cus / wgs, MAX_SPLITS);
    p.splits = (int)std::max<int64_t>(1, std::min(want, steps / least));
    p.steps = (int)ceil_div<int64_t>(steps, p.splits);
    return p;
}
size_t plan_bytes(const Plan &p, const mw_kv_cache &c, const mw_kv_batch &b, int n_heads) {
    return p.splits == 1 ? 0 : (size_t)p.splits * b.n_rows * n_heads * (c.head_dim + 2) * sizeof(float);
}

}  // namespace

size_t kv_attend_workspace(int n_cus, const mw_kv_cache &c, const mw_kv_batch &b, int n_heads, int window, int sinks) {
    check_kv(c, b);
    MW_CHECK(n_heads > 0 && n_heads % c.n_kv_heads == 0, "kv attend: n_heads is a multiple of n_kv_heads");
    if (b.n_rows == 0 || b.n_seqs == 0) return 0;
    MW_CHECK(window >= 0 && sinks >= 0, "kv attend: window and sinks are not negative");
    return plan_bytes(plan(n_cus, c, b, n_heads, window, sinks), c, b, n_heads);
}

void check_kv_attend(const mw_kv_cache &c, const mw_kv_batch &b, const KvAttendArgs &a) {
    check_kv(c, b);
    MW_CHECK(a.n_heads > 0 && a.n_heads % c.n_kv_heads == 0, "kv attend: n_heads is a multiple of n_kv_heads");
    MW_CHECK(a.scale > 0.0f && a.scale < INFINITY, "kv attend: scale is positive and finite");
    MW_CHECK(a.window >= 0 && a.sinks >= 0, "kv attend: window and sinks are not negative");
    if (b.n_rows == 0 || b.n_seqs == 0) return;
    MW_CHECK(a.q && a.out && ((uintptr_t)a.q | (uintptr_t)a.out) % 16 == 0 && a.q_row >= 0 && a.q_head >= 0 && a.o_row >= 0 && a.o_head >= 0 &&
                 a.q_row % 8 == 0 && a.q_head % 8 == 0 && a.o_row % 8 == 0 && a.o_head % 8 == 0,
             "kv attend: q and out pointers and strides are multiples of 16 bytes");
    // (an expanded tensor has strides of 0: q may be one, out not)
    MW_CHECK((b.n_rows == 1 || a.o_row >= c.head_dim) && (a.n_heads == 1 || a.o_head >= c.head_dim), "kv attend: the result's rows overlap");
    MW_CHECK((int64_t)b.n_rows * a.n_heads < (1LL << 26), "kv attend: too many rows");  // a grid holds 2^32 threads
}

void launch_kv_attend(int n_cus, const mw_kv_cache &c, const mw_kv_batch &b, const KvAttendArgs &a, hipStream_t st) {
    check_kv_attend(c, b, a);
    if (b.n_rows == 0 || b.n_seqs == 0) return;
    const Plan p = plan(n_cus, c, b, a.n_heads, a.window, a.sinks);
    const size_t need = plan_bytes(p, c, b, a.n_heads);
    MW_CHECK(a.ws_bytes >= need && (need == 0 || (a.ws && (uintptr_t)a.ws % 16 == 0)), "kv attend: workspace too small or not 16-byte aligned");
    AttendP A{make_view(c, b), a.n_heads, a.n_heads / c.n_kv_heads, (const bf16_t *)a.q, a.q_row, a.q_head, (bf16_t *)a.out, a.o_row, a.o_head,
              a.scale * 1.4426950408889634f, a.window, a.sinks, p.splits, p.steps, (int)p.tiles, (float *)a.ws,
              (float *)a.ws + (size_t)p.splits * b.n_rows * a.n_heads * c.head_dim};
    const int64_t blocks = p.tiles * c.n_kv_heads * p.splits;
    MW_CHECK(blocks < (1LL << 24), "kv attend: too many tiles");
    const dim3 grid((unsigned)blocks), block(64 * RW);
#define KV_GO(KIND, DH)                                                                            \
    do {                                                                                           \
        if (p.rows == CR) hipLaunchKernelGGL((attend_chunk_kernel<KIND, DH, 1>), grid, block, 0, st, A); \
        else if (KIND == BF16 && p.rows == CR / 2) hipLaunchKernelGGL((attend_chunk_kernel<BF16, DH, 2>), grid, block, 0, st, A); \
        else hipLaunchKernelGGL((attend_rows_kernel<KIND, DH>), grid, block, 0, st, A);              \
    } while (0)
#define KV_DIM(KIND)                          \
    do {                                      \
        if (c.head_dim == 64) KV_GO(KIND, 64); \
        else KV_GO(KIND, 128);                \
    } while (0)
    if (c.dtype == BF16) KV_DIM(BF16);
    else if (c.dtype == E4M3) KV_DIM(E4M3);
    else KV_DIM(INT8);
#undef KV_DIM
#undef KV_GO
    MW_HIP(hipGetLastError());
    if (p.splits > 1) {
        const dim3 jg((unsigned)((int64_t)b.n_rows * a.n_heads));
        if (c.head_dim == 64) hipLaunchKernelGGL(attend_join_kernel<64>, jg, dim3(64), 0, st, A);
        else hipLaunchKernelGGL(attend_join_kernel<128>, jg, dim3(64), 0, st, A);
        MW_HIP(hipGetLastError());
    }
}

}  // namespace mw
