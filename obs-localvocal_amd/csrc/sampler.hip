// sampler.hip — one token per row of logits: temperature, top-k, top-p, min-p and a draw with a given uniform number.
//
// The order of the tokens of a row is never formed by sorting.  With x = logit / temperature and d = (max x - x) log2(e), a
// token's weight is 2^-d; weights are held as whole numbers W = floor(2^(40 - d)) in 64 bits, so that every sum is exact and
// independent of the order it is formed in (LDS atomics included).  A token's place in the order is the 64-bit key
// (falling logit, rising index), unique in the row.
//   1. maximum of the row;
//   2. total weight; when top-k or top-p cut, a histogram over d in 2048 bins (count and weight of each);
//   3. the bin in which the cut falls, its members in a list, the cut among them by counting (a bin with more members than
//      the list holds is divided again by the key, 2048 ways at a time).  First the cut of top-k, then that of top-p, whose
//      threshold needs the weight top-k left;
//   4. the weight of what is kept, its share u, and the first token in the order of the index at which the running weight
//      reaches it: wave totals, then tiles of the one wave, then lanes of the one tile.
// One 1024-thread workgroup per row; wave w owns a contiguous piece of the row, 16 bytes a lane and load.  Rows up to 64 k
// tokens stay in registers between the passes; longer ones are read again (from L2 / the memory-side cache).
#include "decoder_ops.hpp"

namespace mw {

namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
using u64 = unsigned long long;

constexpr int ST = 1024;          // threads
constexpr int SW = ST / 64;       // waves
constexpr int NB = 2048;          // bins
constexpr int LIST = 256;         // members of a bin resolved by counting
constexpr int REG_VALS = 64;      // values a thread keeps
constexpr double LOG2E = 1.4426950408889634, LN2 = 0.6931471805599453;

struct Shared {
    u64 mass[NB], mass2[NB];
    unsigned cnt[NB], cnt2[NB];
    u64 list_r[LIST], list_w[LIST];
    u64 wave64[SW];
    unsigned wave32[SW];
    u64 lo, hi;                   // key range of a division
    u64 cut, cut_mass;            // last kept key, weight up to and including it
    u64 found_mass;               // weight before the bin found
    unsigned found_bin, found_before, found_count, n_list, best_i;
};

// weights and keys of a row's values
struct Row {
    double inv;  // log2(e) / temperature
    double max;
    __device__ __forceinline__ float dist(float x) const { return (float)((max - (double)x) * inv); }
    __device__ __forceinline__ int bin(float x) const { return (int)fminf(dist(x) * 64.0f, (float)(NB - 1)); }
    // 2^-d = 2^-whole 2^-part, |part| <= 1/2: the exponential of a small number keeps its last place
    __device__ __forceinline__ void split(float x, int &whole, float &e) const {
        const double d = (max - (double)x) * inv;
        const double w = rint(fmin(d, 256.0));
        whole = (int)w;
        e = __builtin_amdgcn_exp2f((float)(w - fmin(d, 256.0)));
    }
    __device__ __forceinline__ u64 weight(float x) const {
        int whole;
        float e;
        split(x, whole, e);
        const u64 m = (u64)(unsigned)(e * 16777216.0f) << 36;  // exact: e has 24 significant bits, 0.7 <= e <= 1.42
        return whole < 44 ? m >> (whole + 20) : 0;
    }
    __device__ __forceinline__ float share(float x) const {  // of the likeliest token's probability
        int whole;
        float e;
        split(x, whole, e);
        return ldexpf(e, -whole);
    }
};
__device__ __forceinline__ u64 rank_key(float x, int i) {
    unsigned b = __float_as_uint(x);
    b ^= (b >> 31) ? 0xffffffffu : 0x80000000u;  // rising with x
    return (u64)(~b) << 32 | (unsigned)i;
}

__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// v summed over the workgroup; every thread gets the sum
__device__ __forceinline__ u64 block_sum64(Shared &S, u64 v) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) S.wave64[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 t = 0;
#pragma unroll
    for (int w = 0; w < SW; ++w) t += S.wave64[w];
    return t;
}

// The first bin whose running count (BY_COUNT: >= want) or running weight (>= want as doubles) is reached; bins follow each other in
// the order of the tokens.  Results in S.found_*.
template <bool BY_COUNT>
__device__ void find_bin(Shared &S, const unsigned *cnt, const u64 *mass, unsigned base_cnt, u64 base_mass, double want) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    unsigned c[2] = {cnt[2 * t], cnt[2 * t + 1]};
    u64 m[2] = {mass[2 * t], mass[2 * t + 1]};
    unsigned ci = c[0] + c[1];
    u64 mi = m[0] + m[1];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned cu = __shfl_up(ci, o);
        const u64 mu = __shfl_up(mi, o);
        if (lane >= o) {
            ci += cu;
            mi += mu;
        }
    }
    __syncthreads();
    if (lane == 63) {
        S.wave32[wave] = ci;
        S.wave64[wave] = mi;
    }
    __syncthreads();
    unsigned cb = base_cnt + ci - c[0] - c[1];
    u64 mb = base_mass + mi - m[0] - m[1];
    for (int w = 0; w < wave; ++w) {
        cb += S.wave32[w];
        mb += S.wave64[w];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const bool before = BY_COUNT ? (double)cb < want : (double)mb < want;
        const bool after = BY_COUNT ? (double)(cb + c[k]) >= want : (double)(mb + m[k]) >= want;
        if (before && after) {  // true in one bin only
            S.found_bin = 2 * t + k;
            S.found_before = cb;
            S.found_mass = mb;
            S.found_count = c[k];
        }
        cb += c[k];
        mb += m[k];
    }
    __syncthreads();
}

template <bool BF, bool REG> struct Source {
    static constexpr int VEC = BF ? 8 : 4;
    const void *row;
    int n, mis, nc, cpw, K, c0;  // values, values before the row in its first 16 bytes, 16-byte pieces, pieces per wave, rounds
    float x[REG ? REG_VALS : 1];

    __device__ __forceinline__ void init(const void *p, int n_) {
        row = p;
        n = n_;
        mis = (int)(((uintptr_t)p & 15) / (BF ? 2 : 4));
        nc = (n + mis + VEC - 1) / VEC;
        cpw = ((nc + SW - 1) / SW + 63) / 64 * 64;
        K = cpw / 64;
        c0 = (threadIdx.x >> 6) * cpw + (threadIdx.x & 63);
    }
    // values of piece c; what lies outside the row is -inf and never read
    __device__ __forceinline__ void load(int c, float (&v)[VEC]) const {
        const int i0 = c * VEC - mis;
        if (i0 >= 0 && i0 + VEC <= n) {
            if constexpr (BF) {
                const u32x4 a = *(const u32x4 *)((const bf16_t *)row + i0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[2 * i] = __uint_as_float(a[i] << 16);
                    v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
                }
            } else {
                const f32x4 a = *(const f32x4 *)((const float *)row + i0);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = a[i];
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[e] = -INFINITY;
                if (i0 + e >= 0 && i0 + e < n) {
                    if constexpr (BF) v[e] = __uint_as_float((unsigned)((const bf16_t *)row)[i0 + e] << 16);
                    else v[e] = ((const float *)row)[i0 + e];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] += 0.0f;  // -0 and 0 are one value
    }
    __device__ __forceinline__ void fill() {
        if constexpr (REG) {
#pragma unroll
            for (int k = 0; k < REG_VALS / VEC; ++k) {
                float v[VEC];
                load(k < K ? c0 + 64 * k : nc, v);  // piece nc and those behind it: nothing
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[k * VEC + e] = v[e];
            }
        }
    }
    // f(value, index) over this thread's values in the order of the index
    template <typename F> __device__ __forceinline__ void each(F &&f) const {
        if constexpr (REG) {
#pragma unroll
            for (int k = 0; k < REG_VALS / VEC; ++k) {
                if (k < K) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) f(x[k * VEC + e], (c0 + 64 * k) * VEC - mis + e);
                }
            }
        } else {
            for (int k = 0; k < K; ++k) {
                float v[VEC];
                load(c0 + 64 * k, v);
#pragma unroll
                for (int e = 0; e < VEC; ++e) f(v[e], (c0 + 64 * k) * VEC - mis + e);
            }
        }
    }
};

// The last kept token when the order is cut at `want` (a count or a weight): S.cut (its key) and S.cut_mass (weight up to and with it).
template <bool BY_COUNT, typename SRC>
__device__ void resolve(Shared &S, const SRC &src, const Row &R, double want) {
    find_bin<BY_COUNT>(S, S.cnt, S.mass, 0, 0, want);
    const int bin = (int)S.found_bin;
    unsigned before = S.found_before, count = S.found_count;
    u64 before_mass = S.found_mass;
    u64 lo = 0, hi = ~0ull;
    if (count > LIST) {  // the members' range of keys
        if (threadIdx.x == 0) {
            S.lo = ~0ull;
            S.hi = 0;
        }
        __syncthreads();
        u64 a = ~0ull, b = 0;
        src.each([&](float x, int i) {
            if (x > -INFINITY && R.bin(x) == bin) {
                const u64 r = rank_key(x, i);
                a = min(a, r);
                b = max(b, r);
            }
        });
        if (a <= b) {
            atomicMin(&S.lo, a);
            atomicMax(&S.hi, b);
        }
        __syncthreads();
        lo = S.lo;
        hi = S.hi;
        // keys are unique: a range divided down to single keys ends the loop at the latest
        while (count > LIST) {
            int s = 0;
            while ((hi - lo) >> s >= NB) ++s;
            for (int b2 = threadIdx.x; b2 < NB; b2 += ST) {
                S.cnt2[b2] = 0;
                S.mass2[b2] = 0;
            }
            __syncthreads();
            src.each([&](float x, int i) {
                if (x > -INFINITY && R.bin(x) == bin) {
                    const u64 r = rank_key(x, i);
                    if (r >= lo && r <= hi) {
                        const int b2 = (int)((r - lo) >> s);
                        atomicAdd(&S.cnt2[b2], 1u);
                        atomicAdd(&S.mass2[b2], R.weight(x));
                    }
                }
            });
            __syncthreads();
            find_bin<BY_COUNT>(S, S.cnt2, S.mass2, before, before_mass, want);
            before = S.found_before;
            before_mass = S.found_mass;
            count = S.found_count;
            lo += (u64)S.found_bin << s;
            hi = min(hi, lo + ((u64)1 << s) - 1);
            __syncthreads();
        }
    }
    if (threadIdx.x == 0) S.n_list = 0;
    __syncthreads();
    src.each([&](float x, int i) {
        if (x > -INFINITY && R.bin(x) == bin) {
            const u64 r = rank_key(x, i);
            if (r >= lo && r <= hi) {
                const unsigned at = atomicAdd(&S.n_list, 1u);
                if (at < LIST) {
                    S.list_r[at] = r;
                    S.list_w[at] = R.weight(x);
                }
            }
        }
    });
    __syncthreads();
    const int n = (int)min(S.n_list, (unsigned)LIST);
    if ((int)threadIdx.x < n) {
        const u64 me = S.list_r[threadIdx.x], w = S.list_w[threadIdx.x];
        unsigned c = before;
        u64 m = before_mass;
        for (int j = 0; j < n; ++j)
            if (S.list_r[j] < me) {
                ++c;
                m += S.list_w[j];
            }
        const bool ahead = BY_COUNT ? (double)c < want : (double)m < want;
        const bool last = BY_COUNT ? (double)(c + 1) >= want : (double)(m + w) >= want;
        if (ahead && last) {
            S.cut = me;
            S.cut_mass = m + w;
        }
    }
    __syncthreads();
}

template <bool BF, bool REG>
__global__ __launch_bounds__(ST) void sample_kernel(SampleArgs A) {
    __shared__ Shared S;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Source<BF, REG> src;
    src.init((const char *)A.logits + (int64_t)row * A.row_stride * (BF ? 2 : 4), A.n_vocab);
    src.fill();
    const float temp = A.temperature ? A.temperature[row] : 1.0f;
    const int k = A.top_k ? A.top_k[row] : 0;
    const float top_p = A.top_p ? A.top_p[row] : 1.0f, min_p = A.min_p ? A.min_p[row] : 0.0f;
    const double u = A.u[row];
    const bool greedy = temp <= 0.0f;

    // ---- 1: maximum ----
    for (int b = tid; b < NB; b += ST) {
        S.cnt[b] = 0;
        S.mass[b] = 0;
    }
    if (tid == 0) {
        S.best_i = 0xffffffffu;
        S.cut = ~0ull;
        S.cut_mass = 0;
    }
    float mx = -INFINITY;
    bool bad = false;
    src.each([&](float x, int) {
        bad |= !(x < INFINITY);  // NaN or +inf
        mx = fmaxf(mx, x);
    });
    mx = wave_max_desc(mx);
    bad = __ballot(bad) != 0;
    if (lane == 0) {
        S.wave32[wave] = __float_as_uint(mx);
        S.wave64[wave] = bad;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SW; ++w) {
        mx = fmaxf(mx, __uint_as_float(S.wave32[w]));
        bad |= S.wave64[w] != 0;
    }
    bad |= temp != temp || top_p != top_p || min_p != min_p || u != u || mx == -INFINITY;
    if (bad) {  // the same for the whole workgroup
        if (tid == 0) {
            A.ids[row] = -1;
            if (A.logprobs) A.logprobs[row] = __uint_as_float(0x7fc00000u);
        }
        return;
    }
    Row R;
    // (a temperature so small that its reciprocal overflows leaves the largest logits alone, an infinite one makes all equal)
    R.inv = greedy ? LOG2E : LOG2E / (double)temp;
    R.max = (double)mx;

    // ---- 2: total weight, histogram ----
    const bool use_k = !greedy && k > 0 && k < A.n_vocab, use_p = !greedy && top_p < 1.0f;
    u64 z = 0;
    unsigned best = 0xffffffffu;
    src.each([&](float x, int i) {
        if (x > -INFINITY) {
            const u64 w = R.weight(x);
            z += w;
            if (x == mx) best = min(best, (unsigned)i);
            if (use_k || use_p) {
                const int b = R.bin(x);
                atomicAdd(&S.cnt[b], 1u);
                atomicAdd(&S.mass[b], w);
            }
        }
    });
    if (greedy && best != 0xffffffffu) atomicMin(&S.best_i, best);
    z = block_sum64(S, z);
    const double log_z = log((double)z * 0x1p-40);

    int id = -1;
    float xi = 0.0f;
    if (greedy) {
        if (tid == 0) {
            A.ids[row] = (int)S.best_i;
            if (A.logprobs) A.logprobs[row] = (float)-log_z;
        }
        return;
    }

    // ---- 3: cuts ----
    u64 cut = ~0ull;
    double kept = (double)z;
    if (use_k) {
        // fewer tokens than k may be left by the suppressed ones: nothing to cut then
        unsigned live = 0;
        {
            unsigned c = S.cnt[2 * tid] + S.cnt[2 * tid + 1];
            live = (unsigned)block_sum64(S, c);
        }
        if ((unsigned)k < live) {
            resolve<true>(S, src, R, (double)k);
            cut = S.cut;
            kept = (double)S.cut_mass;
        }
    }
    if (use_p) {
        const double want = fmax((double)top_p * kept, 0.5);
        __syncthreads();
        resolve<false>(S, src, R, want);
        cut = S.cut;
    }

    // ---- 4: draw ----
    u64 mine = 0;
    auto weight_kept = [&](float x, int i) -> u64 {
        if (!(x > -INFINITY) || rank_key(x, i) > cut) return 0;
        if (min_p > 0.0f && x != mx && R.share(x) < min_p) return 0;
        return R.weight(x);
    };
    src.each([&](float x, int i) { mine += weight_kept(x, i); });
    const u64 wsum = wave_sum64(mine);
    __syncthreads();
    if (lane == 0) S.wave64[wave] = wsum;
    __syncthreads();
    u64 total = 0, below = 0;
#pragma unroll
    for (int w = 0; w < SW; ++w) {
        if (w == wave) below = total;
        total += S.wave64[w];
    }
    // the first whole weight that is at least u total (at least 1: a token of weight 0 is never drawn)
    const double want = fmin(fmax(ceil(u * (double)total), 1.0), (double)total);
    u64 target = (u64)want;
    target = min(max(target, (u64)1), total);
    if (!(below < target && below + wsum >= target)) return;  // one wave goes on
    u64 run = below;
    for (int kk = 0; kk < src.K; ++kk) {
        float v[Source<BF, REG>::VEC];
        const int c = src.c0 + 64 * kk;
        src.load(c, v);
        u64 s = 0;
#pragma unroll
        for (int e = 0; e < Source<BF, REG>::VEC; ++e) s += weight_kept(v[e], c * Source<BF, REG>::VEC - src.mis + e);
        u64 incl = s;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const u64 t = __shfl_up(incl, o);
            if (lane >= o) incl += t;
        }
        const u64 all = __shfl(incl, 63);
        if (run + all >= target) {
            u64 at = run + incl - s;
            if (at < target && at + s >= target) {  // one lane
#pragma unroll
                for (int e = 0; e < Source<BF, REG>::VEC; ++e) {
                    const int i = c * Source<BF, REG>::VEC - src.mis + e;
                    const u64 w = weight_kept(v[e], i);
                    if (id < 0 && w != 0 && at + w >= target) {
                        id = i;
                        xi = v[e];
                    }
                    at += w;
                }
                A.ids[row] = id;
                if (A.logprobs) A.logprobs[row] = (float)(-(R.max - (double)xi) * R.inv * LN2 - log_z);
            }
            break;
        }
        run += all;
    }
}

}  // namespace

void check_sample(const SampleArgs &a) {
    MW_CHECK(a.dtype == MW_ELEM_F32 || a.dtype == MW_ELEM_BF16, "sample: logits are f32 or bf16");
    MW_CHECK(a.n_rows >= 0 && a.n_rows < (1 << 22) && a.n_vocab > 0 && a.n_vocab <= (1 << 20), "sample: row count / vocabulary size");
    if (a.n_rows == 0) return;
    const int eb = a.dtype == MW_ELEM_F32 ? 4 : 2;
    MW_CHECK(a.logits && a.u && a.ids, "sample: null logits, u or ids");
    MW_CHECK((uintptr_t)a.logits % eb == 0 && (uintptr_t)a.u % 8 == 0 && (uintptr_t)a.ids % 4 == 0 && (uintptr_t)a.logprobs % 4 == 0 &&
                 ((uintptr_t)a.temperature | (uintptr_t)a.top_k | (uintptr_t)a.top_p | (uintptr_t)a.min_p) % 4 == 0,
             "sample: unaligned array");
    MW_CHECK(a.row_stride >= 0, "sample: negative row stride");
}

void launch_sample(const SampleArgs &a, hipStream_t st) {
    check_sample(a);
    if (a.n_rows == 0) return;
    const bool reg = a.n_vocab + 8 <= SW * 64 * REG_VALS;
    const dim3 grid(a.n_rows), block(ST);
    if (a.dtype == MW_ELEM_BF16) {
        if (reg) hipLaunchKernelGGL((sample_kernel<true, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((sample_kernel<true, false>), grid, block, 0, st, a);
    } else {
        if (reg) hipLaunchKernelGGL((sample_kernel<false, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((sample_kernel<false, false>), grid, block, 0, st, a);
    }
    MW_HIP(hipGetLastError());
}

}  // namespace mw
