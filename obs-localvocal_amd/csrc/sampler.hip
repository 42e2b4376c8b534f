// sampler.hip — one token per row of logits: temperature, top-k, top-p, min-p and a draw with a given uniform number.
//
// The order of the tokens of a row is never formed by sorting.  With x = logit / temperature and d = (max x - x) log2(e), a
// token's weight is 2^-d.  Where weights are added in an order that may change (LDS atomics) they are whole numbers, so that
// the sums are exact; the others are formed in one fixed order, in 64 bits beyond 16 bytes of a row (a tile of the draw: in fp32).  A token's place in the order is the 64-bit key
// (falling logit, rising index), unique in the row.
//   1. maximum of the row;
//   2. total weight; when top-k or top-p cut, a histogram over d in 2048 bins (count and weight of each);
//   3. the bin in which the cut falls, its members in a list, the cut among them by counting (a bin with more members than
//      the list holds is divided again by the key, 2048 ways at a time).  First the cut of top-k, then that of top-p, whose
//      threshold needs the weight top-k left;
//   4. the weight of what is kept, its share u, and the first token in the order of the index at which the running weight
//      reaches it: wave totals, then tiles of the one wave, then lanes of the one tile.
// One 1024-thread workgroup per row; every pass reads the row again (207 KB of 51 866 tokens: from L2 after the first).  Kept in
// registers between the passes (56 a thread) the same code unrolled to 40 k instructions.
// Bound: the latency of the passes one after the other, and in step 2 the histogram's LDS atomics (the same time with their branches
// taken out).  f32, 51 866 tokens: one row with top-k 50, top-p and min-p 17 us (maximum 3, bound 1, total and list 5, two sorts and
// the draw 3, launch); 64 rows of mixed settings 46 us, those with top-k 1000 and top-p the longest (histogram 10, a cut 9 each);
// bf16, 128 000 tokens, 256 rows 79 us, of which it reads 140 MB from memory: every row twice.  Loads of 64 bytes a thread at once
// changed none of them.
#include "decoder_ops.hpp"

namespace mw {

namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
using u64 = unsigned long long;

constexpr int ST = 1024;          // threads
constexpr int SW = ST / 64;       // waves
constexpr int NB = 2048;          // bins: bin b holds -64 d in (-b - 1, -b], the last one all from there on
constexpr int LIST = 1024;        // tokens of a list, one a thread (a place takes 10 bits beside an index)
constexpr int FEW = 512;          // a cut of top-k up to here is looked for among the largest tokens
constexpr double LN2 = 0.6931471805599453;

struct Shared {
    u64 mass[NB], mass2[NB];
    unsigned cnt[NB], cnt2[NB];
    u64 list_r[LIST], list_w[LIST], sorted[LIST];
    u64 wave64[SW], wave64b[SW];
    double wave_d[SW];
    float wave_f[SW], most[ST], bound;
    unsigned wave32[SW];
    u64 lo, hi;                   // key range of a division
    u64 cut, cut_mass;            // last kept key, weight up to and including it
    u64 found_mass;               // weight before the bin found
    u64 kept, total, extra[SW];
    unsigned found_bin, found_before, found_count, n_list;
};

// weights and keys of a row's values
struct Row {
    float max, c;  // c = log2(e) / temperature
    double c_d;
    float half, c2;  // -max / 2, 2 c
    __device__ __forceinline__ void init(float max_, double temperature) {
        max = max_;
        // a temperature so small that its reciprocal overflows leaves the largest alone; an infinite one makes all tokens equal (in fp32
        // to 10^-6 of a share, over the whole range of logits: -inf times 0 would be no number)
        c_d = fmin(fmax(1.4426950408889634 / temperature, 0.0), 1e37);
        c = fmaxf((float)c_d, 1.4e-45f);
        half = -0.5f * max;
        c2 = 2.0f * c;
    }
    // -d = (x - max) log2(e) / temperature; -inf stays -inf.  Both roundings keep the order of the tokens.  (By halves: the
    // difference of two finite logits need not be finite.  The bits are the same where it is.)
    __device__ __forceinline__ float power(float x) const { return fmaf(x, 0.5f, half) * c2; }
    __device__ __forceinline__ float share(float x) const { return __builtin_amdgcn_exp2f(power(x)); }  // of the likeliest token's probability
    // 2^43 of a share, to the nearest: 2^20 of them fit in 64 bits, and what 2^20 tokens of less than half a unit leave out is 2^-24 of the
    // likeliest one's (with 2^31 units top-p did not see tails that it has to cut)
    static __device__ __forceinline__ u64 units(float share) {
        const float f = fmaf(share, 8796093022208.0f, 0.5f);
        const unsigned hi = (unsigned)(f * 2.3283064365386963e-10f);  // 2^-32
        return (u64)hi << 32 | (unsigned)fmaf((float)hi, -4294967296.0f, f);
    }
    // floor(2^(40 - d)), from d in 64 bits: 2^-d = 2^-whole 2^-part, |part| <= 1/2
    __device__ __forceinline__ u64 weight(float x) const {
        const double d = fmin(((double)max - (double)x) * c_d, 200.0), w = rint(d);
        const u64 m = (u64)(unsigned)(__builtin_amdgcn_exp2f((float)(w - d)) * 16777216.0f) << 36;  // 24 significant bits
        return w < 44.0 ? m >> ((int)w + 20) : 0;
    }
    __device__ __forceinline__ float logprob(float x, double z) const { return (float)(((double)x - (double)max) * c_d * LN2 - log(z)); }
};
__device__ __forceinline__ unsigned ordered(float x) {  // rising with x
    const unsigned b = __float_as_uint(x + 0.0f);  // -0 and 0 are one value
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(unsigned b) { return __uint_as_float(b ^ ((b >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 rank_key(float x, int i) { return (u64)(~ordered(x)) << 32 | (unsigned)i; }
__device__ __forceinline__ float key_value(u64 r) { return unordered(~(unsigned)(r >> 32)); }

__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// a and b summed over the workgroup; every thread gets the sums
__device__ __forceinline__ void block_sum64(Shared &S, u64 &a, u64 &b) {
    a = wave_sum64(a);
    b = wave_sum64(b);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        S.wave64[threadIdx.x >> 6] = a;
        S.wave64b[threadIdx.x >> 6] = b;
    }
    __syncthreads();
    a = b = 0;
#pragma unroll
    for (int w = 0; w < SW; ++w) {
        a += S.wave64[w];
        b += S.wave64b[w];
    }
}
// how many threads of the workgroup say yes
__device__ __forceinline__ int block_count(Shared &S, bool yes) {
    const int n = __popcll(__ballot(yes));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) S.wave32[threadIdx.x >> 6] = n;
    __syncthreads();
    int t = 0;
#pragma unroll
    for (int w = 0; w < SW; ++w) t += (int)S.wave32[w];
    return t;
}
// v summed over the workgroup in one order; every thread gets the sum, S.wave_d the waves' parts
__device__ __forceinline__ double block_sum_d(Shared &S, double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) S.wave_d[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < SW; ++w) t += S.wave_d[w];
    return t;
}
// A value that at least `want` of the threads' largest values reach, and not many more: bisection between the row's maximum and
// 2^-32 of its weight, by one wave (no barrier inside).  Up to a quarter of 256 it looks at the largest of every four threads.
// -FLT_MAX when that many do not exist there.
__device__ __forceinline__ float bound_of(Shared &S, float mine, const Row &R, int want) {
    S.most[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x < 64) {
        float v[SW];
#pragma unroll
        for (int i = 0; i < SW; ++i) v[i] = S.most[i * 64 + threadIdx.x];
        const bool few = want <= 64;
        if (few) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = fmaxf(fmaxf(v[i], v[i + 4]), fmaxf(v[i + 8], v[i + 12]));
        }
        auto reach = [&](float x) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) n += __popcll(__ballot(v[i] >= x));
            if (!few) {
#pragma unroll
                for (int i = 4; i < SW; ++i) n += __popcll(__ballot(v[i] >= x));
            }
            return n;
        };
        float hi = R.max, lo = fmaxf(R.max - 32.0f / R.c, -3.4028235e38f);
        if (reach(lo) < want) {
            lo = -3.4028235e38f;
        } else {
            for (int i = 0; i < 14; ++i) {
                const float mid = 0.5f * lo + 0.5f * hi;
                const int n = reach(mid);
                if (n >= want) {
                    lo = mid;
                    if (n <= want + 8 + want / 8) break;
                } else {
                    hi = mid;
                }
            }
        }
        if (threadIdx.x == 0) S.bound = lo;
    }
    __syncthreads();
    return S.bound;
}

template <int N> __device__ __forceinline__ u64 lane_xor64(u64 v) {
    const unsigned lo = (unsigned)v, hi = (unsigned)(v >> 32);
    if constexpr (N < 16) {
        return (u64)__float_as_uint(lane_xor<N>(__uint_as_float(hi))) << 32 | __float_as_uint(lane_xor<N>(__uint_as_float(lo)));
    } else {  // both copies go in: a lane gets its own row's (half's) value in one result and the partner's in the other
        unsigned a, b;
        if constexpr (N == 16) {
            const auto p = __builtin_amdgcn_permlane16_swap(lo, lo, false, false), q = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
            a = p[0] ^ p[1] ^ lo;
            b = q[0] ^ q[1] ^ hi;
        } else {
            const auto p = __builtin_amdgcn_permlane32_swap(lo, lo, false, false), q = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
            a = p[0] ^ p[1] ^ lo;
            b = q[0] ^ q[1] ^ hi;
        }
        return (u64)b << 32 | a;
    }
}
template <int STRIDE> __device__ __forceinline__ void sort_step(u64 &key, int size) {
    if (size <= STRIDE) return;
    const u64 o = lane_xor64<STRIDE>(key);
    const bool low = (threadIdx.x & STRIDE) == 0, up = (threadIdx.x & size) == 0;
    key = (low == up) == (o < key) ? o : key;
}
// The keys of threads 0 .. n - 1 in rising order (bitonic; strides inside a wave without LDS); the others give ~0.  Every thread
// of the workgroup calls; n <= 64 is one wave's work without barriers.
__device__ __forceinline__ u64 block_sort(Shared &S, u64 key, int n) {
    const int t = threadIdx.x;
    int N = 64;
    while (N < n) N *= 2;
    for (int size = 2; size <= N; size *= 2) {
        for (int stride = size / 2; stride >= 64; stride /= 2) {
            S.sorted[t] = key;
            __syncthreads();
            const u64 o = S.sorted[t ^ stride];
            const bool low = (t & stride) == 0, up = (t & size) == 0;
            key = (low == up) == (o < key) ? o : key;
            __syncthreads();
        }
        if (t < N) {
            sort_step<32>(key, size);
            sort_step<16>(key, size);
            sort_step<8>(key, size);
            sort_step<4>(key, size);
            sort_step<2>(key, size);
            sort_step<1>(key, size);
        }
    }
    return key;
}
// w summed over threads 0 .. this one; n: threads that have any
__device__ __forceinline__ u64 block_scan(Shared &S, u64 w, int n) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 u = __shfl_up(w, o);
        if (lane >= o) w += u;
    }
    __syncthreads();
    if (lane == 63) S.wave64[wave] = w;
    __syncthreads();
    if (n > 64)
        for (int q = 0; q < wave; ++q) w += S.wave64[q];
    return w;
}
// the key of list entry t with its place in the list: (value, index, place) in one number; indices are below 2^20
__device__ __forceinline__ u64 placed_key(u64 r, int place) { return (r >> 32) << 32 | (unsigned)r << 10 | (unsigned)place; }

// The first bin whose running count (BY_COUNT: >= want) or running weight (>= want as doubles) is reached; bins follow each other in
// the order of the tokens.  Results in S.found_*; when no bin reaches it, found_bin is NB and found_count 0.
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
    if (t == 0) {
        S.found_bin = NB;
        S.found_count = 0;
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

// A row's values as a thread goes through them: wave w owns a contiguous piece of the row, in rounds of 64 x 16 bytes.
template <bool BF> struct Source {
    static constexpr int VEC = BF ? 8 : 4;
    const void *row;
    int n, mis, K, c0;  // values, values before the row in its first 16 bytes, rounds, the thread's first 16-byte piece

    __device__ __forceinline__ void init(const void *p, int n_) {
        row = p;
        n = n_;
        mis = (int)(((uintptr_t)p & 15) / (BF ? 2 : 4));
        const int nc = (n + mis + VEC - 1) / VEC;
        K = ((nc + SW - 1) / SW + 63) / 64;
        c0 = (threadIdx.x >> 6) * K * 64 + (threadIdx.x & 63);
    }
    __device__ __forceinline__ int owner(int i) const { return (i + mis) / VEC / (64 * K); }  // the wave that has token i
    __device__ __forceinline__ int first(int k) const { return (c0 + 64 * k) * VEC - mis; }
    __device__ __forceinline__ int first(int w, int k) const { return ((w * K + k) * 64 + (int)(threadIdx.x & 63)) * VEC - mis; }  // of wave w
    // the values from index i0 on; what lies outside the row is -inf and never read
    __device__ __forceinline__ void load(int i0, float (&v)[VEC]) const {
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
    }
    // f(values, index of the first) over this thread's pieces in the order of the index
    template <typename F> __device__ __forceinline__ void pieces(F &&f) const {
        for (int k = 0; k < K; ++k) {
            float v[VEC];
            load(first(k), v);
            f(v, first(k));
        }
    }
    // f(value, index) over this thread's values in the order of the index
    template <typename F> __device__ __forceinline__ void each(F &&f) const {
        pieces([&](const float (&v)[VEC], int i0) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f(v[e], i0 + e);
        });
    }
};

// The last kept token when the order is cut at `want` (a count or a weight): S.cut (its key) and S.cut_mass (weight up to and with it);
// false, and both as they were, when there is less than `want`.
// On the way (SUMS) mine gets the thread's share of what is kept ahead of the list (tokens of at least `least`), S.extra what is kept of the
// list for the wave that owns the token.
template <bool BY_COUNT, bool SUMS, typename SRC>
__device__ __forceinline__ bool resolve(Shared &S, const SRC &src, const Row &R, double want, float least, double &mine) {
    find_bin<BY_COUNT>(S, S.cnt, S.mass, 0, 0, want);
    const int bin = (int)S.found_bin;
    if (bin == NB) return false;
    unsigned before = S.found_before;
    u64 before_mass = S.found_mass, lo = 0, hi = ~0ull;
    // The bin's members by the rule that counted them, end <= q <= top (64 q is exact; one end is the next number above -(bin + 1) / 64).
    // The last bin goes down to -inf: a token far away (a mask of the type's lowest value) has that power and belongs to it, a
    // suppressed one has it too and belongs to none.  (The test of x stands behind those of q, which few pass: in one expression 256 rows of
    // 128 000 took 82 us instead of 78.)
    const float top = (float)(-bin) / 64.0f, end = bin == NB - 1 ? -INFINITY : __uint_as_float(__float_as_uint((float)(-bin - 1) / 64.0f) - 1);
    auto in_bin = [&](float x) {
        const float q = R.power(x);
        return q >= end && q <= top && x > -INFINITY;
    };
    // the bin's members with keys lo .. hi; returns how many there are (the list holds the first LIST that came)
    auto gather = [&]() -> unsigned {
        __syncthreads();
        if (threadIdx.x == 0) S.n_list = 0;
        if (threadIdx.x < SW) S.extra[threadIdx.x] = 0;
        __syncthreads();
        mine = 0.0;
        src.pieces([&](const float (&v)[SRC::VEC], int i0) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < SRC::VEC; ++e) {
                const float q = R.power(v[e]), w = SUMS ? __builtin_amdgcn_exp2f(q) : 0.0f;
                if (SUMS) sum += q > top && w >= least ? w : 0.0f;
                if (q >= end && q <= top) {  // (few)
                    const u64 r = rank_key(v[e], i0 + e);
                    if (!(v[e] > -INFINITY)) continue;
                    if (r < lo) {
                        if (SUMS) sum += w >= least ? w : 0.0f;
                    } else if (r <= hi) {
                        const unsigned at = atomicAdd(&S.n_list, 1u);
                        if (at < LIST) S.list_r[at] = r;
                    }
                }
            }
            if (SUMS) mine += (double)sum;
        });
        __syncthreads();
        return S.n_list;
    };
    unsigned count = gather();
    if (count > LIST) {  // the members' range of keys
        if (threadIdx.x == 0) {
            S.lo = ~0ull;
            S.hi = 0;
        }
        __syncthreads();
        u64 a = ~0ull, b = 0;
        src.each([&](float x, int i) {
            if (in_bin(x)) {
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
        // keys are unique: a range divided down to single keys ends the loop at the latest, 2048 ways at a time after six rounds
        while (count > LIST) {
            int s = 0;
            while ((hi - lo) >> s >= NB) ++s;
            for (int b2 = threadIdx.x; b2 < NB; b2 += ST) {
                S.cnt2[b2] = 0;
                S.mass2[b2] = 0;
            }
            __syncthreads();
            src.each([&](float x, int i) {
                if (in_bin(x)) {
                    const u64 r = rank_key(x, i);
                    if (r >= lo && r <= hi) {
                        const int b2 = (int)((r - lo) >> s);
                        atomicAdd(&S.cnt2[b2], 1u);
                        atomicAdd(&S.mass2[b2], Row::units(R.share(x)));
                    }
                }
            });
            __syncthreads();
            find_bin<BY_COUNT>(S, S.cnt2, S.mass2, before, before_mass, want);
            if (S.found_bin == NB) return false;
            before = S.found_before;
            before_mass = S.found_mass;
            count = S.found_count;
            lo += (u64)S.found_bin << s;
            hi = min(hi, lo + ((u64)1 << s) - 1);
            __syncthreads();
        }
        gather();
    }
    // the list in order; the cut is where the running count or weight passes `want`
    const int n = (int)min(S.n_list, (unsigned)LIST), tid = threadIdx.x;
    const u64 key = block_sort(S, tid < n ? placed_key(S.list_r[tid], tid) : ~0ull, n);
    const float x = key_value(key);
    const u64 w = tid < n ? Row::units(R.share(x)) : 0;
    const u64 mass = before_mass + block_scan(S, w, n);
    if (tid < n) {
        const bool ahead = BY_COUNT ? (double)(before + tid) < want : (double)(mass - w) < want;
        const bool last = BY_COUNT ? (double)(before + tid + 1) >= want : (double)mass >= want;
        if (ahead && last) {
            S.cut = (key >> 32) << 32 | ((unsigned)key >> 10);
            S.cut_mass = mass;
        }
        if (SUMS && ahead && R.share(x) >= least) atomicAdd(&S.extra[src.owner((int)((unsigned)key >> 10))], R.weight(x));
    }
    __syncthreads();
    return true;
}

template <bool BF>
__global__ __launch_bounds__(ST) void sample_kernel(SampleArgs A) {
    __shared__ Shared S;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Source<BF> src;
    src.init((const char *)A.logits + (int64_t)row * A.row_stride * (BF ? 2 : 4), A.n_vocab);
    const float temp = A.temperature ? A.temperature[row] : 1.0f;
    const int k = A.top_k ? A.top_k[row] : 0;
    const float top_p = A.top_p ? A.top_p[row] : 1.0f, min_p = A.min_p ? A.min_p[row] : 0.0f;
    const double u = A.u[row];
    const bool greedy = temp <= 0.0f;

    // ---- 1: maximum ----
    if (tid == 0) S.n_list = 0;
    float mx = -INFINITY;
    src.each([&](float x, int) { mx = fmaxf(mx, x); });
    const float my_max = mx;
    mx = wave_max_desc(mx);
    if (lane == 0) S.wave_f[wave] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SW; ++w) mx = fmaxf(mx, S.wave_f[w]);
    Row R;
    R.init(mx, greedy ? 1.0 : (double)temp);

    // ---- 2: total weight; the likeliest tokens into a list, or a histogram ----
    const bool use_k = !greedy && k > 0 && k < A.n_vocab, use_p = !greedy && top_p < 1.0f, use_m = !greedy && min_p > 0.0f;
    const float least = use_m ? fminf(min_p, 1.0f) : 0.0f;  // (the likeliest token's share is 1)
    float bound = INFINITY;
    if (greedy) bound = mx;
    else if (use_k) bound = k <= FEW ? bound_of(S, my_max, R, k) : INFINITY;
    else if (use_m && !use_p) bound = mx + (__builtin_amdgcn_logf(least) - 1e-5f) / R.c;  // (log2; a little more than what is kept)
    bound = fmaxf(bound, -3.4028235e38f);  // (-inf is never listed)
    const bool lists = bound < INFINITY;
    // the thread's sum: fp32 inside 16 bytes of a row, 64 bits over them (in fp32 a long row of equal small weights was off by 3e-6)
    double zd = 0.0;
    constexpr int VEC = Source<BF>::VEC;
    // histogram over 64 d: counts if top-k asks for them, weights if top-p does.  The last bin takes all that is far away: in
    // registers first, or its one address would be waited for by every lane.
    auto histogram = [&]() {
        for (int b = tid; b < NB; b += ST) {
            S.cnt[b] = 0;
            S.mass[b] = 0;
        }
        __syncthreads();
        unsigned far = 0;
        u64 far_mass = 0;
        src.pieces([&](const float (&v)[VEC], int) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float q = R.power(v[e]), w = __builtin_amdgcn_exp2f(q);
                sum += w;
                const u64 un = Row::units(w);  // (ahead of the branch: inside it 256 rows of 128 000 took 84 us, not 80)
                if (q > -(float)(NB - 1) / 64.0f) {
                    const int b = (int)(-64.0f * q);
                    if (use_k) atomicAdd(&S.cnt[b], 1u);
                    if (use_p) atomicAdd(&S.mass[b], un);
                } else if (v[e] > -INFINITY) {
                    ++far;
                    far_mass += un;
                }
            }
            zd += (double)sum;
        });
        if (far) {
            atomicAdd(&S.cnt[NB - 1], far);
            atomicAdd(&S.mass[NB - 1], far_mass);
        }
        __syncthreads();
    };
    if (lists) {
        src.pieces([&](const float (&v)[VEC], int i0) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                sum += R.share(v[e]);
                if (v[e] >= bound) {
                    const unsigned at = atomicAdd(&S.n_list, 1u);
                    if (at < LIST) S.list_r[at] = rank_key(v[e], i0 + e);
                }
            }
            zd += (double)sum;
        });
    } else if (use_k || use_p) {
        histogram();
    } else {
        src.pieces([&](const float (&v)[VEC], int) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += R.share(v[e]);
            zd += (double)sum;
        });
    }
    const double z = block_sum_d(S, zd);
    // a NaN anywhere is one in the sum; with a maximum of +inf or -inf nothing can be drawn
    if (z != z || !(mx < INFINITY) || mx == -INFINITY || temp != temp || top_p != top_p || min_p != min_p || u != u) {
        if (tid == 0) {
            A.ids[row] = -1;
            if (A.logprobs) A.logprobs[row] = __uint_as_float(0x7fc00000u);
        }
        return;
    }
    const int n = (int)min(S.n_list, (unsigned)LIST);
    if (greedy && S.n_list <= LIST) {
        unsigned best = tid < n ? (unsigned)S.list_r[tid] : 0xffffffffu;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) best = min(best, (unsigned)__shfl_xor((int)best, o));
        if (lane == 0) S.wave32[wave] = best;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < SW; ++w) best = min(best, S.wave32[w]);
            A.ids[row] = (int)best;
            if (A.logprobs) A.logprobs[row] = R.logprob(mx, z);
        }
        return;
    }
    const u64 me = tid < n ? S.list_r[tid] : ~0ull;
    const float listed_x = key_value(me);
    S.list_w[tid] = tid < n ? R.weight(listed_x) : 0;
    // (a list that ran over: equal or very near tokens in numbers; the histogram then divides them)
    const bool listed = lists && !greedy && S.n_list <= LIST;
    if (listed) {
        // in the order of the tokens: what is kept is a stretch from the first on
        u64 key = block_sort(S, tid < n ? placed_key(me, tid) : ~0ull, n);
        const float x = key_value(key);
        bool keep = tid < n && (!use_k || tid < k);
        if (use_p) {
            const u64 wt = tid < n ? S.list_w[key & (LIST - 1)] : 0, upto = block_scan(S, wt, n);
            if (tid == min(k, n) - 1) S.kept = upto;  // (a list without top-k has no top-p either)
            __syncthreads();
            keep &= tid == 0 || (double)(upto - wt) < (double)top_p * (double)S.kept;
        }
        keep &= R.share(x) >= least;
        const int nk = block_count(S, keep);
        // in the order of the index: the draw
        key = block_sort(S, tid < nk ? (u64)(unsigned)key : ~0ull, nk);
        const u64 wi = tid < nk ? S.list_w[key & (LIST - 1)] : 0, upto = block_scan(S, wi, nk);
        if (tid == nk - 1) S.total = upto;
        __syncthreads();
        const u64 total = S.total;
        const u64 target = min(max((u64)fmin(fmax(ceil(u * (double)total), 1.0), (double)total), (u64)1), total);
        if (tid < nk && upto - wi < target && upto >= target) {
            A.ids[row] = (int)((unsigned)key >> 10);
            if (A.logprobs) A.logprobs[row] = R.logprob(key_value(S.list_r[key & (LIST - 1)]), z);
        }
        return;
    }
    __syncthreads();

    // ---- 3: cuts ----
    u64 cut = ~0ull;
    if (greedy) cut = (u64)(~ordered(mx)) << 32 | 0x7fffffffu;  // more equal largest logits than the list holds: the first of them is drawn
    double mine = 0.0;
    bool have_sums = false;  // what each wave keeps is known from the last cut
    if (use_k || use_p) {
        if (lists) histogram();
        // what there is by the histogram's own sums: top-p's share of any other total could be more than its bins hold
        u64 live = S.cnt[2 * tid] + S.cnt[2 * tid + 1], mass = S.mass[2 * tid] + S.mass[2 * tid + 1];
        block_sum64(S, live, mass);
        double kept = (double)mass;
        if (use_k) {
            // fewer tokens than k may be left by the suppressed ones: nothing to cut then
            if ((u64)k < live) {
                const bool found = use_p ? resolve<true, false>(S, src, R, (double)k, least, mine) : resolve<true, true>(S, src, R, (double)k, least, mine);
                if (found) {
                    have_sums = !use_p;
                    cut = S.cut;
                    kept = (double)S.cut_mass;
                }
            }
        }
        if (use_p) {
            __syncthreads();
            have_sums = resolve<false, true>(S, src, R, fmax((double)top_p * kept, 0.5), least, mine);
            if (have_sums) cut = S.cut;
        }
    }

    // ---- 4: draw ----
    const float cut_x = cut == ~0ull ? -INFINITY : key_value(cut);
    const int cut_i = cut == ~0ull ? 0x7fffffff : (int)(unsigned)cut;
    auto weight_kept = [&](float x, int i) -> float {
        const float w = R.share(x);
        const bool keep = x > cut_x || (x == cut_x && i <= cut_i);
        return keep && w >= least ? w : 0.0f;
    };
    auto piece_kept = [&](const float (&v)[VEC], int i0) -> float {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += weight_kept(v[e], i0 + e);
        return s;
    };
    // (nothing dropped: the sums of the waves are those of step 2; after a cut they were formed on the way)
    const bool all_kept = !use_k && !use_p && !use_m && !greedy;
    if (!all_kept && !have_sums) {
        mine = 0.0;
        src.pieces([&](const float (&v)[VEC], int i0) { mine += (double)piece_kept(v, i0); });
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o);
    __syncthreads();
    if (lane == 0) S.wave_d[wave] = all_kept ? S.wave_d[wave] : have_sums ? mine + (double)S.extra[wave] * 0x1p-40 : mine;
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < SW; ++w) total += S.wave_d[w];
    // The first token with which the running weight reaches u of the total.  Wave, tile and lane are found one after the other;
    // where the last places of two sums disagree, the last one with weight is it.
    const double target = greedy ? 0.0 : fmin(fmax(u, 0.0) * total, total);
    double below = 0.0, run = 0.0;
    int owner = -1;
    bool done = false;
#pragma unroll
    for (int w = 0; w < SW; ++w) {
        const double s = S.wave_d[w];
        if (!done && s > 0.0) {
            owner = w;
            below = run;
            done = run + s >= target;
        }
        run += s;
    }
    if (owner < 0) return;  // (not reached: the likeliest token has weight)
    // the tiles of its piece, shared by all waves
    for (int kk = wave; kk < src.K; kk += SW) {
        float v[VEC];
        const int i0 = src.first(owner, kk);
        src.load(i0, v);
        const float s = wave_sum_desc(piece_kept(v, i0));
        if (lane == 0) S.most[kk] = s;
    }
    __syncthreads();
    if (wave != owner) return;  // one wave goes on
    run = below;
    int tile = 0;
    double tile_run = below;
    done = false;
    for (int kk = 0; kk < src.K && !done; ++kk) {
        const double s = (double)S.most[kk];
        if (s > 0.0) {
            tile = kk;
            tile_run = run;
        }
        run += s;
        done = s > 0.0 && run >= target;
    }
    float v[VEC];
    const int i0 = src.first(owner, tile);
    src.load(i0, v);
    const double s = (double)piece_kept(v, i0);
    double incl = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double t = __shfl_up(incl, o);
        if (lane >= o) incl += t;
    }
    u64 yes = __ballot(s > 0.0 && tile_run + incl >= target);
    if (yes == 0) yes = 1ull << (63 - __clzll(__ballot(s > 0.0)));
    if (lane == __ffsll(yes) - 1) {
        int id = -1;
        float xi = 0.0f;
        double at = tile_run + incl - s;
        bool reached = false;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float w = weight_kept(v[e], i0 + e);
            at += (double)w;
            if (!reached && w > 0.0f) {
                id = i0 + e;
                xi = v[e];
                reached = at >= target;
            }
        }
        A.ids[row] = id;
        if (A.logprobs) A.logprobs[row] = R.logprob(xi, z);
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
    const dim3 grid(a.n_rows), block(ST);
    if (a.dtype == MW_ELEM_BF16) hipLaunchKernelGGL(sample_kernel<true>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(sample_kernel<false>, grid, block, 0, st, a);
    MW_HIP(hipGetLastError());
}

}  // namespace mw
