// kv_cache.hip — writing keys and values into the pages of a cache and reading them back.
//
// A row of one head (64 or 128 elements) is held as bf16, or as 8-bit codes with one fp32 scale:
//   e4m3  scale = the smallest power of two >= 2^-126 with max|x| <= 448 scale; x / scale is then exact (a shift of the
//         exponent) and the code is the one rounding the format cannot do without
//   int8  scale = max|x| x (1 / 127 rounded to fp32), what dividing a tensor by 127 on the GPU gives: a cache that a program fills by
//         tensor operations holds the same bits (one row in 20 would have another last place, and a code in 10^7 would follow it).
//         code = rne(x / scale).  The quotient is not formed in fp32 (its rounding could carry a value
//         over the half between two codes): the nearest whole number q of a product with the reciprocal is corrected by
//         the remainder x - q scale, which fma gives exactly.
// Bound: HBM bytes (each element is read once and written once), the launch when few rows are written.  int8, 8 heads of 128, f32
// rows: 9 k rows written in 31 us, 34 k read back in 80 (3.9 TB/s; a copy reaches 4.7); one row of 64 streams, 20 heads of 64, 4 us.
#include "decoder_ops.hpp"

namespace mw {

void check_kv(const mw_kv_cache &c, const mw_kv_batch &b) {
    MW_CHECK(c.k && c.v, "kv cache: null pages");
    MW_CHECK(c.dtype == MW_ELEM_BF16 || c.dtype == MW_ELEM_E4M3 || c.dtype == MW_ELEM_INT8, "kv cache: element type is bf16, e4m3 or int8");
    MW_CHECK(c.head_dim == 64 || c.head_dim == 128, "kv cache: head_dim is 64 or 128");
    MW_CHECK(c.n_pages > 0 && c.n_kv_heads > 0 && c.n_kv_heads <= 65535, "kv cache: page / head count");
    MW_CHECK(c.page_size > 0 && c.page_size <= 32768 && (c.page_size & (c.page_size - 1)) == 0, "kv cache: page_size is a power of two up to 32768");
    const int64_t al = c.dtype == MW_ELEM_BF16 ? 8 : 16;  // elements in 16 bytes
    MW_CHECK(c.page_stride >= 0 && c.head_stride >= 0 && c.row_stride >= 0 && c.page_stride % al == 0 && c.head_stride % al == 0 &&
                 c.row_stride % al == 0 && ((uintptr_t)c.k | (uintptr_t)c.v) % 16 == 0,
             "kv cache: strides and bases are multiples of 16 bytes");
    if (c.dtype != MW_ELEM_BF16)
        MW_CHECK(c.k_scale && c.v_scale && ((uintptr_t)c.k_scale | (uintptr_t)c.v_scale) % 4 == 0 && c.scale_page_stride >= 0 &&
                     c.scale_head_stride >= 0 && c.scale_row_stride >= 0,
                 "kv cache: an 8-bit cache needs its scales");
    MW_CHECK(b.n_seqs >= 0 && b.n_rows >= 0 && b.n_seqs <= (1 << 20), "kv batch: sequence / row count");
    if (b.n_seqs > 0) {
        MW_CHECK(b.cu_rows && b.kv_len && (b.block_table || b.table_cols == 0), "kv batch: null cu_rows, kv_len or block_table");
        MW_CHECK(b.table_cols >= 0 && b.table_stride >= b.table_cols, "kv batch: table_stride below table_cols");
    }
    MW_CHECK(b.max_rows >= 0 && b.max_kv >= 0, "kv batch: expected lengths");
}

void check_kv_rows(const mw_kv_cache &c, const mw_kv_batch &b, int dtype, const void *k, const void *v, int64_t row_stride, int64_t head_stride,
                   bool write) {
    check_kv(c, b);
    MW_CHECK(dtype == MW_ELEM_F32 || dtype == MW_ELEM_BF16, "kv rows: element type is f32 or bf16");
    if (b.n_rows == 0 || b.n_seqs == 0) return;
    const int64_t al = dtype == MW_ELEM_F32 ? 4 : 8;
    MW_CHECK(k && v && ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && row_stride >= 0 && head_stride >= 0 && row_stride % al == 0 && head_stride % al == 0,
             "kv rows: pointers and strides are multiples of 16 bytes");
    MW_CHECK((int64_t)b.n_rows * c.n_kv_heads < (1LL << 28), "kv rows: too many rows");  // a grid holds 2^32 threads
    // what is written must not share memory with itself (an expanded tensor has strides of 0); what is read may
    auto apart = [](int64_t n, int64_t stride, int64_t least) { return n <= 1 || stride >= least; };
    if (write) {
        MW_CHECK(apart(c.n_pages, c.page_stride, c.head_dim) && apart(c.n_kv_heads, c.head_stride, c.head_dim) && apart(c.page_size, c.row_stride, c.head_dim),
                 "kv rows: the cache's rows overlap");
        MW_CHECK(c.dtype == MW_ELEM_BF16 || (apart(c.n_pages, c.scale_page_stride, 1) && apart(c.n_kv_heads, c.scale_head_stride, 1) &&
                                             apart(c.page_size, c.scale_row_stride, 1)),
                 "kv rows: the cache's scales overlap");
    } else {
        MW_CHECK(apart(b.n_rows, row_stride, c.head_dim) && apart(c.n_kv_heads, head_stride, c.head_dim), "kv rows: the result's rows overlap");
    }
}

namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x2 = __attribute__((ext_vector_type(2))) float;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
using u32x2 = __attribute__((ext_vector_type(2))) unsigned;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;

constexpr int BF16 = MW_ELEM_BF16, E4M3 = MW_ELEM_E4M3, INT8 = MW_ELEM_INT8;
constexpr float SCALE_MIN = 1.17549435e-38f;  // 2^-126

template <int KIND> __host__ __device__ constexpr int elem_bytes() { return KIND == BF16 ? 2 : 1; }

__device__ __forceinline__ unsigned pack_bf16(float a, float b) { return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, bf16x2)); }

// A lane's 8 elements of a row: adjacent ones where rows come and go as bf16; 4 and 4, half a row apart, where they do as fp32, so
// that every load and store of 16 bytes a lane covers whole lines (two of them 16 bytes apart wrote every line twice by halves).
template <bool F32, int DH> __device__ __forceinline__ int first_of(int sub) { return sub * (F32 ? 4 : 8); }

// 8 elements of a row of bf16 or fp32
template <bool F32, int DH> __device__ __forceinline__ void load8(const void *p, int64_t at, float (&x)[8]) {
    if constexpr (F32) {
        const f32x4 a = *(const f32x4 *)((const float *)p + at), b = *(const f32x4 *)((const float *)p + at + DH / 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = a[i];
            x[4 + i] = b[i];
        }
    } else {
        const u32x4 a = *(const u32x4 *)((const bf16_t *)p + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(a[i] << 16);
            x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
        }
    }
}
template <bool F32, int DH> __device__ __forceinline__ void store8(void *p, int64_t at, const float (&x)[8]) {
    if constexpr (F32) {
        *(f32x4 *)((float *)p + at) = f32x4{x[0], x[1], x[2], x[3]};
        *(f32x4 *)((float *)p + at + DH / 2) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        *(u32x4 *)((bf16_t *)p + at) = u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
    }
}

// the row's largest magnitude over its DH / 8 lanes, as ordered bits: a NaN or an infinity among them gives >= 0x7f800000
template <int DH> __device__ __forceinline__ unsigned row_amax_bits(const float (&x)[8]) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    // (as floats the lanes' exchange would drop a NaN; lane_xor moves bits)
    m = max(m, __float_as_uint(lane_xor<1>(__uint_as_float(m))));
    m = max(m, __float_as_uint(lane_xor<2>(__uint_as_float(m))));
    m = max(m, __float_as_uint(lane_xor<4>(__uint_as_float(m))));
    if constexpr (DH == 128) m = max(m, __float_as_uint(lane_xor<8>(__uint_as_float(m))));
    return m;
}

__device__ __forceinline__ int int8_code(float x, float scale, float inv) {
    float q = rintf(x * inv);
    const float r = fmaf(-q, scale, x);  // exact: |r| <= scale and a multiple of both last places
    const float h = 0.5f * scale;
    if (r > h) q += 1.0f;
    if (r < -h) q -= 1.0f;
    // a half exactly between two codes goes to the even one
    if (r == h && ((int)q & 1)) q += 1.0f;
    if (r == -h && ((int)q & 1)) q -= 1.0f;
    return (int)q;
}

template <int KIND, int DH, bool F32> __device__ __forceinline__ void write_row(char *dst, float *scale_at, const float (&x)[8], int sub) {
    dst += first_of<F32, DH>(sub) * elem_bytes<KIND>();
    if constexpr (KIND == BF16) {
        const u32x4 c = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
        if constexpr (F32) {
            *(u32x2 *)dst = u32x2{c.x, c.y};
            *(u32x2 *)(dst + DH) = u32x2{c.z, c.w};
        } else {
            *(u32x4 *)dst = c;
        }
    } else {
        const unsigned ub = row_amax_bits<DH>(x);
        const bool bad = ub >= 0x7f800000u;
        u32x2 code = {0, 0};
        float scale;
        if constexpr (KIND == E4M3) {
            // 448 = 1.75 x 2^8: exponent of the maximum minus 8, one more when its mantissa is above 1.75
            int e = (int)(ub >> 23) - ((ub & 0x7fffffu) > 0x600000u ? 7 : 8);
            e = max(e, 1);
            scale = __uint_as_float((unsigned)e << 23);
            const float inv = __uint_as_float((unsigned)(254 - e) << 23);  // e <= 248: a normal number
            if (!bad) {
                int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
                code.x = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, c, true);
                c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] * inv, x[5] * inv, 0, false);
                code.y = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[6] * inv, x[7] * inv, c, true);
            }
        } else {
            scale = fmaxf(__uint_as_float(ub) * (1.0f / 127.0f), SCALE_MIN);
            const float inv = 1.0f / scale;
            if (!bad) {
                unsigned c[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) c[i] = (unsigned)int8_code(x[i], scale, inv) & 255u;
                code.x = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
                code.y = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
            }
        }
        if (bad) scale = __uint_as_float(0x7fc00000u);
        if constexpr (F32) {
            *(unsigned *)dst = code.x;
            *(unsigned *)(dst + DH / 2) = code.y;
        } else {
            *(u32x2 *)dst = code;
        }
        if (sub == 0) *scale_at = scale;
    }
}
template <int KIND, int DH, bool F32> __device__ __forceinline__ void read_row(const char *src, const float *scale_at, float (&x)[8], int sub) {
    src += first_of<F32, DH>(sub) * elem_bytes<KIND>();
    if constexpr (KIND == BF16) {
        u32x4 a;
        if constexpr (F32) {
            const u32x2 lo = *(const u32x2 *)src, hi = *(const u32x2 *)(src + DH);
            a = u32x4{lo.x, lo.y, hi.x, hi.y};
        } else {
            a = *(const u32x4 *)src;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(a[i] << 16);
            x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
        }
    } else {
        u32x2 c;
        if constexpr (F32) c = u32x2{*(const unsigned *)src, *(const unsigned *)(src + DH / 2)};
        else c = *(const u32x2 *)src;
        const float s = *scale_at;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (KIND == E4M3) {
                const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
                x[4 * i] = lo.x * s;
                x[4 * i + 1] = lo.y * s;
                x[4 * i + 2] = hi.x * s;
                x[4 * i + 3] = hi.y * s;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * i + e] = (float)(signed char)(c[i] >> (8 * e)) * s;
            }
        }
    }
}

constexpr int KT = 256;  // threads of a workgroup

// One group of DH / 8 lanes per (row, head): its key and its value, 8 elements a lane.
template <int KIND, int DH, bool F32, bool WRITE>
__global__ __launch_bounds__(KT) void kv_rows_kernel(KvView V, const void *__restrict__ kr, const void *__restrict__ vr, void *__restrict__ kw,
                                                     void *__restrict__ vw, int64_t row_stride, int64_t head_stride, int64_t n_items) {
    constexpr int L = DH / 8;
    const int64_t item = (int64_t)blockIdx.x * (KT / L) + threadIdx.x / L;
    const int sub = threadIdx.x % L;
    if (item >= n_items) return;  // whole groups leave together
    const int t = (int)(item / V.n_kv_heads), h = (int)(item % V.n_kv_heads);
    const int b = kv_seq_of_row(V, t);
    if (b < 0) return;
    const int64_t p = (int64_t)V.kv_len[b] - ((int64_t)V.cu[b + 1] - t);
    const int page = p >= 0 ? kv_page(V, b, p) : -1;
    const int64_t at = t * row_stride + h * head_stride + first_of<F32, DH>(sub);
    const int64_t off = page * V.page_stride + h * V.head_stride + (p & V.mask) * V.row_stride;
    const int64_t soff = page * V.s_page + h * V.s_head + (p & V.mask) * V.s_row;
    if constexpr (WRITE) {
        if (page < 0) return;
        float x[8], y[8];
        load8<F32, DH>(kr, at, x);
        load8<F32, DH>(vr, at, y);
        write_row<KIND, DH, F32>(V.k + off * elem_bytes<KIND>(), V.ks + soff, x, sub);
        write_row<KIND, DH, F32>(V.v + off * elem_bytes<KIND>(), V.vs + soff, y, sub);
    } else {
        float x[8] = {}, y[8] = {};
        if (page >= 0) {
            read_row<KIND, DH, F32>(V.k + off * elem_bytes<KIND>(), V.ks + soff, x, sub);
            read_row<KIND, DH, F32>(V.v + off * elem_bytes<KIND>(), V.vs + soff, y, sub);
        }
        store8<F32, DH>(kw, at, x);
        store8<F32, DH>(vw, at, y);
    }
}

template <bool WRITE>
void launch_rows(const mw_kv_cache &c, const mw_kv_batch &b, int dtype, const void *k, const void *v, void *kw, void *vw, int64_t row_stride,
                 int64_t head_stride, hipStream_t st) {
    check_kv_rows(c, b, dtype, WRITE ? k : kw, WRITE ? v : vw, row_stride, head_stride, WRITE);
    if (b.n_rows == 0 || b.n_seqs == 0) return;
    const KvView V = make_view(c, b);
    const int64_t items = (int64_t)b.n_rows * c.n_kv_heads;
    const int per = KT / (c.head_dim / 8);
    const int64_t blocks = ceil_div<int64_t>(items, per);
#define KV_GO(KIND, DH, F32) \
    hipLaunchKernelGGL((kv_rows_kernel<KIND, DH, F32, WRITE>), dim3((unsigned)blocks), dim3(KT), 0, st, V, k, v, kw, vw, row_stride, head_stride, items)
#define KV_DIM(KIND)                                                  \
    do {                                                              \
        if (c.head_dim == 64) {                                       \
            if (dtype == MW_ELEM_F32) KV_GO(KIND, 64, true);          \
            else KV_GO(KIND, 64, false);                              \
        } else {                                                      \
            if (dtype == MW_ELEM_F32) KV_GO(KIND, 128, true);         \
            else KV_GO(KIND, 128, false);                             \
        }                                                             \
    } while (0)
    if (c.dtype == BF16) KV_DIM(BF16);
    else if (c.dtype == E4M3) KV_DIM(E4M3);
    else KV_DIM(INT8);
#undef KV_DIM
#undef KV_GO
    MW_HIP(hipGetLastError());
}

}  // namespace

void launch_kv_write(const mw_kv_cache &c, const mw_kv_batch &b, int dtype, const void *k, const void *v, int64_t row_stride,
                     int64_t head_stride, hipStream_t st) {
    launch_rows<true>(c, b, dtype, k, v, nullptr, nullptr, row_stride, head_stride, st);
}
void launch_kv_read(const mw_kv_cache &c, const mw_kv_batch &b, int dtype, void *k, void *v, int64_t row_stride, int64_t head_stride,
                    hipStream_t st) {
    launch_rows<false>(c, b, dtype, nullptr, nullptr, k, v, row_stride, head_stride, st);
}

}  // namespace mw
