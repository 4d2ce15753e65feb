// Matrix product in 8-bit integers with one scale per row of the input (a pixel of a 1x1 convolution, a token) and one
// per output channel, for gfx950 (MI355X): y3_quantize_rows_i8, y3_linear_i8_layout / _pack / _workspace_bytes, y3_linear_i8.
//
//   s_m = max(max_k |x_mk|, 127 * 2^-126) / 127        q_mk = round_half_even(x_mk * (127 / max_k |x_mk|))
//   y_mn = act((float(sum_k q_mk w_nk) * t_n) * s_m + b_n)
//
// The sum is exact: v_mfma_i32_16x16x64_i8 accumulates in 32-bit integers and 128^2 * k < 2^31 for every k accepted, so no
// order of summation, tile or split changes a bit of it.  What is rounded: x to q (half a step of s_m, the definition), the
// integer sum to fp32 (2^-24), one product, one fused multiply-add, and the store to bf16 where that is asked for.
//
// Packed weights: MFMA fragments, [n_pad / 16][k_pad / 64][64 lanes][16 bytes]; lane l of a fragment holds channel l & 15,
// inputs 16 (l >> 4) .. + 15 of the 64.  A wave's fragment load is one contiguous KB whatever n and k are.
#include "common.h"

typedef __attribute__((ext_vector_type(4))) int i32x4;

namespace {

constexpr float QTINY = 127.0f * 1.17549435082228750797e-38f;        // 127 * 2^-126: the scale of any row is a normal number

// 16 / 8 bytes at any element's alignment: global memory takes unaligned vector accesses
typedef u32x4 __attribute__((aligned(2))) u32x4_u2;
typedef u32x4 __attribute__((aligned(4))) u32x4_u4;
typedef f32x4 __attribute__((aligned(4))) f32x4_u4;
typedef unsigned long long __attribute__((aligned(2))) u64_u2;

// ---- eight consecutive elements of a row as fp32 bit patterns ------------------------------------------------------
template <int DT> struct Chunk;
template <> struct Chunk<Y3_BF16> {
    static __device__ __forceinline__ void load(const char *row, long k0, int left, unsigned (&v)[8]) {
        const unsigned short *p = (const unsigned short *)row + k0;
        if (left >= 8) {
            const u32x4 r = *(const u32x4_u2 *)p;
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[2 * j] = r[j] << 16; v[2 * j + 1] = r[j] & 0xffff0000u; }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < left ? (unsigned)p[j] << 16 : 0u;
        }
    }
};
template <> struct Chunk<Y3_F32> {
    static __device__ __forceinline__ void load(const char *row, long k0, int left, unsigned (&v)[8]) {
        const unsigned *p = (const unsigned *)row + k0;
        if (left >= 8) {
            const u32x4 a = *(const u32x4_u4 *)p, b = *(const u32x4_u4 *)(p + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0u;
        }
    }
};

// largest magnitude as a bit pattern: integers order like magnitudes, with infinities and NaN above every finite value
__device__ __forceinline__ unsigned amax8(const unsigned (&v)[8], unsigned m) {
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, v[j] & 0x7fffffffu);
    return m;
}

struct RowScale { float s, inv; bool finite; };
__device__ __forceinline__ RowScale row_scale(unsigned amax_bits) {
    RowScale r;
    r.finite = amax_bits < 0x7f800000u;
    const float a = fmaxf(__uint_as_float(amax_bits), QTINY);
    r.s = r.finite ? a / 127.0f : __builtin_nanf("");       // a row with a NaN or an infinity: every product of it is NaN
    r.inv = 127.0f / a;
    return r;
}

// 8 quantised bytes.  Adding 1.5 * 2^23 rounds half to even and leaves the integer in the low byte (two's complement);
// the product is rounded to fp32 first (no fused multiply-add), as the definition says.
__device__ __forceinline__ unsigned q4(unsigned a, unsigned b, unsigned c, unsigned d, float inv) {
    constexpr float MAGIC = 12582912.0f;
    const unsigned qa = __float_as_uint(__uint_as_float(a) * inv + MAGIC), qb = __float_as_uint(__uint_as_float(b) * inv + MAGIC);
    const unsigned qc = __float_as_uint(__uint_as_float(c) * inv + MAGIC), qd = __float_as_uint(__uint_as_float(d) * inv + MAGIC);
    const unsigned lo = __builtin_amdgcn_perm(qb, qa, 0x0c0c0400u);     // bytes {a, b, 0, 0}
    const unsigned hi = __builtin_amdgcn_perm(qd, qc, 0x04000c0cu);     // bytes {0, 0, c, d}
    return lo | hi;
}

__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o));
    return v;
}

// ---- rows -> 8-bit rows + scales --------------------------------------------------------------------------------
// One workgroup of TPR threads per row, the row read twice (the second time from cache).
template <int DT, int TPR>
__global__ __launch_bounds__(TPR) void quant_rows_kernel(const char *x, long x_ld, long rows, int k, char *q, long q_ld, int k_fill, float *scale) {
    __shared__ unsigned red[TPR / 64];
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const char *xr = x + row * x_ld * (DT == Y3_BF16 ? 2 : 4);
    char *qr = q + row * q_ld;
    unsigned m = 0;
    for (int k0 = threadIdx.x * 8; k0 < k; k0 += TPR * 8) {
        unsigned v[8];
        Chunk<DT>::load(xr, k0, k - k0, v);
        m = amax8(v, m);
    }
    m = wave_umax(m);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
        __syncthreads();
        m = red[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) m = max(m, red[w]);
    }
    const RowScale r = row_scale(m);
    for (int k0 = threadIdx.x * 8; k0 < k_fill; k0 += TPR * 8) {
        unsigned v[8];
        Chunk<DT>::load(xr, k0, k - k0, v);
        unsigned lo = q4(v[0], v[1], v[2], v[3], r.inv), hi = q4(v[4], v[5], v[6], v[7], r.inv);
        if (!r.finite) lo = hi = 0;
        *(unsigned long long *)(qr + k0) = (unsigned long long)hi << 32 | lo;
    }
    if (threadIdx.x == 0) scale[row] = r.s;
    __syncthreads();                                        // (red is written again)
    }
}

// 8-bit rows of any pitch and alignment -> rows on a 16-byte pitch, zero filled
__global__ __launch_bounds__(256) void repitch_rows_kernel(const char *x, long x_ld, long rows, int k, char *q, long q_ld, int k_fill) {
    for (long row = blockIdx.x; row < rows; row += gridDim.x)
        for (int k0 = threadIdx.x; k0 < k_fill; k0 += 256) q[row * q_ld + k0] = k0 < k ? x[row * x_ld + k0] : 0;
}

// rows [n][ld] of 8-bit weights -> fragments
__global__ __launch_bounds__(256) void pack_i8_kernel(const char *w, long ld, int n, int k, int kb_total, long chunks, char *packed) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;               // one 16-byte lane of a fragment
    if (i >= chunks) return;
    const long frag = i >> 6;
    const int lane = (int)(i & 63), ch = (int)(frag / kb_total) * 16 + (lane & 15);
    const int k0 = (int)(frag % kb_total) * 64 + (lane >> 4) * 16;
    unsigned r[4] = {0, 0, 0, 0};
    if (ch < n)
        for (int j = 0; j < 16; ++j)
            if (k0 + j < k) r[j >> 2] |= (unsigned)(unsigned char)w[ch * ld + k0 + j] << (8 * (j & 3));
    *(u32x4 *)(packed + i * 16) = u32x4{r[0], r[1], r[2], r[3]};
}

// float weights [n][ld] -> fragments + scales: one workgroup per channel
template <int DT>
__global__ __launch_bounds__(256) void pack_float_kernel(const char *w, long ld, int n, int k, int kb_total, char *packed, float *scale) {
    __shared__ unsigned red[4];
    const int ch = blockIdx.x;                                          // < n_pad
    const char *wr = w + (long)ch * ld * (DT == Y3_BF16 ? 2 : 4);
    const int kk = ch < n ? k : 0;
    unsigned m = 0;
    for (int k0 = threadIdx.x * 8; k0 < kk; k0 += 256 * 8) {
        unsigned v[8];
        Chunk<DT>::load(wr, k0, kk - k0, v);
        m = amax8(v, m);
    }
    m = wave_umax(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = max(max(red[0], red[1]), max(red[2], red[3]));
    const RowScale r = row_scale(m);
    for (int k0 = threadIdx.x * 8; k0 < kb_total * 64; k0 += 256 * 8) {
        unsigned v[8];
        Chunk<DT>::load(wr, k0, kk - k0, v);
        unsigned lo = q4(v[0], v[1], v[2], v[3], r.inv), hi = q4(v[4], v[5], v[6], v[7], r.inv);
        if (!r.finite) lo = hi = 0;
        const long frag = (long)(ch >> 4) * kb_total + (k0 >> 6);
        const int lane = (ch & 15) + 16 * ((k0 >> 4) & 3);
        *(unsigned long long *)(packed + frag * 1024 + lane * 16 + (k0 & 8)) = (unsigned long long)hi << 32 | lo;
    }
    if (threadIdx.x == 0 && ch < n) scale[ch] = r.s;
}

// ---- the product ------------------------------------------------------------------------------------------------
struct LinArgs {
    const char *x;                     // 8-bit rows, 16-byte pitch and alignment
    const float *x_scale;
    const char *w;
    const float *w_scale, *bias;       // bias may be null
    char *out;
    long rows, x_ld, out_ld;
    int k16, n, kb;                    // k rounded up to 16 (bytes of a row that may be read), channels, 64-deep k-blocks
    int leaky, n_blocks;
};

// four channels nl .. nl + 3 of one row
template <int OUT>
__device__ __forceinline__ void store4(const LinArgs &p, long row, int nl, const i32x4 &acc, float s) {
    if (row >= p.rows || nl >= p.n) return;
    const bool full = nl + 4 <= p.n;
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = full ? nl + j : min(nl + j, p.n - 1);
        y[j] = fmaf((float)acc[j] * p.w_scale[c], s, p.bias ? p.bias[c] : 0.0f);
        if (p.leaky) y[j] = y[j] > 0.0f ? y[j] : 0.1f * y[j];
    }
    if constexpr (OUT == Y3_F32) {
        float *o = (float *)p.out + row * p.out_ld + nl;
        if (full) *(f32x4_u4 *)o = f32x4{y[0], y[1], y[2], y[3]};
        else
            for (int j = 0; j < p.n - nl; ++j) o[j] = y[j];
    } else {
        unsigned short *o = (unsigned short *)p.out + row * p.out_ld + nl;
        if (full) *(u64_u2 *)o = (unsigned long long)pack_bf16x2(y[2], y[3]) << 32 | pack_bf16x2(y[0], y[1]);
        else
            for (int j = 0; j < p.n - nl; ++j) o[j] = f32_to_bf16(y[j]);
    }
}

// Four waves per workgroup, each 16 rows x 64 channels, everything straight from global memory.
template <int OUT>
__global__ __launch_bounds__(256) void linear_i8_kernel(const LinArgs p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int nb = blockIdx.x % p.n_blocks;
    const long m0 = ((long)(blockIdx.x / p.n_blocks) * 4 + wave) * 16;
    if (m0 >= p.rows) return;
    const long row = m0 + (lane & 15), rr = row < p.rows ? row : p.rows - 1;
    const char *xr = p.x + rr * p.x_ld;
    const int frags = (p.n + 15) / 16;
    i32x4 acc[4] = {};
    for (int kb = 0; kb < p.kb; ++kb) {
        const int k0 = kb * 64 + (lane >> 4) * 16;
        i32x4 xf = {};
        if (k0 < p.k16) xf = *(const i32x4 *)(xr + k0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (nb * 4 + i >= frags) break;
            const i32x4 wf = *(const i32x4 *)(p.w + (((long)(nb * 4 + i) * p.kb + kb) * 64 + lane) * 16);
            acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, xf, acc[i], 0, 0, 0);
        }
    }
    const float s = p.x_scale[rr];
#pragma unroll
    for (int i = 0; i < 4; ++i) store4<OUT>(p, row, (nb * 4 + i) * 16 + (lane >> 4) * 4, acc[i], s);
}

constexpr int MAX_K = 131071;          // 128 * 128 * k < 2^31
long round_up(long v, long m) { return (v + m - 1) / m * m; }
int es_of(int dt) { return dt == Y3_F32 ? 4 : dt == Y3_BF16 ? 2 : 1; }

int check_desc(const y3_linear_i8_desc *d) {
    Y3_REQUIRE(d, Y3_E_INVALID, "linear_i8: null descriptor");
    Y3_REQUIRE(d->dtype == Y3_F32 || d->dtype == Y3_BF16 || d->dtype == Y3_I8, Y3_E_INVALID, "linear_i8: dtype %d", d->dtype);
    Y3_REQUIRE(d->out_dtype == Y3_F32 || d->out_dtype == Y3_BF16, Y3_E_INVALID, "linear_i8: out_dtype %d", d->out_dtype);
    Y3_REQUIRE(d->k >= 1 && d->k <= MAX_K, Y3_E_INVALID, "linear_i8: k = %d outside 1 .. %d", d->k, MAX_K);
    Y3_REQUIRE(d->n >= 1 && d->n <= (1 << 24), Y3_E_INVALID, "linear_i8: n = %d outside 1 .. 2^24", d->n);
    Y3_REQUIRE(d->k_pad == round_up(d->k, 128) && d->n_pad == round_up(d->n, 16), Y3_E_INVALID,
               "linear_i8: k_pad %d / n_pad %d are not y3_linear_i8_layout's", d->k_pad, d->n_pad);
    Y3_REQUIRE(d->rows >= 0 && d->rows <= (1ll << 40) / d->k_pad, Y3_E_INVALID, "linear_i8: %lld rows", (long long)d->rows);
    Y3_REQUIRE((d->flags & ~Y3_CONV_LEAKY) == 0, Y3_E_INVALID, "linear_i8: flags 0x%x", d->flags);
    Y3_REQUIRE(d->x_ld >= d->k && d->out_ld >= d->n, Y3_E_INVALID, "linear_i8: x_ld %lld < k or out_ld %lld < n",
               (long long)d->x_ld, (long long)d->out_ld);
    return Y3_OK;
}

unsigned rows_grid(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : 1 << 20); }

template <int TPR>
void launch_quant(int dtype, const void *x, int64_t rows, int k, int64_t x_ld, void *q, int64_t q_ld, int k_fill, float *scale, hipStream_t st) {
    const unsigned grid = rows_grid(rows);
    if (dtype == Y3_BF16) hipLaunchKernelGGL((quant_rows_kernel<Y3_BF16, TPR>), dim3(grid), dim3(TPR), 0, st, (const char *)x, (long)x_ld, (long)rows, k, (char *)q, (long)q_ld, k_fill, scale);
    else hipLaunchKernelGGL((quant_rows_kernel<Y3_F32, TPR>), dim3(grid), dim3(TPR), 0, st, (const char *)x, (long)x_ld, (long)rows, k, (char *)q, (long)q_ld, k_fill, scale);
}

bool overlap(const void *a, long na, const void *b, long nb) {
    return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

}  // namespace

extern "C" int y3_quantize_rows_i8(int dtype, const void *x, int64_t rows, int k, int64_t x_ld, void *q, int64_t q_ld, float *scale, void *stream) {
    Y3_REQUIRE(dtype == Y3_F32 || dtype == Y3_BF16 || dtype == Y3_I8, Y3_E_INVALID, "quantize_rows_i8: dtype %d", dtype);
    Y3_REQUIRE(k >= 1 && k <= MAX_K, Y3_E_INVALID, "quantize_rows_i8: k = %d outside 1 .. %d", k, MAX_K);
    Y3_REQUIRE(rows >= 0 && rows <= (1ll << 40) / k, Y3_E_INVALID, "quantize_rows_i8: %lld rows", (long long)rows);
    Y3_REQUIRE(x_ld >= k, Y3_E_INVALID, "quantize_rows_i8: x_ld %lld < k", (long long)x_ld);
    Y3_REQUIRE(q_ld >= round_up(k, 16) && q_ld % 16 == 0, Y3_E_ALIGN, "quantize_rows_i8: q_ld %lld must be a multiple of 16 that holds k", (long long)q_ld);
    if (rows == 0) return Y3_OK;
    Y3_REQUIRE(x && q && (scale || dtype == Y3_I8), Y3_E_INVALID, "quantize_rows_i8: null pointer");
    Y3_REQUIRE((uintptr_t)x % es_of(dtype) == 0 && aligned16(q) && (uintptr_t)scale % 4 == 0, Y3_E_ALIGN, "quantize_rows_i8: pointer not aligned");
    Y3_REQUIRE(!overlap(x, ((rows - 1) * x_ld + k) * es_of(dtype), q, rows * q_ld), Y3_E_INVALID, "quantize_rows_i8: x and q overlap");
    const hipStream_t st = (hipStream_t)stream;
    const int fill = (int)round_up(k, 16);
    if (dtype == Y3_I8) hipLaunchKernelGGL(repitch_rows_kernel, dim3(rows_grid(rows)), dim3(256), 0, st, (const char *)x, (long)x_ld, (long)rows, k, (char *)q, (long)q_ld, fill);
    else launch_quant<256>(dtype, x, rows, k, x_ld, q, q_ld, fill, scale, st);
    return y3_check_launch("quantize_rows_i8");
}

extern "C" int y3_linear_i8_layout(y3_linear_i8_desc *d) {
    Y3_REQUIRE(d, Y3_E_INVALID, "linear_i8: null descriptor");
    Y3_REQUIRE(d->k >= 1 && d->k <= MAX_K, Y3_E_INVALID, "linear_i8: k = %d outside 1 .. %d", d->k, MAX_K);
    Y3_REQUIRE(d->n >= 1 && d->n <= (1 << 24), Y3_E_INVALID, "linear_i8: n = %d outside 1 .. 2^24", d->n);
    d->k_pad = (int)round_up(d->k, 128);
    d->n_pad = (int)round_up(d->n, 16);
    return Y3_OK;
}

extern "C" int y3_linear_i8_pack(const y3_linear_i8_desc *d, int w_dtype, const void *w, int64_t w_ld, void *packed, float *scale, void *stream) {
    y3_linear_i8_desc l;
    Y3_REQUIRE(d, Y3_E_INVALID, "linear_i8_pack: null descriptor");
    l = *d;
    const int rc = y3_linear_i8_layout(&l);
    if (rc) return rc;
    Y3_REQUIRE(l.k_pad == d->k_pad && l.n_pad == d->n_pad, Y3_E_INVALID, "linear_i8_pack: k_pad %d / n_pad %d are not y3_linear_i8_layout's", d->k_pad, d->n_pad);
    Y3_REQUIRE(w_dtype == Y3_F32 || w_dtype == Y3_BF16 || w_dtype == Y3_I8, Y3_E_INVALID, "linear_i8_pack: dtype %d", w_dtype);
    Y3_REQUIRE(w_ld >= d->k, Y3_E_INVALID, "linear_i8_pack: w_ld %lld < k", (long long)w_ld);
    Y3_REQUIRE(w && packed && (scale || w_dtype == Y3_I8), Y3_E_INVALID, "linear_i8_pack: null pointer");
    Y3_REQUIRE((uintptr_t)w % es_of(w_dtype) == 0 && aligned16(packed) && (uintptr_t)scale % 4 == 0, Y3_E_ALIGN, "linear_i8_pack: pointer not aligned");
    const hipStream_t st = (hipStream_t)stream;
    const int kb = d->k_pad / 64;
    if (w_dtype == Y3_I8) {
        const long chunks = (long)d->n_pad / 16 * kb * 64;
        hipLaunchKernelGGL(pack_i8_kernel, dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, st, (const char *)w, (long)w_ld, d->n, d->k, kb, chunks, (char *)packed);
    } else if (w_dtype == Y3_BF16) hipLaunchKernelGGL(pack_float_kernel<Y3_BF16>, dim3(d->n_pad), dim3(256), 0, st, (const char *)w, (long)w_ld, d->n, d->k, kb, (char *)packed, scale);
    else hipLaunchKernelGGL(pack_float_kernel<Y3_F32>, dim3(d->n_pad), dim3(256), 0, st, (const char *)w, (long)w_ld, d->n, d->k, kb, (char *)packed, scale);
    return y3_check_launch("linear_i8_pack");
}

extern "C" int y3_linear_i8_workspace_bytes(const y3_linear_i8_desc *d, int64_t *bytes) {
    const int rc = check_desc(d);
    if (rc) return rc;
    Y3_REQUIRE(bytes, Y3_E_INVALID, "linear_i8: null pointer");
    *bytes = d->dtype == Y3_I8 ? 0 : round_up(d->rows * d->k_pad, 256) + round_up(d->rows * 4, 256);
    return Y3_OK;
}

extern "C" int y3_linear_i8(const y3_linear_i8_desc *d, const void *x, const float *x_scale, const void *w, const float *w_scale,
                            const float *bias, void *out, void *workspace, int64_t workspace_bytes, void *stream) {
    int rc = check_desc(d);
    if (rc) return rc;
    if (d->rows == 0) return Y3_OK;
    int64_t need = 0;
    rc = y3_linear_i8_workspace_bytes(d, &need);
    if (rc) return rc;
    Y3_REQUIRE(x && w && w_scale && out, Y3_E_INVALID, "linear_i8: null pointer");
    Y3_REQUIRE((d->dtype == Y3_I8) == (x_scale != nullptr), Y3_E_INVALID, "linear_i8: x_scale goes with 8-bit rows, and only with them");
    Y3_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), Y3_E_INVALID, "linear_i8: workspace of %lld bytes, needs %lld", (long long)workspace_bytes, (long long)need);
    Y3_REQUIRE((uintptr_t)x % es_of(d->dtype) == 0 && aligned16(w) && (uintptr_t)out % es_of(d->out_dtype) == 0 && aligned16(workspace) &&
               (uintptr_t)x_scale % 4 == 0 && (uintptr_t)w_scale % 4 == 0 && (uintptr_t)bias % 4 == 0, Y3_E_ALIGN, "linear_i8: pointer not aligned");
    if (d->dtype == Y3_I8) Y3_REQUIRE(aligned16(x) && d->x_ld % 16 == 0 && d->x_ld >= round_up(d->k, 16), Y3_E_ALIGN, "linear_i8: 8-bit rows start on 16 bytes: x_ld %lld", (long long)d->x_ld);
    const long x_bytes = ((d->rows - 1) * d->x_ld + (d->dtype == Y3_I8 ? round_up(d->k, 16) : d->k)) * es_of(d->dtype);
    const long out_bytes = ((d->rows - 1) * d->out_ld + d->n) * es_of(d->out_dtype);
    Y3_REQUIRE(!overlap(x, x_bytes, out, out_bytes), Y3_E_INVALID, "linear_i8: x and out overlap");
    const hipStream_t st = (hipStream_t)stream;
    LinArgs a;
    a.x = (const char *)x; a.x_scale = x_scale; a.x_ld = d->x_ld; a.k16 = (int)round_up(d->k, 16);
    if (d->dtype != Y3_I8) {
        float *s = (float *)((char *)workspace + round_up(d->rows * d->k_pad, 256));
        launch_quant<256>(d->dtype, x, d->rows, d->k, d->x_ld, workspace, d->k_pad, d->k_pad, s, st);
        rc = y3_check_launch("linear_i8 (rows)");
        if (rc) return rc;
        a.x = (const char *)workspace; a.x_scale = s; a.x_ld = d->k_pad; a.k16 = d->k_pad;
    }
    a.w = (const char *)w; a.w_scale = w_scale; a.bias = bias; a.out = (char *)out;
    a.rows = d->rows; a.out_ld = d->out_ld; a.n = d->n; a.kb = d->k_pad / 64; a.leaky = d->flags & Y3_CONV_LEAKY;
    a.n_blocks = (d->n + 63) / 64;
    const long grid = (d->rows + 63) / 64 * a.n_blocks;
    Y3_REQUIRE(grid < (1 << 24), Y3_E_INVALID, "linear_i8: grid of %ld workgroups", grid);
    if (d->out_dtype == Y3_BF16) hipLaunchKernelGGL(linear_i8_kernel<Y3_BF16>, dim3((unsigned)grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(linear_i8_kernel<Y3_F32>, dim3((unsigned)grid), dim3(256), 0, st, a);
    return y3_check_launch("linear_i8");
}
