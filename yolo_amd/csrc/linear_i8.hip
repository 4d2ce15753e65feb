// Matrix product in 8-bit integers with one scale per row of the input (a pixel of a 1x1 convolution, a token) and one
// per output channel, for gfx950 (MI355X): y3_quantize_rows_i8, y3_linear_i8_layout / _pack / _workspace_bytes, y3_linear_i8.
//
//   a_m = max(max_k |x_mk|, 127 * 2^-126)    s_m = a_m / 127    q_mk = round_half_even(x_mk * (127 * (1 / a_m)))
//   y_mn = act((float(sum_k q_mk w_nk) * t_n) * s_m + b_n)
//
// The sum is exact: v_mfma_i32_16x16x64_i8 accumulates in 32-bit integers and 128^2 * k < 2^31 for every k accepted, so no
// order of summation, tile or split changes a bit of it.  What is rounded: x to q (half a step of s_m, the definition), the
// integer sum to fp32 (2^-24), one product, one fused multiply-add, and the store to bf16 where that is asked for.
//
// Packed weights: MFMA fragments, [n_pad / 16][k_pad / 64][64 lanes][16 bytes]; lane l of a fragment holds channel l & 15,
// inputs 16 (l >> 4) .. + 15 of the 64.  A wave's fragment load is one contiguous KB whatever n and k are.
#include "linear_i8.h"
#include <type_traits>

namespace {

constexpr float QTINY = 127.0f * 1.17549435082228750797e-38f;        // 127 * 2^-126: the scale of any row is a normal number

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
__device__ __forceinline__ RowScale row_scale(unsigned amax_bits);
__device__ __forceinline__ unsigned q4(unsigned a, unsigned b, unsigned c, unsigned d, float inv);

// ---- the same eight elements as they are stored (registers are what a kernel that keeps many of them is short of) -------
typedef unsigned short __attribute__((ext_vector_type(2))) u16x2;
__device__ __forceinline__ unsigned pk_umax16(unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

template <int DT> struct Raw;
template <> struct Raw<Y3_BF16> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(const char *row, unsigned k0, int left, unsigned (&v)[4]) {
        const unsigned short *p = (const unsigned short *)(row + k0 * 2);
        if (left >= 8) {
            const u32x4 r = *(const u32x4_u2 *)p;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = r[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (2 * j < left ? p[2 * j] : 0u) | (2 * j + 1 < left ? (unsigned)p[2 * j + 1] << 16 : 0u);
        }
    }
    static __device__ __forceinline__ unsigned amax(const unsigned (&v)[4]) {      
        const unsigned m = magnitudes(v);
        return max(m << 16, m & 0xffff0000u);
    }
    // the largest magnitudes of the even and of the odd elements, as bf16 bits in the two halves
    static __device__ __forceinline__ unsigned magnitudes(const unsigned (&v)[4]) {
        unsigned m = v[0] & 0x7fff7fffu;
#pragma unroll
        for (int j = 1; j < 4; ++j) m = pk_umax16(m, v[j] & 0x7fff7fffu);
        return m;
    }
    static __device__ __forceinline__ unsigned long long quantize(const unsigned (&v)[4], float inv) {
        const unsigned lo = q4(v[0] << 16, v[0] & 0xffff0000u, v[1] << 16, v[1] & 0xffff0000u, inv);
        const unsigned hi = q4(v[2] << 16, v[2] & 0xffff0000u, v[3] << 16, v[3] & 0xffff0000u, inv);
        return (unsigned long long)hi << 32 | lo;
    }
};
template <> struct Raw<Y3_F32> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const char *row, unsigned k0, int left, unsigned (&v)[8]) { Chunk<Y3_F32>::load(row + k0 * 4, 0, left, v); }
    static __device__ __forceinline__ unsigned amax(const unsigned (&v)[8]) { return amax8(v, 0); }
    static __device__ __forceinline__ unsigned long long quantize(const unsigned (&v)[8], float inv) {
        return (unsigned long long)q4(v[4], v[5], v[6], v[7], inv) << 32 | q4(v[0], v[1], v[2], v[3], inv);
    }
};

__device__ __forceinline__ RowScale row_scale(unsigned amax_bits) {
    RowScale r;
    r.finite = amax_bits < 0x7f800000u;
    const float a = fmaxf(__uint_as_float(amax_bits), QTINY);
    r.s = r.finite ? a / 127.0f : __builtin_nanf("");       // a row with a NaN or an infinity: every product of it is NaN
    r.inv = 127.0f * (1.0f / a);                            // (two roundings: the definition)
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

// Maximum over the LPR lanes of a row, in all of them: DPP within 16, then the halves of 32 and 64 side by side.
template <int LPR, typename F> __device__ __forceinline__ unsigned lanes_max(unsigned v, F f) {
    v = f(v, dpp_u<0xB1>(v));
    v = f(v, dpp_u<0x4E>(v));
    v = f(v, dpp_u<0x141>(v));
    v = f(v, dpp_u<0x140>(v));
    if constexpr (LPR >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = f(s[0], s[1]);
    }
    if constexpr (LPR >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = f(s[0], s[1]);
    }
    return v;
}

// ---- rows -> 8-bit rows + scales --------------------------------------------------------------------------------
// TPR threads per row, 256 / TPR rows per workgroup (TPR = 64: a wave each), a thread's NI chunks kept in registers between
// the maximum and the division; rows of more than 8 TPR NI values are read twice, the second time from cache.  Bound by
// memory, or by the latency of one round trip: 24 rows of 8192 bf16 3.4 us, 8192 x 8192 fp32 63 us, 5.3 TB/s.
template <int DT, int TPR, int NI>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void quant_rows_kernel(const char *x, long x_ld, long rows, int k, char *q, long q_ld, int k_fill, float *scale) {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1, WAVES = TPR / 64;
    __shared__ unsigned red[RPB * WAVES];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    for (long row0 = (long)blockIdx.x * RPB; row0 < rows; row0 += (long)gridDim.x * RPB) {
        const long row = min(row0 + sub, rows - 1);                // (a row past the end: the last one once more, the same bytes)
        const char *xr = x + row * x_ld * (DT == Y3_BF16 ? 2 : 4);
        char *qr = q + row * q_ld;
        unsigned v[NI][Raw<DT>::N], m = 0;
        const auto fetch = [&](int g) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int k0 = (g + i * TPR + t) * 8;
                Raw<DT>::load(xr, k0, k - k0, v[i]);
            }
        };
        for (int g = 0; g * 8 < k; g += NI * TPR) {
            fetch(g);
#pragma unroll
            for (int i = 0; i < NI; ++i) m = max(m, Raw<DT>::amax(v[i]));
        }
        m = lanes_max<64>(m, [](unsigned a, unsigned b) { return max(a, b); });
        if constexpr (WAVES > 1) {
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; ++w) m = max(m, red[w]);
            __syncthreads();                                        // (red is written again)
        }
        const RowScale r = row_scale(m);
        for (int g = 0; g * 8 < k_fill; g += NI * TPR) {
            if (k_fill > NI * TPR * 8) fetch(g);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int k0 = (g + i * TPR + t) * 8;
                if (k0 < k_fill) *(unsigned long long *)(qr + k0) = r.finite ? Raw<DT>::quantize(v[i], r.inv) : 0;
            }
        }
        if (t == 0) scale[row] = r.s;
    }
}

// 8-bit rows of any pitch and alignment: 16 bytes of a row, `left` of them there
constexpr int I8_ANY = Y3_I8 + 1;
__device__ __forceinline__ u32x4 row16(const char *at, int left) {
    u32x4 v = {0, 0, 0, 0};
    if (left >= 16) __builtin_memcpy(&v, at, 16);
    else
#pragma unroll 1
        for (int j = 0; j < left; ++j) {
            const unsigned b = (unsigned)(unsigned char)at[j] << (8 * (j & 3));
#pragma unroll
            for (int w = 0; w < 4; ++w) v[w] |= j >> 2 == w ? b : 0;
        }
    return v;
}
// ... -> rows on a 16-byte pitch, zero filled: a wave each
__global__ __launch_bounds__(256) void repitch_rows_kernel(const char *x, long x_ld, long rows, int k, char *q, long q_ld, int k_fill) {
    for (long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (long)gridDim.x * 4)
        for (int k0 = (threadIdx.x & 63) * 16; k0 < k_fill; k0 += 1024) *(u32x4 *)(q + row * q_ld + k0) = row16(x + row * x_ld + k0, k - k0);
}

// rows [n][ld] of 8-bit weights -> fragments
__global__ __launch_bounds__(256) void pack_i8_kernel(const char *w, long ld, int n, int k, int kb_total, long chunks, char *packed) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (long)gridDim.x * 256) {          // one 16-byte lane of a fragment
        const long frag = i >> 6;
        const int lane = (int)(i & 63), ch = (int)(frag / kb_total) * 16 + (lane & 15);
        const int k0 = (int)(frag % kb_total) * 64 + (lane >> 4) * 16;
        unsigned r[4] = {0, 0, 0, 0};
        if (ch < n)
            for (int j = 0; j < 16; ++j)
                if (k0 + j < k) r[j >> 2] |= (unsigned)(unsigned char)w[ch * ld + k0 + j] << (8 * (j & 3));
        *(u32x4 *)(packed + i * 16) = u32x4{r[0], r[1], r[2], r[3]};
    }
}

// float weights [n][ld] -> fragments + scales: one workgroup per channel
template <int DT>
__global__ __launch_bounds__(256) void pack_float_kernel(const char *w, long ld, int n, int n_pad, int k, int kb_total, char *packed, float *scale) {
    __shared__ unsigned red[4];
    for (int ch = blockIdx.x; ch < n_pad; ch += gridDim.x) {
        const char *wr = w + (long)ch * ld * (DT == Y3_BF16 ? 2 : 4);
        const int kk = ch < n ? k : 0;
        unsigned m = 0;
        for (int k0 = threadIdx.x * 8; k0 < kk; k0 += 256 * 8) {
            unsigned v[8];
            Chunk<DT>::load(wr, k0, kk - k0, v);
            m = amax8(v, m);
        }
        m = lanes_max<64>(m, [](unsigned a, unsigned b) { return max(a, b); });
        __syncthreads();                                                // (red has been read)
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
}

// ---- the product ------------------------------------------------------------------------------------------------
// Panel kernel: a workgroup of eight waves takes 16 RT rows and 16 NT WN channels (WN WK = 8: WN waves side by side along the
// channels, WK along k).  The rows' 8-bit values are in LDS -- quantised there from float rows, all of k at once, or copied
// from 8-bit rows in slabs of k, the next one requested before this one is multiplied -- and every wave reads its weights as
// whole fragments straight into registers, one k-block ahead (waves along k: four): weights are used by one wave each, LDS
// would only add a copy.  Waves along k take aligned 8-bit rows as fragments from memory as well.
//   Bound by: few rows, the row's way from memory and its quantisation, then the weights', which are requested behind them
//   (1 x 4096 -> 4096, 17 MB: 5.0 us); the middle, the latencies of rows, weights and stores in turn (1777 x 1003 -> 777
//   fp32 10 us, 7.4 without the products); many rows, the CUs' reads of
//   weights from L2 and the stores, all workgroups in the same phase (23104 x 1024 -> 512: 24 us, 15.8 without the products,
//   21.3 without the stores).  Four k-blocks of weights ahead, or 96 and 128 rows at two waves a SIMD: no faster.
//   LDS: rows on a pitch of 32 bytes more than their length (16 rows on 16 different 16-byte slots), then per row its scale,
//   per channel its scale and bias; the area of the rows is used again for the sums of the waves along k.
constexpr int PN_THREADS = 512, PN_WAVES = 8;
constexpr int PN_LDS_MAX = 160 * 1024;
constexpr int pn_slab(int nt) { return nt == 4 ? 32 * 1024 : 64 * 1024; }        // bytes of a slab of 8-bit rows: two workgroups per CU, registers

// Float rows -> 8-bit rows in LDS.  A wave takes 64 / LPR rows at a time, LPR lanes each, a lane's CPL chunks of eight values
// LPR chunks apart, and NB such groups at once: all their loads are in flight together, the maxima of a group are one
// register, and lane n of every 16 divides for group n.  Rows from nr on repeat the last one.
template <int XT, int WAVES, int BM, int LPR, int CPL, int REGS>
struct FloatRows {
    static constexpr int ES = XT == Y3_BF16 ? 2 : 4, N = Raw<XT>::N, RG = 64 / LPR;
    static constexpr int FIT = REGS / N / CPL < 1 ? 1 : REGS / N / CPL, EACH = (BM / RG + WAVES - 1) / WAVES, NB0 = FIT < EACH ? FIT : EACH;
    static constexpr int NB = NB0 < 8 ? NB0 : 8, BATCH = WAVES * NB * RG;        // rows that all waves take at once
    unsigned v[NB][CPL][N];

    // every lane's chunks are whole and every group has its rows: nothing to look at
    static __device__ __forceinline__ bool full(const LinArgs &p, int nr) { return p.k == LPR * CPL * 8 && nr == BM; }
    static __device__ __forceinline__ int group_of(int n, int row0, int wave) { return min(row0 + (wave + WAVES * n) * RG, BM - RG); }
    static __device__ __forceinline__ int row_of(int n, int row0, int nr, int wave, int lane) {
        return min(row0 + (wave + WAVES * n) * RG + (LPR == 64 ? 0 : lane / LPR), nr - 1);
    }

    // rows row0 .. row0 + BATCH - 1 of the panel at x0
    template <bool FULL> __device__ __forceinline__ void load(const LinArgs &p, const char *x0, int row0, int nr, int wave, int lane) {
        const int l = lane & (LPR - 1);
        const long ld = p.x_ld * ES, lane_ld = (LPR == 64 ? 0 : lane / LPR) * ld;
        const auto request = [&](auto WHOLE) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const char *xr = FULL ? x0 + group_of(n, row0, wave) * ld + lane_ld : x0 + row_of(n, row0, nr, wave, lane) * ld;
#pragma unroll
                for (int c = 0; c < CPL; ++c) {
                    const int k0 = (l + c * LPR) * 8;
                    if constexpr (decltype(WHOLE)::value) Raw<XT>::load(xr, FULL ? k0 : min(k0, p.k - 8), 8, v[n][c]);
                    else Raw<XT>::load(xr, k0, p.k - k0, v[n][c]);
                }
            }
        };
        // Whole chunks: lanes past the end of k take the last one once more (the maximum stays, and their weights are zero)
        // instead of a branch at every load: 369664 rows of 384 -> 128: 139 -> 91 us.
        if (FULL || p.k % 8 == 0) request(std::true_type{});
        else request(std::false_type{});
    }

    // ... to LDS, with their scales.  The division is lane n's for group n.
    template <bool FULL> __device__ __forceinline__ void quantize(int k_bytes, int row0, int nr, char *rows_lds, int pitch, float *row_s, int wave, int lane) {
        const int l = lane & (LPR - 1), lane_pitch = (LPR == 64 ? 0 : lane / LPR) * pitch + l * 8;
        unsigned m[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            if constexpr (XT == Y3_BF16) {
                m[n] = Raw<XT>::magnitudes(v[n][0]);
#pragma unroll
                for (int c = 1; c < CPL; ++c) m[n] = pk_umax16(m[n], Raw<XT>::magnitudes(v[n][c]));
                m[n] = max(m[n] >> 16, m[n] & 0xffffu);
            } else {
                m[n] = Raw<XT>::amax(v[n][0]);
#pragma unroll
                for (int c = 1; c < CPL; ++c) m[n] = max(m[n], Raw<XT>::amax(v[n][c]));
            }
        }
        if constexpr (XT == Y3_BF16 && NB % 2 == 0) {            // two groups' 16-bit maxima in one register
#pragma unroll
            for (int n = 0; n < NB; n += 2) {
                const unsigned both = lanes_max<LPR>(m[n] | m[n + 1] << 16, [](unsigned a, unsigned b) { return pk_umax16(a, b); });
                m[n] = both << 16;
                m[n + 1] = both & 0xffff0000u;
            }
        } else {
#pragma unroll
            for (int n = 0; n < NB; ++n) m[n] = lanes_max<LPR>(XT == Y3_BF16 ? m[n] << 16 : m[n], [](unsigned a, unsigned b) { return max(a, b); });
        }
        unsigned mine = m[0];
        int row = row_of(0, row0, nr, wave, lane);
#pragma unroll
        for (int n = 1; n < NB; ++n)
            if ((lane & 15) == n) { mine = m[n]; row = row_of(n, row0, nr, wave, lane); }
        const RowScale r = row_scale(mine);
        if (l < NB) row_s[row] = r.s;                            // (NB <= 8 <= LPR)
        const unsigned inv_bits = __float_as_uint(r.finite ? r.inv : 0.0f);
        const auto write = [&](auto NN) {
            constexpr int n = decltype(NN)::value;
            if constexpr (n < NB) {
                const float inv = __uint_as_float(dpp_u<0x150 + n>(inv_bits));
                char *to = rows_lds + (FULL ? group_of(n, row0, wave) * pitch + lane_pitch : row_of(n, row0, nr, wave, lane) * pitch + l * 8);
#pragma unroll
                for (int c = 0; c < CPL; ++c)
                    if (FULL || (l + c * LPR) * 8 < k_bytes) *(unsigned long long *)(to + c * LPR * 8) = Raw<XT>::quantize(v[n][c], inv);
                __builtin_amdgcn_sched_barrier(0);               // (one group after the other: registers)
            }
        };
        write(std::integral_constant<int, 0>{}); write(std::integral_constant<int, 1>{}); write(std::integral_constant<int, 2>{});
        write(std::integral_constant<int, 3>{}); write(std::integral_constant<int, 4>{}); write(std::integral_constant<int, 5>{});
        write(std::integral_constant<int, 6>{}); write(std::integral_constant<int, 7>{});
    }
};

template <int XT, int BM, int LPR, int CPL, int REGS>
__device__ __forceinline__ void quantize_panel(const LinArgs &p, const char *x0, int nr, char *rows_lds, int pitch, float *row_s, int wave, int lane) {
    typedef FloatRows<XT, PN_WAVES, BM, LPR, CPL, REGS> Rows;
    Rows rows;
    const bool full = Rows::full(p, nr);
    for (int row0 = 0; row0 + wave * Rows::RG < nr; row0 += Rows::BATCH) {
        if (full) rows.template load<true>(p, x0, row0, nr, wave, lane);
        else rows.template load<false>(p, x0, row0, nr, wave, lane);
        if (full) rows.template quantize<true>(p.kb * 64, row0, nr, rows_lds, pitch, row_s, wave, lane);
        else rows.template quantize<false>(p.kb * 64, row0, nr, rows_lds, pitch, row_s, wave, lane);
    }
}

// The wave's 16 RT x 16 NT block: scaled, activated and stored.  base: element (first row, first channel) of the block, the same
// in all lanes; row_bytes * 64 is below 2 GB; s(r): the scale of this lane's row of 16-row block r; rows: how many rows of the
// block there are; channels: of its channels, those that exist.
template <int RT, int NT, bool F32, typename S>
__device__ __forceinline__ void store_block(const LinArgs &p, char *base, int frow, int fq, const i32x4 (&acc)[RT][NT], const f32x4 (&t)[NT], const f32x4 (&b)[NT],
                                            int rows, int channels, S s) {
    constexpr int ES = F32 ? 4 : 2;
    const unsigned row_bytes = (unsigned)p.out_ld * ES, lane_row = (unsigned)frow * row_bytes;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        f32x4 y[NT];
        const float sr = s(r);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) y[i][j] = leaky_max(fmaf((float)acc[r][i][j] * t[i][j], sr, b[i][j]), p.slope);
        if (r * 16 + frow >= rows) continue;                     // (lanes that trade places in a swap share their row)
        char *o = base + (unsigned)(r * 16) * row_bytes;
        if (channels < 16 * NT) {                                // whole quads in one piece, the last one's channels one by one
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int left = channels - i * 16 - fq * 4;
                char *q = o + (lane_row + (unsigned)(i * 16 + fq * 4) * ES);
                if (left >= 4) {
                    if constexpr (F32) *(f32x4_u4 *)q = y[i];
                    else *(u64_u2 *)q = (unsigned long long)pack_bf16x2(y[i][2], y[i][3]) << 32 | pack_bf16x2(y[i][0], y[i][1]);
                } else {
#pragma unroll
                    for (int j = 0; j < 3; ++j)
                        if (j < left) {
                            if constexpr (F32) ((float *)q)[j] = y[i][j];
                            else ((unsigned short *)q)[j] = f32_to_bf16(y[i][j]);
                        }
                }
            }
        } else if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < NT; ++i) *(f32x4_u4 *)(o + (lane_row + fq * 16u) + i * 64) = y[i];
        } else if constexpr (NT == 1) {
            *(u64_u2 *)(o + lane_row + fq * 8u) = (unsigned long long)pack_bf16x2(y[0][2], y[0][3]) << 32 | pack_bf16x2(y[0][0], y[0][1]);
        } else {
#pragma unroll
            for (int i = 0; i < NT; i += 2) {                    // two blocks change places between quarter-waves: eight channels per lane
                const auto s0 = __builtin_amdgcn_permlane16_swap(pack_bf16x2(y[i][0], y[i][1]), pack_bf16x2(y[i + 1][0], y[i + 1][1]), false, false);
                const auto s1 = __builtin_amdgcn_permlane16_swap(pack_bf16x2(y[i][2], y[i][3]), pack_bf16x2(y[i + 1][2], y[i + 1][3]), false, false);
                *(u32x4_u2 *)(o + (lane_row + ((fq & 1) ? 16 + (fq - 1) * 4 : fq * 4) * 2u) + i * 32) = u32x4{s0[0], s1[0], s0[1], s1[1]};
            }
        }
    }
}

// Resident kernel: few enough weights for the registers of a workgroup (k up to 64 KB, channels up to 64 NT), many rows.
// Workgroups of four waves, two to four per CU, walk panels of 32 rows; a wave keeps the weights of its 16 NT channels for
// the whole launch and one panel's float rows on their way: the next panel is requested as soon as this one is quantised, and arrives
// under its products and stores.  LDS holds two panels, so that one barrier per panel is enough.  The waves of a SIMD
// belong to different workgroups, so that one's quantisation and stores (vector ALU) run beside the other's products; one
// workgroup of eight waves and 64 rows, all in step, took 37 us for 92416 x 512 -> 256, the panel kernel 38 us.  Bound by
// memory: 92416 x 512 -> 256 bf16 34.5 us, 4.1 TB/s.  Output rows that lie end to end but not on 16 bytes are put together
// in LDS (in a graph over different inputs and outputs: 92416 x 256 -> 255 fp32 34 us, stored quad by quad 40; bf16 28, 34;
// rows on 16 bytes, 256 channels, are not: bf16 38 that way, 26).  fp32 rows of k > 256 with n > 128 have 12 to 40 registers
// of the rows on their way in memory (92416 x 512 -> 256 in a graph 66 us, its bytes 46), ragged ones of k 129 to 256 with n
// <= 128 19.
constexpr int RS_THREADS = 256, RS_ROWS = 32;

// Workgroups per CU: what the registers allow for up to 128 channels (100000 x 100 -> 64 11.7 us, with two 15.9; 1478656 x 128
// -> 64 107, 119), two for more (92416 x 256 -> 256 fp32 with three 8 % slower: more rows written at a time).
constexpr int rs_per_cu(int xt, int kb, int nt) { return nt == 4 || kb > 8 || (xt == Y3_F32 && kb > 4) ? 2 : kb > 4 ? 3 : 4; }
// FULL: k = 8 LPR CPL and every panel has its rows (the launcher sees to that), so that no load looks at an end; not `flat`.
template <int XT, int LPR, int CPL, int KB, int NT, bool FULL, bool F32>
__global__ __launch_bounds__(RS_THREADS) __attribute__((amdgpu_waves_per_eu(rs_per_cu(XT, KB, NT), rs_per_cu(XT, KB, NT))))
void linear_i8_resident_kernel(const LinArgs p, int panels) {
    constexpr int BM = RS_ROWS, RT = 2, PITCH = KB * 64 + 32, PANEL = BM * PITCH;
    typedef FloatRows<XT, RS_THREADS / 64, BM, LPR, CPL, 1024> Rows;
    static_assert(Rows::BATCH >= BM, "a panel at once");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float *row_s = (float *)(smem + 2 * PANEL), *col_t = row_s + 2 * BM, *col_b = col_t + RS_THREADS / 4 * NT;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int frow = lane & 15, fq = lane >> 4;
    const int n0 = wave * 16 * NT, frags = (p.n + 15) >> 4;
    const auto rows_at = [&](int panel) { return FULL ? BM : (int)min(p.rows - (long)panel * BM, (long)BM); };
    const auto x_at = [&](int panel) { return p.x + (long)panel * BM * p.x_ld * (XT == Y3_BF16 ? 2 : 4); };

    Rows rows;
    const auto request = [&](int panel) {
        const int nr = rows_at(panel);
        rows.template load<FULL>(p, x_at(panel), 0, nr, wave, lane);
    };
    i32x4 wf[NT][KB];
    for (int c = tid; c < RS_THREADS / 4 * NT; c += RS_THREADS) {            // (in LDS: registers are for the weights)
        col_t[c] = p.w_scale[min(c, p.n - 1)];
        col_b[c] = p.bias ? p.bias[min(c, p.n - 1)] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const char *w = p.w + (long)min(wave * NT + i, frags - 1) * p.kb * 1024 + lane * 16;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            wf[i][kb] = i32x4{0, 0, 0, 0};
            if (kb < p.kb) wf[i][kb] = *(const i32x4 *)(w + kb * 1024);
        }
    }
    const auto quantize = [&](int panel, int buf) {
        const int nr = rows_at(panel);
        rows.template quantize<FULL>(KB * 64, 0, nr, smem + buf * PANEL, PITCH, row_s + buf * BM, wave, lane);
    };
    const int step = (int)gridDim.x;
    int panel = blockIdx.x;                                      // (the grid is at most `panels`)
    request(panel);
    __builtin_amdgcn_s_waitcnt(0x0f70);                          // vmcnt(0): nothing of this is waited for inside the loop
    quantize(panel, 0);
    if (panel + step < panels) request(panel + step);
    // Products of this panel, then the next one's 8-bit rows (its float rows have arrived), the request for the one after
    // it, and this panel's stores: the wait for float rows comes before stores that it would have to wait for as well.
    // k-blocks past the end of k multiply zero weights, by whatever LDS holds there (of the panel's own pitch).
    for (int buf = 0; panel < panels; buf ^= 1, panel += step) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        const int nr = rows_at(panel);
        i32x4 acc[RT][NT] = {};
        const char *xl = smem + buf * PANEL + frow * PITCH + fq * 16;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            if (kb % 2 == 0) __builtin_amdgcn_sched_barrier(0);  // (row fragments are read two k-blocks at a time, not all at once)
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const i32x4 xf = *(const i32x4 *)(xl + r * 16 * PITCH + kb * 64);
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[r][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[i][kb], xf, acc[r][i], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        float s[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r] = row_s[buf * BM + r * 16 + frow];
        if (panel + step < panels) {
            quantize(panel + step, buf ^ 1);
            if (panel + 2 * step < panels) request(panel + 2 * step);
        }
        const long m0 = (long)panel * BM;
        if (!FULL && p.flat) {                                   // rows end to end: by way of LDS, stored in whole lines
            constexpr int ES = F32 ? 4 : 2;
            char *ob = (char *)(col_b + RS_THREADS / 4 * NT), *o = p.out + m0 * p.out_ld * ES;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int ch = n0 + i * 16 + fq * 4;
                const f32x4 t = *(const f32x4 *)(col_t + ch), b = *(const f32x4 *)(col_b + ch);
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float y = leaky_max(fmaf((float)acc[r][i][j] * t[j], s[r], b[j]), p.slope);
                        char *at = ob + ((r * 16 + frow) * p.n + ch + j) * ES;
                        if (ch + j >= p.n) continue;
                        if constexpr (F32) *(float *)at = y;
                        else *(unsigned short *)at = f32_to_bf16(y);
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
            const int whole = nr * p.n * ES / 16;
            for (int c = tid; c < whole; c += RS_THREADS) *(u32x4 *)(o + c * 16) = *(const u32x4 *)(ob + c * 16);
            for (int e = whole * 16 / ES + tid; e < nr * p.n; e += RS_THREADS) {
                if constexpr (F32) ((float *)o)[e] = ((const float *)ob)[e];
                else ((unsigned short *)o)[e] = ((const unsigned short *)ob)[e];
            }
            __builtin_amdgcn_sched_barrier(0);
            continue;
        }
#pragma unroll
        for (int i0 = 0; i0 < NT; i0 += 2) {                     // two blocks of channels at a time: registers
            f32x4 t[2], b[2];
            i32x4 part[RT][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                t[i] = *(const f32x4 *)(col_t + n0 + (i0 + i) * 16 + fq * 4);
                b[i] = *(const f32x4 *)(col_b + n0 + (i0 + i) * 16 + fq * 4);
#pragma unroll
                for (int r = 0; r < RT; ++r) part[r][i] = acc[r][i0 + i];
            }
            if (n0 + i0 * 16 < p.n)
                store_block<RT, 2, F32>(p, p.out + (m0 * p.out_ld + n0 + i0 * 16) * (F32 ? 4 : 2), frow, fq, part, t, b, nr, p.n - n0 - i0 * 16, [&](int r) { return s[r]; });
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// (registers: the widest kernels, 8-bit rows and fp32 rows of up to 32 a workgroup take two workgroups per CU, the others
// three; 32 registers of 64 fp32 rows' kernel are in memory, 8 and 17 of the 64 x 512 ones of 8-bit rows, 2 of bf16 rows')
template <int XT, int RT, int NT, int WK>
__global__ __launch_bounds__(PN_THREADS) __attribute__((amdgpu_waves_per_eu(NT == 4 || XT >= Y3_I8 || (XT == Y3_F32 && RT <= 2) ? 4 : 6)))
void linear_i8_panel_kernel(const LinArgs p) {
    constexpr int REGS = NT == 4 ? 64 : 32;                      // of float rows on their way, per lane
    constexpr int BM = 16 * RT, wn_count = PN_WAVES / WK, cols = 16 * NT * wn_count;         // rows, channels of the workgroup
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int frow = lane & 15, fq = lane >> 4;
    const int wn = wave % wn_count, wk = wave / wn_count;
    const int pitch = p.slab * 64 + 32;
    const long m0 = (long)(blockIdx.x / p.n_groups) * BM;
    const int n0 = (int)(blockIdx.x % p.n_groups) * cols;
    const int nr = (int)(p.rows - m0 < BM ? p.rows - m0 : BM);   // rows that are there
    constexpr bool DIRECT = XT == Y3_I8 && WK > 1;               // few 8-bit rows: their fragments straight from memory, no panel
    const int area = max(DIRECT ? 0 : BM * pitch, WK > 1 ? PN_WAVES * RT * NT * 1024 : 0);
    float *row_s = (float *)(smem + area), *row_inv = row_s + BM, *col_t = row_inv + BM, *col_b = col_t + cols;
    unsigned *row_max = (unsigned *)row_inv;

    const int frags = (p.n + 15) >> 4;
    // this wave's fragments (past the last channel: the last one's), as offsets from the workgroup's first: below 64 MB
    const auto rs_w = __builtin_amdgcn_make_buffer_rsrc((void *)(p.w + (long)(n0 >> 4) * p.kb * 1024), 0, 0x7fffffff, 0x00020000);
    unsigned w_off[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) w_off[i] = (unsigned)min(wn * NT + i, frags - 1 - (n0 >> 4)) * (unsigned)p.kb * 1024u;

    for (int c = tid; c < cols; c += PN_THREADS) {
        const int ch = min(n0 + c, p.n - 1);
        col_t[c] = p.w_scale[ch];
        col_b[c] = p.bias ? p.bias[ch] : 0.0f;
    }
    if constexpr (XT >= Y3_I8) {
        if (tid < BM) row_s[tid] = p.x_scale[min(m0 + tid, p.rows - 1)];
    } else {
        const char *x0 = p.x + m0 * p.x_ld * (XT == Y3_BF16 ? 2 : 4);
        const int chunks = p.kb * 8;
        if (RT == 1 && (nr < PN_WAVES || chunks > 512)) {
            // few or long rows: all waves on the chunks of all of them, sixteen neighbouring lanes always in one row
            constexpr int NI = 4;                                // chunks a thread keeps between the two looks at them
            const int items = nr * chunks;
            if (tid < BM) row_max[tid] = 0;
            __syncthreads();
            const auto at = [&](int item, int &row, int &k0) {
                row = fast_div(item, p.fd_items);
                k0 = (item - row * chunks) * 8;
            };
            unsigned v[NI][Raw<XT>::N];
            const auto fetch = [&](int g) {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    int row, k0;
                    at(min(g + i * PN_THREADS + tid, items - 1), row, k0);
                    Raw<XT>::load(x0 + row * p.x_ld * (XT == Y3_BF16 ? 2 : 4), k0, p.k - k0, v[i]);
                }
            };
            for (int g = 0; g < items; g += NI * PN_THREADS) {
                fetch(g);
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    int row, k0;
                    at(min(g + i * PN_THREADS + tid, items - 1), row, k0);
                    const unsigned m = lanes_max<16>(Raw<XT>::amax(v[i]), [](unsigned a, unsigned b) { return max(a, b); });
                    if (frow == 0 && g + i * PN_THREADS + tid < items) atomicMax(&row_max[row], m);
                }
            }
            __syncthreads();
            if (tid < BM) {
                const RowScale r = row_scale(row_max[tid]);
                row_s[tid] = r.s;
                row_inv[tid] = r.finite ? r.inv : 0.0f;
            }
            __syncthreads();
            for (int g = 0; g < items; g += NI * PN_THREADS) {
                if (items > NI * PN_THREADS) fetch(g);
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    if (g + i * PN_THREADS + tid >= items) break;
                    int row, k0;
                    at(g + i * PN_THREADS + tid, row, k0);
                    *(unsigned long long *)(smem + row * pitch + k0) = Raw<XT>::quantize(v[i], row_inv[row]);
                }
            }
        } else if (chunks <= 16) quantize_panel<XT, BM, 16, 1, REGS>(p, x0, nr, smem, pitch, row_s, wave, lane);
        else if (chunks <= 32) quantize_panel<XT, BM, 32, 1, REGS>(p, x0, nr, smem, pitch, row_s, wave, lane);
        else if (chunks <= 64) quantize_panel<XT, BM, 64, 1, REGS>(p, x0, nr, smem, pitch, row_s, wave, lane);
        else if (chunks <= 128) quantize_panel<XT, BM, 64, 2, REGS>(p, x0, nr, smem, pitch, row_s, wave, lane);
        else if (chunks <= 256) quantize_panel<XT, BM, 64, 4, REGS>(p, x0, nr, smem, pitch, row_s, wave, lane);
        else quantize_panel<XT, BM, 64, 8, REGS>(p, x0, nr, smem, pitch, row_s, wave, lane);
    }

    i32x4 acc[RT][NT] = {};
    const auto weight = [&](int i, int kb) {
        return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs_w, lane * 16, w_off[i] + (unsigned)kb * 1024u, 0));
    };
    // 8-bit rows: a slab of k is on its way to registers while the one before it is multiplied
    constexpr int SLAB_REGS = XT >= Y3_I8 && !DIRECT ? pn_slab(NT) / PN_THREADS / 16 : 1;
    u32x4 sv[SLAB_REGS];
    const auto slab_chunk = [&](int j, int kbs, int &row, int &c) {         // 16 bytes c of row `row`, for this thread's j-th
        const int i = tid + j * PN_THREADS, per_row = kbs * 4;
        row = i / per_row;
        c = i - row * per_row;
        return i < nr * per_row;
    };
    const auto request_slab = [&](int s0) {
        if constexpr (XT >= Y3_I8 && !DIRECT) {
            const int kbs = min(p.slab, p.kb - s0);
#pragma unroll
            for (int j = 0; j < SLAB_REGS; ++j) {
                int row, c;
                sv[j] = u32x4{0, 0, 0, 0};
                if (!slab_chunk(j, kbs, row, c) || s0 * 64 + c * 16 >= p.k) continue;
                const char *at = p.x + (m0 + row) * p.x_ld + s0 * 64 + c * 16;
                sv[j] = XT == I8_ANY ? row16(at, p.k - s0 * 64 - c * 16) : *(const u32x4 *)at;
            }
        }
    };
    request_slab(0);
    for (int s0 = 0; s0 < p.kb; s0 += p.slab) {
        const int s_kb = min(p.slab, p.kb - s0);                 // k-blocks of this slab: an even number
        const auto slab = [&]() {
            if constexpr (XT >= Y3_I8 && !DIRECT) {
                if (s0) __syncthreads();                         // (the previous slab has been read)
#pragma unroll
                for (int j = 0; j < SLAB_REGS; ++j) {
                    int row, c;
                    if (slab_chunk(j, s_kb, row, c)) *(u32x4 *)(smem + row * pitch + c * 16) = sv[j];
                }
            }
            __syncthreads();
        };
        const char *xl[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) xl[r] = smem + min(r * 16 + frow, nr - 1) * pitch + fq * 16;
        if constexpr (WK == 1) {                                 // two k-blocks' weights in turn: one multiplied, one on its way
            i32x4 wa[NT], wb[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) wa[i] = weight(i, s0);
            slab();
            if (s0 + p.slab < p.kb) request_slab(s0 + p.slab);
            const auto multiply = [&](const i32x4 (&f)[NT], int at) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const i32x4 xf = *(const i32x4 *)(xl[r] + at);
#pragma unroll
                    for (int i = 0; i < NT; ++i) acc[r][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[i], xf, acc[r][i], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            for (int kb = 0; kb < s_kb; kb += 2) {
#pragma unroll
                for (int i = 0; i < NT; ++i) wb[i] = weight(i, s0 + kb + 1);
                multiply(wa, 0);
                const int next = min(s0 + kb + 2, p.kb - 1);
#pragma unroll
                for (int i = 0; i < NT; ++i) wa[i] = weight(i, next);
                multiply(wb, 64);
#pragma unroll
                for (int r = 0; r < RT; ++r) xl[r] += 128;
            }
        } else {                                                 // this wave's k-blocks: wk, wk + WK, ..., in groups of U
            static_assert(NT == 1, "waves along k have one block of channels");
            constexpr int U = 4;
            const int mine = s_kb > wk ? (s_kb - wk + WK - 1) / WK : 0;
            i32x4 wf[2][U], xg[2][U][DIRECT ? RT : 1];
            const char *xr[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) xr[r] = DIRECT ? p.x + (m0 + min(r * 16 + frow, nr - 1)) * p.x_ld : nullptr;
            const auto request = [&](int g, int buf) {           // (past the end: any fragment, not multiplied)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int kb = min(s0 + wk + (g * U + u) * WK, p.kb - 1);
                    wf[buf][u] = weight(0, kb);
                    if constexpr (DIRECT) {                      // (past the end of k the weights are zero: any bytes of the row)
                        const unsigned k0 = (unsigned)min(kb * 64 + fq * 16, p.k16 - 16);
#pragma unroll
                        for (int r = 0; r < RT; ++r) xg[buf][u][r] = *(const i32x4 *)(xr[r] + k0);
                    }
                }
            };
            request(0, 0);
            if constexpr (!DIRECT) {
                slab();
                if (s0 + p.slab < p.kb) request_slab(s0 + p.slab);
            }
            const auto multiply = [&](int g, int buf) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (g * U + u >= mine) break;
                    const int kb = wk + (g * U + u) * WK;
#pragma unroll
                    for (int r = 0; r < RT; ++r)
                        acc[r][0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[buf][u], DIRECT ? xg[buf][u][DIRECT ? r : 0] : *(const i32x4 *)(xl[r] + kb * 64), acc[r][0], 0, 0, 0);
                }
            };
            const int groups = (mine + U - 1) / U;
            for (int g = 0; g < groups; g += 2) {
                if (g + 1 < groups) request(g + 1, 1);
                multiply(g, 0);
                if (g + 1 < groups) {
                    if (g + 2 < groups) request(g + 2, 0);
                    multiply(g + 1, 1);
                }
            }
        }
    }

    const auto put = [&](int r, int c, const i32x4 &v) {         // 16 x 16 block: rows r .. r + 15, channels c .. c + 15 of the workgroup's
        store4(p, m0 + r + frow, n0 + c + fq * 4, v, row_s[r + frow], *(const f32x4 *)(col_t + c + fq * 4), *(const f32x4 *)(col_b + c + fq * 4));
    };
    if (WK == 1 && p.out_ld < (1 << 23)) {                       // (64 rows: below 2 GB)
        if (n0 + wn * NT * 16 >= p.n) return;
        f32x4 t[NT], b[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            t[i] = *(const f32x4 *)(col_t + (wn * NT + i) * 16 + fq * 4);
            b[i] = *(const f32x4 *)(col_b + (wn * NT + i) * 16 + fq * 4);
        }
        const int c = n0 + wn * NT * 16;
        char *base = p.out + (m0 * p.out_ld + c) * (p.out_f32 ? 4 : 2);
        if (p.out_f32) store_block<RT, NT, true>(p, base, frow, fq, acc, t, b, nr, p.n - c, [&](int r) { return row_s[r * 16 + frow]; });
        else store_block<RT, NT, false>(p, base, frow, fq, acc, t, b, nr, p.n - c, [&](int r) { return row_s[r * 16 + frow]; });
    } else if (WK == 1) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int i = 0; i < NT; ++i) put(r * 16, (wn * NT + i) * 16, acc[r][i]);
    } else {
        __syncthreads();                                         // (the rows have been read)
        i32x4 *sums = (i32x4 *)smem;                             // [wave][r][i][lane]
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int i = 0; i < NT; ++i) sums[((wave * RT + r) * NT + i) * 64 + lane] = acc[r][i];
        __syncthreads();
        for (int b = wave; b < wn_count * RT * NT; b += PN_WAVES) {          // block b = (wn, r, i)
            const int bw = b / (RT * NT), ri = b % (RT * NT);
            i32x4 v = sums[(bw * RT * NT + ri) * 64 + lane];
            for (int k = 1; k < WK; ++k) v += sums[((k * wn_count + bw) * RT * NT + ri) * 64 + lane];
            put(ri / NT * 16, (bw * NT + ri % NT) * 16, v);
        }
    }
}

int panel_area(int rt, int nt, int wk, int slab, bool direct) {
    const int rows = direct ? 0 : 16 * rt * (slab * 64 + 32), sums = wk > 1 ? PN_WAVES * rt * nt * 1024 : 0;
    return rows > sums ? rows : sums;
}
int panel_lds(int rt, int nt, int wk, int slab, bool direct) { return panel_area(rt, nt, wk, slab, direct) + (2 * 16 * rt + 2 * 16 * nt * (PN_WAVES / wk)) * 4; }

template <int XT, int RT, int NT, int WK>
int launch_panel_as(LinArgs a, hipStream_t st) {
    static thread_local int attr_dev = -1;
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (attr_dev != dev) {
        if (hipFuncSetAttribute((const void *)linear_i8_panel_kernel<XT, RT, NT, WK>, hipFuncAttributeMaxDynamicSharedMemorySize, PN_LDS_MAX) != hipSuccess) {
            y3_set_error("linear_i8: cannot reserve %d bytes of LDS", PN_LDS_MAX);
            return Y3_E_LAUNCH;
        }
        attr_dev = dev;
    }
    constexpr int cols = 16 * NT * (PN_WAVES / WK);
    a.n_groups = (a.n + cols - 1) / cols;
    constexpr bool lds_direct = XT == Y3_I8 && WK > 1;
    const long most = ((1 << 23) - 1) / a.n_groups * 16 * RT;    // rows of a grid (fewer than 2^32 threads)
    for (long m = 0; m < a.rows; m += most) {
        LinArgs s = a;
        s.rows = a.rows - m < most ? a.rows - m : most;
        s.x += m * a.x_ld * (XT == Y3_F32 ? 4 : XT == Y3_BF16 ? 2 : 1);
        if (XT >= Y3_I8) s.x_scale += m;
        s.out += m * a.out_ld * (a.out_f32 ? 4 : 2);
        hipLaunchKernelGGL((linear_i8_panel_kernel<XT, RT, NT, WK>), dim3((unsigned)((s.rows + 16 * RT - 1) / (16 * RT) * a.n_groups)), dim3(PN_THREADS),
                           panel_lds(RT, NT, WK, a.slab, lds_direct), st, s);
    }
    return y3_check_launch("linear_i8");
}

struct Panel { int rt, nt, wk, slab; };
int panel_fit(int bm) {                // k-blocks of bm rows that LDS holds, and quantize_panel takes (RT > 1: up to 4096)
    const int fit = (PN_LDS_MAX - 6 * 1024) / bm / 64 - 1;
    return bm > 16 && fit > 64 ? 64 : fit;
}
template <int XT> int launch_panel(const LinArgs &a, const Panel &c, hipStream_t st) {
    LinArgs b = a;
    b.slab = c.slab;
    b.fd_items = make_fastdiv(a.kb * 8);
    if (c.rt == 1) return c.wk == 2 ? launch_panel_as<XT, 1, 1, 2>(b, st) : c.wk == 4 ? launch_panel_as<XT, 1, 1, 4>(b, st) : launch_panel_as<XT, 1, 1, 8>(b, st);
    if (c.rt == 2) return c.nt == 1 ? launch_panel_as<XT, 2, 1, 1>(b, st) : launch_panel_as<XT, 2, 2, 1>(b, st);
    if (c.nt == 2) return launch_panel_as<XT, 4, 2, 1>(b, st);
    if constexpr (XT < Y3_I8)
        if (c.rt == 3) return launch_panel_as<XT, 3, 4, 1>(b, st);
    return launch_panel_as<XT, 4, 4, 1>(b, st);
}

template <int XT, int LPR, int CPL, int KB, int NT, bool FULL, bool F32>
int launch_resident_as(const LinArgs &a, long cus, hipStream_t st) {
    constexpr int ES = F32 ? 4 : 2, lds_most = 2 * RS_ROWS * (KB * 64 + 32) + 2 * RS_ROWS * 4 + 2 * (RS_THREADS / 4 * NT) * 4 + RS_ROWS * RS_THREADS / 4 * NT * ES;
    const int lds = lds_most - (a.flat ? 0 : RS_ROWS * RS_THREADS / 4 * NT * ES);
    static thread_local int attr_dev = -1;
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (attr_dev != dev) {
        if (hipFuncSetAttribute((const void *)linear_i8_resident_kernel<XT, LPR, CPL, KB, NT, FULL, F32>, hipFuncAttributeMaxDynamicSharedMemorySize, lds_most) != hipSuccess) {
            y3_set_error("linear_i8: cannot reserve %d bytes of LDS", lds_most);
            return Y3_E_LAUNCH;
        }
        attr_dev = dev;
    }
    const long panels = (a.rows + RS_ROWS - 1) / RS_ROWS, most = rs_per_cu(XT, KB, NT) * cus, groups = panels < 2 * most ? 2 * cus : most;
    hipLaunchKernelGGL((linear_i8_resident_kernel<XT, LPR, CPL, KB, NT, FULL, F32>), dim3((unsigned)(panels < groups ? panels : groups)), dim3(RS_THREADS), lds, st, a, (int)panels);
    return y3_check_launch("linear_i8 (resident)");
}
// Two panels per workgroup at least, and all channels and k in its registers.
template <int XT> bool resident_ok(const LinArgs &a, long cus) {
    return a.rows >= 2 * 2 * RS_ROWS * cus && a.rows <= RS_ROWS * 0x3fffffffl && a.n <= 256 && a.out_ld < (1 << 23) && a.kb <= (XT == Y3_BF16 && a.n <= 128 ? 12 : 8);
}
template <int XT, int NT, bool F32> int launch_resident(const LinArgs &a, long cus, hipStream_t st) {
    const bool whole = a.rows % RS_ROWS == 0 && !a.flat;
    if (a.kb <= 2) return whole && a.k == 128 ? launch_resident_as<XT, 16, 1, 2, NT, true, F32>(a, cus, st) : launch_resident_as<XT, 16, 1, 2, NT, false, F32>(a, cus, st);
    if (a.kb <= 4) return whole && a.k == 256 ? launch_resident_as<XT, 32, 1, 4, NT, true, F32>(a, cus, st) : launch_resident_as<XT, 32, 1, 4, NT, false, F32>(a, cus, st);
    if constexpr (XT == Y3_BF16 && NT == 2)
        if (a.kb > 8) return launch_resident_as<XT, 64, 2, 12, NT, false, F32>(a, cus, st);
    return whole && a.k == 512 ? launch_resident_as<XT, 64, 1, 8, NT, true, F32>(a, cus, st) : launch_resident_as<XT, 64, 1, 8, NT, false, F32>(a, cus, st);
}
template <int XT, int NT> int launch_resident_out(const LinArgs &a, long cus, hipStream_t st) {
    return a.out_f32 ? launch_resident<XT, NT, true>(a, cus, st) : launch_resident<XT, NT, false>(a, cus, st);
}
template <int XT> int launch_float(const LinArgs &a, const Panel &c, long cus, hipStream_t st) {
    if (!resident_ok<XT>(a, cus)) return launch_panel<XT>(a, c, st);
    return a.n <= 128 ? launch_resident_out<XT, 2>(a, cus, st) : launch_resident_out<XT, 4>(a, cus, st);
}

// The largest block of rows and channels (weights are read once per 16 RT rows, rows once per 16 NT WN channels) that does not
// leave half of the waves without channels and still gives six CUs in ten a workgroup.  RT, NT (WK), 8-bit rows, us: 512 x
// 4096 -> 4096: 2, 2 (256 workgroups) 24, 4, 2 (128) 31, 4, 4 (64) 48; 2048 rows: 62, 53, 57.  bfloat16 rows: 361 x 1024 ->
// 512: 1, 1, 2 (184) 4.1, 1, 1, 4 (368) 4.6; 8266 x 1717 -> 60: 1, 1, 2 11.5, 2, 1 14.7.  But
//   4, 2 from two workgroups per CU on, where two fit the LDS: 23104 x 512 -> 255 (361) 15.6, 2, 2 13.6; 46208 x 1024 -> 256
//   29.6, 31.9; 60000 x 1280 -> 256 (its rows fill half of the LDS) 67, 51;
//   2, 1 from half of the CUs on, as 16 rows are all that is left, with 8-bit rows (which 16 rows do without LDS, a fragment at
//   a time) from a third on: 128 x 4096 -> 4096 (128) 15.7, 1, 1, 2 (512) 23.7; 731 x 4096 -> 512 (92) 11.7, 20.3; 731 x 6624
//   -> 352 (69) 25.6, 1, 1, 4 17.4; bfloat16 200 x 1024 -> 2048 (112) 5.8, 1, 1, 2 5.3;
//   at most 32 k-blocks a wave where they are along k: 731 x 6624 -> 352 8-bit 1, 1, 2 (276) 25.0, 1, 1, 4 17.4;
//   3, 4 instead of 4, 4 where the fullest CU then has fewer rows (23104 x 1024 -> 512: 96 rows, 24.3, 128, 26.3; 16384: 96,
//   28.6, 64, 25.7), or where it fits the LDS twice (60000 x 1280 -> 512: 75, 88).
Panel panel_of(long rows, int n, int kb, int xt, long cus) {
    static const Panel all[] = {{4, 4, 1, 0}, {4, 2, 1, 0}, {2, 2, 1, 0}, {2, 1, 1, 0}, {1, 1, 2, 0}, {1, 1, 4, 0}, {1, 1, 8, 0}};
    const auto twice = [&](int rt) { return xt >= Y3_I8 || kb <= panel_fit(16 * rt) / 2; };
    const auto fullest = [&](int bm, long groups) { return ((rows + bm - 1) / bm * groups + cus - 1) / cus * bm; };
    Panel best = {0, 0, 0, 0};
    for (const Panel &c : all) {
        const int bm = 16 * c.rt, cols = 16 * c.nt * (PN_WAVES / c.wk);
        if (n <= cols / 2 && (c.nt > 1 || (c.wk < 8 && 2 * c.wk <= kb))) continue;
        if (c.rt > 1 && rows <= bm / 2) continue;
        if (c.wk > kb) continue;
        Panel t = c;
        t.slab = kb;
        if (xt >= Y3_I8) {
            const int most = pn_slab(c.nt) / bm / 64 / 2 * 2;
            t.slab = (c.wk > 1 && xt == Y3_I8) || kb < most ? kb : most;     // (waves along k read aligned 8-bit rows from memory)
        } else if (kb > panel_fit(bm)) continue;
        best = t;
        const long groups = (n + cols - 1) / cols, all_of = (rows + bm - 1) / bm * groups;
        if (c.rt == 4 && c.nt == 2 ? all_of < 2 * cus || !twice(4) : all_of < (c.rt == 2 && c.nt == 1 ? xt >= Y3_I8 ? cus / 3 : cus / 2 : cus * 6 / 10)) continue;
        if (c.wk > 1 && c.wk < 8 && kb > 32 * c.wk) continue;
        if (c.nt == 4 && xt < Y3_I8 && (fullest(48, groups) < fullest(64, groups) || (!twice(4) && twice(3) && all_of >= 2 * cus))) best.rt = 3;
        break;
    }
    return best;
}

constexpr int MAX_K = 131071;          // 128 * 128 * k < 2^31
long round_up(long v, long m) { return (v + m - 1) / m * m; }
int es_of(int dt) { return dt == Y3_F32 ? 4 : dt == Y3_BF16 ? 2 : 1; }

// Float rows go through the panel kernel at once where its LDS holds all of k for as many rows as it takes best; otherwise
// 8-bit rows are made in the workspace first.
//   Up to 16 rows are quantised by every workgroup, and 64K values take one as long as a launch does (16 rows of 4096 -> 4096:
//   7.3 us against 7.9, of 8192 -> 8192: 26 against 15.6).
//   One group of channels quantises each row once, 32 or 16 rows to a workgroup: 8000 x 4096 -> 200 24 us against 40, 60000 x
//   4096 -> 64 119, 192; from 4096 channels on 16 rows are no better than two launches (60000 x 8192 -> 64: 412, 369).
//   A tile for every CU and two million weights: a pass over the rows is little beside the product, which the tile kernel
//   computes faster (8192 x 2048 -> 4096: 116 us against 75, 16384 x 1024 -> 2048: 62, 54; fewer weights or tiles, 32768 x
//   1024 -> 1024: 58, 62, 65536 x 2048 -> 512: 125, 147, 4096 x 2048 -> 2048: 32, 35).
bool fused(const y3_linear_i8_desc *d) {
    const int bm = d->rows <= 32 ? 32 : 64;
    if (d->rows <= 16) return d->k_pad / 64 <= panel_fit(16) && d->rows * d->k_pad <= 65536;
    if (d->n <= 256 && d->k_pad <= 4096) return true;
    if (d->k_pad / 64 > panel_fit(bm)) return false;
    const long tiles = (d->rows + 255) / 256 * ((d->n + 255) / 256);
    return tiles < 256 || (long)d->n * d->k_pad < (1l << 21) || d->k_pad < 512;
}

// 8-bit rows that are read 16 aligned bytes at a time, up to k16
bool rows_aligned(const LinArgs &a) { return aligned16(a.x) && a.x_ld % 16 == 0 && a.x_ld >= a.k16; }

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
    Y3_REQUIRE(d->rows == 0 || (d->x_ld <= (1ll << 44) / d->rows && d->out_ld <= (1ll << 44) / d->rows), Y3_E_INVALID, "linear_i8: %lld rows on x_ld %lld, out_ld %lld",
               (long long)d->rows, (long long)d->x_ld, (long long)d->out_ld);
    Y3_REQUIRE(d->x_ld >= d->k && d->out_ld >= d->n, Y3_E_INVALID, "linear_i8: x_ld %lld < k or out_ld %lld < n",
               (long long)d->x_ld, (long long)d->out_ld);
    return Y3_OK;
}

unsigned rows_grid(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : 1 << 20); }

template <int DT, int TPR, int NI>
void launch_quant_as(const void *x, int64_t rows, int k, int64_t x_ld, void *q, int64_t q_ld, int k_fill, float *scale, hipStream_t st) {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    hipLaunchKernelGGL((quant_rows_kernel<DT, TPR, NI>), dim3(rows_grid((rows + RPB - 1) / RPB)), dim3(TPR < 256 ? 256 : TPR), 0, st, (const char *)x, (long)x_ld, (long)rows, k,
                       (char *)q, (long)q_ld, k_fill, scale);
}
// A wave per row where that fills the card; the fewer and longer the rows, the more threads each.
template <int DT>
void launch_quant(const void *x, int64_t rows, int k, int64_t x_ld, void *q, int64_t q_ld, int k_fill, float *scale, hipStream_t st) {
    if (rows < 512 && k > 4096) launch_quant_as<DT, 1024, 2>(x, rows, k, x_ld, q, q_ld, k_fill, scale, st);
    else if (k > 2048 || (rows < 2048 && k > 512)) launch_quant_as<DT, 256, 4>(x, rows, k, x_ld, q, q_ld, k_fill, scale, st);
    else launch_quant_as<DT, 64, 4>(x, rows, k, x_ld, q, q_ld, k_fill, scale, st);
}
void quantize_to(int dtype, const void *x, int64_t rows, int k, int64_t x_ld, void *q, int64_t q_ld, int k_fill, float *scale, hipStream_t st) {
    if (dtype == Y3_BF16) launch_quant<Y3_BF16>(x, rows, k, x_ld, q, q_ld, k_fill, scale, st);
    else launch_quant<Y3_F32>(x, rows, k, x_ld, q, q_ld, k_fill, scale, st);
}

bool overlap(const void *a, long na, const void *b, long nb) {
    return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}
// Rows of a_row bytes against rows of b_row bytes, `rows` each: two channel slices of one buffer (the same pitch, apart
// within it) do not overlap.
bool rows_overlap(const void *a, long a_pitch, long a_row, const void *b, long b_pitch, long b_row, long rows) {
    if (!overlap(a, (rows - 1) * a_pitch + a_row, b, (rows - 1) * b_pitch + b_row)) return false;
    if (a_pitch != b_pitch) return true;
    const long apart = ((long)((uintptr_t)b - (uintptr_t)a) % a_pitch + a_pitch) % a_pitch;
    return apart < a_row || apart + b_row > a_pitch;
}
// A block of bytes against rows: between two rows it may lie.
bool block_overlaps_rows(const void *block, long bytes, const void *base, long pitch, long row, long rows) {
    if (!block || bytes == 0 || !overlap(block, bytes, base, (rows - 1) * pitch + row)) return false;
    const long at = (long)((uintptr_t)block - (uintptr_t)base);      // (negative: it reaches into the first row)
    if (at < 0) return true;
    const long in_row = at % pitch;
    return in_row < row || (at / pitch + 1 < rows && in_row + bytes > pitch);
}

}  // namespace

extern "C" int y3_quantize_rows_i8(int dtype, const void *x, int64_t rows, int k, int64_t x_ld, void *q, int64_t q_ld, float *scale, void *stream) {
    Y3_REQUIRE(dtype == Y3_F32 || dtype == Y3_BF16 || dtype == Y3_I8, Y3_E_INVALID, "quantize_rows_i8: dtype %d", dtype);
    Y3_REQUIRE(k >= 1 && k <= MAX_K, Y3_E_INVALID, "quantize_rows_i8: k = %d outside 1 .. %d", k, MAX_K);
    Y3_REQUIRE(rows >= 0 && rows <= (1ll << 40) / k, Y3_E_INVALID, "quantize_rows_i8: %lld rows", (long long)rows);
    Y3_REQUIRE(x_ld >= k && (rows == 0 || (x_ld <= (1ll << 44) / rows && q_ld <= (1ll << 44) / rows)), Y3_E_INVALID, "quantize_rows_i8: k %d, x_ld %lld, q_ld %lld", k, (long long)x_ld, (long long)q_ld);
    Y3_REQUIRE(q_ld >= round_up(k, 16) && q_ld % 16 == 0, Y3_E_ALIGN, "quantize_rows_i8: q_ld %lld must be a multiple of 16 that holds k", (long long)q_ld);
    if (rows == 0) return Y3_OK;
    Y3_REQUIRE(x && q && (scale || dtype == Y3_I8), Y3_E_INVALID, "quantize_rows_i8: null pointer");
    Y3_REQUIRE((uintptr_t)x % es_of(dtype) == 0 && aligned16(q) && (uintptr_t)scale % 4 == 0, Y3_E_ALIGN, "quantize_rows_i8: pointer not aligned");
    Y3_REQUIRE(!overlap(x, ((rows - 1) * x_ld + k) * es_of(dtype), q, rows * q_ld), Y3_E_INVALID, "quantize_rows_i8: x and q overlap");
    Y3_REQUIRE(dtype == Y3_I8 || !(block_overlaps_rows(scale, rows * 4, x, x_ld * es_of(dtype), (long)k * es_of(dtype), rows) ||
                                   block_overlaps_rows(scale, rows * 4, q, q_ld, round_up(k, 16), rows)), Y3_E_INVALID, "quantize_rows_i8: scale overlaps x or q");
    const hipStream_t st = (hipStream_t)stream;
    const int fill = (int)round_up(k, 16);
    if (dtype == Y3_I8) hipLaunchKernelGGL(repitch_rows_kernel, dim3(rows_grid((rows + 3) / 4)), dim3(256), 0, st, (const char *)x, (long)x_ld, (long)rows, k, (char *)q, (long)q_ld, fill);
    else quantize_to(dtype, x, rows, k, x_ld, q, q_ld, fill, scale, st);
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
    Y3_REQUIRE(w_ld >= d->k && w_ld <= (1ll << 44) / d->n, Y3_E_INVALID, "linear_i8_pack: %d channels of k = %d on w_ld %lld", d->n, d->k, (long long)w_ld);
    Y3_REQUIRE(w && packed && (scale || w_dtype == Y3_I8), Y3_E_INVALID, "linear_i8_pack: null pointer");
    Y3_REQUIRE((uintptr_t)w % es_of(w_dtype) == 0 && aligned16(packed) && (uintptr_t)scale % 4 == 0, Y3_E_ALIGN, "linear_i8_pack: pointer not aligned");
    const long es = es_of(w_dtype), packed_bytes = (long)d->k_pad * d->n_pad;
    Y3_REQUIRE(!block_overlaps_rows(packed, packed_bytes, w, w_ld * es, d->k * es, d->n) &&
               (w_dtype == Y3_I8 || !(block_overlaps_rows(scale, d->n * 4l, w, w_ld * es, d->k * es, d->n) || overlap(scale, d->n * 4l, packed, packed_bytes))), Y3_E_INVALID,
               "linear_i8_pack: packed, scale and w overlap");
    const hipStream_t st = (hipStream_t)stream;
    const int kb = d->k_pad / 64;
    if (w_dtype == Y3_I8) {
        const long chunks = (long)d->n_pad / 16 * kb * 64;
        hipLaunchKernelGGL(pack_i8_kernel, dim3(rows_grid((chunks + 255) / 256)), dim3(256), 0, st, (const char *)w, (long)w_ld, d->n, d->k, kb, chunks, (char *)packed);
    } else if (w_dtype == Y3_BF16) hipLaunchKernelGGL(pack_float_kernel<Y3_BF16>, dim3(rows_grid(d->n_pad)), dim3(256), 0, st, (const char *)w, (long)w_ld, d->n, d->n_pad, d->k, kb, (char *)packed, scale);
    else hipLaunchKernelGGL(pack_float_kernel<Y3_F32>, dim3(rows_grid(d->n_pad)), dim3(256), 0, st, (const char *)w, (long)w_ld, d->n, d->n_pad, d->k, kb, (char *)packed, scale);
    return y3_check_launch("linear_i8_pack");
}

extern "C" int y3_linear_i8_workspace_bytes(const y3_linear_i8_desc *d, int64_t *bytes) {
    const int rc = check_desc(d);
    if (rc) return rc;
    Y3_REQUIRE(bytes, Y3_E_INVALID, "linear_i8: null pointer");
    *bytes = d->dtype == Y3_I8 || fused(d) ? 0 : round_up(d->rows * d->k_pad, 256) + round_up(d->rows * 4, 256);
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
    Y3_REQUIRE((uintptr_t)x % es_of(d->dtype) == 0 && aligned16(w) && (uintptr_t)out % es_of(d->out_dtype) == 0 && aligned16(workspace) &&
               (uintptr_t)x_scale % 4 == 0 && (uintptr_t)w_scale % 4 == 0 && (uintptr_t)bias % 4 == 0, Y3_E_ALIGN, "linear_i8: pointer not aligned");
    const int xs = es_of(d->dtype), os = es_of(d->out_dtype);
    Y3_REQUIRE(!rows_overlap(x, d->x_ld * xs, (long)d->k * xs, out, d->out_ld * os, (long)d->n * os, d->rows),
               Y3_E_INVALID, "linear_i8: x and out overlap");
    Y3_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), Y3_E_INVALID, "linear_i8: workspace of %lld bytes, needs %lld", (long long)workspace_bytes, (long long)need);
    const struct { const void *p; long bytes; } read[4] = {{w, (long)d->k_pad * d->n_pad}, {w_scale, d->n * 4l}, {bias, bias ? d->n * 4l : 0}, {x_scale, x_scale ? d->rows * 4 : 0}};
    for (const auto &r : read) {
        Y3_REQUIRE(!block_overlaps_rows(r.p, r.bytes, out, d->out_ld * os, (long)d->n * os, d->rows), Y3_E_INVALID, "linear_i8: out overlaps the weights, the scales or the bias");
        Y3_REQUIRE(need == 0 || r.bytes == 0 || !overlap(r.p, r.bytes, workspace, need), Y3_E_INVALID, "linear_i8: the workspace overlaps the weights, the scales or the bias");
    }
    Y3_REQUIRE(need == 0 || !(block_overlaps_rows(workspace, need, x, d->x_ld * xs, (long)d->k * xs, d->rows) || block_overlaps_rows(workspace, need, out, d->out_ld * os, (long)d->n * os, d->rows)),
               Y3_E_INVALID, "linear_i8: the workspace overlaps x or out");
    const hipStream_t st = (hipStream_t)stream;
    LinArgs a;
    a.x = (const char *)x; a.x_scale = x_scale; a.x_ld = d->x_ld; a.k16 = (int)round_up(d->k, 16);
    if (need) {
        float *s = (float *)((char *)workspace + round_up(d->rows * d->k_pad, 256));
        quantize_to(d->dtype, x, d->rows, d->k, d->x_ld, workspace, d->k_pad, d->k_pad, s, st);
        rc = y3_check_launch("linear_i8 (rows)");
        if (rc) return rc;
        a.x = (const char *)workspace; a.x_scale = s; a.x_ld = d->k_pad; a.k16 = d->k_pad;
    }
    const long cus = y3_device_cus();
    a.w = (const char *)w; a.w_scale = w_scale; a.bias = bias; a.out = (char *)out;
    a.rows = d->rows; a.out_ld = d->out_ld; a.n = d->n; a.k = d->k; a.kb = d->k_pad / 64;
    a.slope = d->flags & Y3_CONV_LEAKY ? 0.1f : 1.0f; a.out_f32 = d->out_dtype == Y3_F32;
    a.flat = d->out_ld == d->n && (long)d->n * os % 16 != 0 && aligned16(out);
    if (d->dtype != Y3_I8 && need == 0) {
        const Panel c = panel_of(d->rows, d->n, a.kb, d->dtype, cus);
        return d->dtype == Y3_BF16 ? launch_float<Y3_BF16>(a, c, cus, st) : launch_float<Y3_F32>(a, c, cus, st);
    }
    if (!rows_aligned(a)) return launch_panel<I8_ANY>(a, panel_of(d->rows, d->n, a.kb, I8_ANY, cus), st);
    if (y3_linear_i8_tile_ok(a, cus)) return y3_linear_i8_tile_launch(a, cus, st);
    return launch_panel<Y3_I8>(a, panel_of(d->rows, d->n, a.kb, Y3_I8, cus), st);
}
