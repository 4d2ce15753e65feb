// Log probabilities of given classes, entropy and the top alternatives of rows of logits, for gfx950 (MI355X): y3_log_probs.
//
//   M = max z    Z = sum exp(z - M)    S = sum exp(z - M) (z - M)    log p_c = (z_c - M) - log Z    H = log Z - S / Z
// Z >= 1 and S <= 0, so the entropy is a sum of two terms that are not negative: nothing cancels.  Everything is fp32.
// The alternatives are the largest 64-bit keys {order of the logit, ~class}: a total order, so ties go to the lowest class
// and no order of arrival shows in the result.
#include "common.h"
#include <type_traits>

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr int MAX_TOP = 32;

struct ProbsArgs {
    const char *z;
    const int64_t *row_offsets;
    const void *ids;
    float *logp, *entropy, *top_logp;
    int32_t *top_ids;
    long rows, group_ld, row_ld, extent, first;
    int classes, group, top, ids_64, fast_group, chunks, chunk_vecs, chunk_more;
    f32x4 *sums;                       // rows of several chunks: {M, Z, S, the id's logit or 0} and `top` keys per chunk
    unsigned long long *keys;
    FastDiv fd_group;                  // r / group where fast_group is set (more than one row per group, fewer than 2^31 rows)
};

template <int DT> __device__ __forceinline__ float logit(const char *z, long i) {
    if constexpr (DT == Y3_F32) return ((const float *)z)[i];
    else return bf16_to_f32(((const unsigned short *)z)[i]);
}

// element offset of a row; -1: skip it, -2: it does not lie within the extent
__device__ __forceinline__ long row_start(const ProbsArgs &p, long r) {
    if (!p.row_offsets) {
        if (p.group == 1) return r * p.group_ld;
        const long g = p.fast_group ? fast_div((int)r, p.fd_group) : r / p.group;
        return g * p.group_ld + (r - g * p.group) * p.row_ld;
    }
    const long o = p.row_offsets[r];
    return o < 0 ? -1 : o > p.extent - p.classes ? -2 : o;
}

__device__ __forceinline__ long row_id(const ProbsArgs &p, long r) {
    return p.ids_64 ? (long)((const int64_t *)p.ids)[r] : (long)((const int32_t *)p.ids)[r];
}

// unsigned order of the floats, NaN above +inf, both zeros alike
__device__ __forceinline__ unsigned order_of(float x) {
    unsigned u = __float_as_uint(x + 0.0f);
    if (x != x) u = 0x7fc00000u;
    return (int)u < 0 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_order(unsigned o) { return __uint_as_float((int)o < 0 ? o & 0x7fffffffu : ~o); }

// log p of a logit, given the row's maximum and log Z (a row of only -inf: everything is -inf; of only NaN: log Z is NaN)
__device__ __forceinline__ float log_prob(float z, float m, float log_z) {
    return m == -__builtin_inff() ? m + log_z : (z - m) - log_z;
}

__device__ __forceinline__ void put_row_outside(const ProbsArgs &p, long r, int lane, int lanes) {
    if (lane == 0) {
        if (p.logp) p.logp[r] = __builtin_nanf("");
        if (p.entropy) p.entropy[r] = __builtin_nanf("");
    }
    for (int j = lane; j < p.top; j += lanes) { p.top_ids[r * p.top + j] = -1; p.top_logp[r * p.top + j] = __builtin_nanf(""); }
}

__device__ __forceinline__ void put_scalars(const ProbsArgs &p, long r, float id_logit, long id, float m, float log_z, float entropy) {
    if (p.logp) p.logp[r] = id < 0 ? 0.0f : id >= p.classes ? __builtin_nanf("") : log_prob(id_logit, m, log_z);
    if (p.entropy) p.entropy[r] = entropy;
}

// Reductions over the L lanes of a row: DPP within 16 lanes (quad_perm xor 1, xor 2, then the mirrors: once the lanes below
// agree, a mirrored lane is as good as the one across), shuffles above.
template <int L, typename T, typename F> __device__ __forceinline__ T lanes_reduce(T v, F f) {
    const auto dpp = [](T x, auto c) { return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(c)::value, 0xf, 0xf, false)); };
    if constexpr (L >= 2) v = f(v, dpp(v, std::integral_constant<int, 0xB1>{}));
    if constexpr (L >= 4) v = f(v, dpp(v, std::integral_constant<int, 0x4E>{}));
    if constexpr (L >= 8) v = f(v, dpp(v, std::integral_constant<int, 0x141>{}));
    if constexpr (L >= 16) v = f(v, dpp(v, std::integral_constant<int, 0x140>{}));
    if constexpr (L >= 32) v = f(v, __shfl_xor(v, 16));
    if constexpr (L >= 64) v = f(v, __shfl_xor(v, 32));
    return v;
}

struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return vmax_raw(a, b); } };      // (NaN: the other one)
struct Add { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct MaxU { __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return max(a, b); } };
struct MinU { __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return min(a, b); } };
struct MinI { __device__ __forceinline__ int operator()(int a, int b) const { return min(a, b); } };

// ---- few classes: L lanes per row, E logits in each lane's registers --------------------------------------------------
// One read of the row.  The alternatives come from 31-bit keys in ascending order, {how far the logit is below the maximum,
// class}: fp32 takes the bits of the difference, which the softmax has computed anyway, bf16 the 16 bits of the logit itself.
// With the previous winner + 1 subtracted, every key that is left keeps its order and the ones taken wrap to the upper half,
// so a round is one subtraction and half a v_min3_u32 per logit (finding the maximum and its class and taking it out costs
// four times as much: 1.1 M rows of 80, three alternatives, 188 us that way).  bf16 keys are exact.  fp32 keys that agree in
// all but the class leave open which logit is larger: one more round shows whether any of the first `top` + 1 do, and the
// wave then settles its rows with whole logits.  Bound by memory: those 1.1 M rows of 80 fp32 91 us, 4.3 TB/s.
template <int DT, int L, int E>
__global__ __launch_bounds__(256) void probs_lanes_kernel(const ProbsArgs p) {
    constexpr int RPW = 64 / L, SURE = E - 2;                    // the first SURE logits of every lane exist (launch_probs)
    constexpr unsigned MASK = L * E <= 128 ? 127 : L * E <= 256 ? 255 : L * E <= 512 ? 511 : 1023;
    const int lane = threadIdx.x & 63, l = lane & (L - 1);
    const float nan = __builtin_nanf(""), ninf = -__builtin_inff();
    const long r = p.first + ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * RPW + lane / L;
    const long at = r < p.rows ? row_start(p, r) : -1;
    if (at < 0) {                                               // (the lanes of a row go together)
        if (at == -2) put_row_outside(p, r, l, L);
        return;
    }
    const char *z = p.z + at * (DT == Y3_F32 ? 4 : 2);
    float x[E];
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = logit<DT>(z, j < SURE ? j * L + l : min(j * L + l, p.classes - 1));
    long id = -1;
    float zid = 0.0f;
    if (p.logp) {
        id = row_id(p, r);
        if (id >= 0 && id < p.classes) zid = logit<DT>(z, id);
    }
#pragma unroll
    for (int j = SURE; j < E; ++j) x[j] = j * L + l < p.classes ? x[j] : ninf;
    float m = x[0];
#pragma unroll
    for (int j = 1; j < E; ++j) m = vmax_raw(m, x[j]);
    m = lanes_reduce<L>(m, Max());
    const float m0 = m == ninf ? 0.0f : m;
    float zs = 0.0f, ss = 0.0f;
    unsigned k[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const float d = x[j] - m0, e = __builtin_amdgcn_exp2f(d * LOG2E);
        zs += e;
        ss = fmaf(e, vmax_raw(d, -1e4f), ss);               // (an e of 0 adds nothing, whatever d is)
        if constexpr (DT == Y3_F32) {
            k[j] = (__float_as_uint(d) & (0x7fffffffu & ~MASK)) | (unsigned)(j * L + l);
        } else {
            const unsigned u = __float_as_uint(x[j] + 0.0f);            // (one zero)
            k[j] = ((((u ^ ~(unsigned)((int)u >> 31)) & 0x7fffffffu) ^ (u & 0x80000000u)) >> 1 & ~MASK) | (unsigned)(j * L + l);
        }
    }
    zs = lanes_reduce<L>(zs, Add());
    ss = lanes_reduce<L>(ss, Add());
    const bool none = zs == 0.0f, bad = !(zs < __builtin_inff());
    const float log_z = none ? 0.0f : __builtin_amdgcn_logf(zs) * LN2;
    if (l == 0) put_scalars(p, r, zid, id, m, log_z, none ? 0.0f : fmaf(-ss, __builtin_amdgcn_rcpf(zs), log_z));
    if (!p.top) return;
    const auto put = [&](int t, int c) {                     // alternative t of the row, by one of its lanes
        p.top_ids[r * p.top + t] = bad ? t : c;
        p.top_logp[r * p.top + t] = bad ? nan : log_prob(logit<DT>(z, c), m, log_z);
    };
    unsigned past = 0, open = 0;                             // the last winner + 1
    int mine = 0;
    const int rounds = DT == Y3_F32 ? min(p.top + 1, p.classes) : p.top;
    for (int t = 0; t < rounds; ++t) {
        unsigned d = ~0u;
#pragma unroll
        for (int j = 0; j < E; ++j) d = min(d, k[j] - past);
        d = lanes_reduce<L>(d, MinU());
        const unsigned next = past + d;
        open |= (unsigned)(t > 0 && (next ^ (past - 1)) <= MASK);
        past = next + 1;
        const int c = min((int)(next & MASK), p.classes - 1);               // (NaN rows: any class, not used)
        if (l == (t & (L - 1))) mine = c;                    // lane t keeps alternative t: rows are stored in one piece
        if ((t & (L - 1)) == L - 1 || t == rounds - 1) {
            const int first = t & ~(L - 1);
            if (first + l < min(t + 1, p.top)) put(first + l, mine);
        }
    }
    if (DT == Y3_F32 && __ballot(open)) {                    // whole logits: the maximum, the lowest class that has it, ...
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = j * L + l < p.classes ? logit<DT>(z, j * L + l) : nan;
        for (int t = 0; t < p.top; ++t) {
            float v = x[0];
#pragma unroll
            for (int j = 1; j < E; ++j) v = vmax_raw(v, x[j]);
            v = lanes_reduce<L>(v, Max());
            int c = 0x7fffffff;
#pragma unroll
            for (int j = E - 1; j >= 0; --j) c = x[j] == v ? j * L + l : c;
            c = lanes_reduce<L>(c, MinI());
#pragma unroll
            for (int j = 0; j < E; ++j) x[j] = c == j * L + l ? nan : x[j];         // ... and that one taken out
            if (l == 0) put(t, min(c, p.classes - 1));
        }
    }
}

// ---- many classes: rows in chunks of up to 8192 logits, one workgroup of four waves per chunk ---------------------------
// A chunk is read once, in 16-byte vectors at whatever address the row starts (the last one moved into place), into
// registers, and everything is done there: the thread's maximum, its sums, and the candidates for the alternatives.  For
// those, the top-th largest of 64 groups' maxima (found by bisection of its upper bits, one ballot each) is a bound that at
// least `top` logits reach and few others do: those are listed, and ranked by counting the larger keys.  A list that
// overflows (hundreds of equal logits at the border) is settled by one search per alternative.  A row of up to 2048 (4096)
// logits is one wave's (two waves'): 20000 rows of 2000 bf16 29 us, by four waves 91.
// Rows of more than one chunk leave {M, Z, S}, the id's logit and the chunk's first `top` keys in the workspace for
// probs_join_kernel, which merges them in a fixed order.  One workgroup walking a whole row instead: 31 us for one row of
// 128000 (its exponentials alone keep one CU busy for 9 us), 98 us for 4096 rows of 32001; chunks of 4096 or 2048 logits:
// 75 and 87 us for the latter against 72.
//   Bound by vector issue (70 % busy) and memory: 4096 rows of 32001 bf16, 262 MB, 73 us with the join (of 32000 68);
//   vectors from the row's first 16-byte border on, its ends one by one: 78.  One row of 128000: 7 us and 6, all of it latency.
constexpr int LIST = 512, CHUNK_THREADS = 256;

typedef unsigned long long u64;
__device__ __forceinline__ u64 key_of(float x, int c) { return (u64)order_of(x) << 32 | (0xffffffffu - (unsigned)c); }

// Over a whole wave, all lanes active: within 16 lanes as lanes_reduce, then row 0 into 1, 2 into 3, and 1 into 2 and 3; the
// last lane's value in every lane.  (`none`: what changes nothing.)
template <typename T, typename F> __device__ __forceinline__ T wave_reduce(T v, T none, F f) {
    v = lanes_reduce<16>(v, f);
    const int n = __builtin_bit_cast(int, none);
    v = f(v, __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(n, __builtin_bit_cast(int, v), 0x142, 0xa, 0xf, false)));
    v = f(v, __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(n, __builtin_bit_cast(int, v), 0x143, 0xc, 0xf, false)));
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ u64 wave_max_u64(u64 v) {
    const unsigned hi = wave_reduce((unsigned)(v >> 32), 0u, MaxU());
    const unsigned lo = wave_reduce((unsigned)(v >> 32) == hi ? (unsigned)v : 0u, 0u, MaxU());
    return (u64)hi << 32 | lo;
}

struct Sums { float m, z, s; };
// scaled to another maximum that is not below (both -inf: the difference is NaN, the factor 0, Z = S = 0)
__device__ __forceinline__ Sums scaled(Sums a, float m) {
    const float d = vmax_raw(a.m - m, -1e4f), f = __builtin_amdgcn_exp2f(d * LOG2E);
    return Sums{m, a.z * f, f * fmaf(d, a.z, a.s)};
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
    const float m = vmax_raw(a.m, b.m);
    a = scaled(a, m);
    b = scaled(b, m);
    return Sums{m, a.z + b.z, a.s + b.s};
}
__device__ __forceinline__ Sums wave_join(Sums a) {
    a = scaled(a, wave_reduce(a.m, -__builtin_inff(), Max()));
    return Sums{a.m, wave_reduce(a.z, 0.0f, Add()), wave_reduce(a.s, 0.0f, Add())};
}

struct Row { float m, log_z, entropy; bool bad; };
__device__ __forceinline__ Row finish(Sums s) {
    const bool none = s.z == 0.0f;
    const float log_z = none ? 0.0f : __builtin_amdgcn_logf(s.z) * LN2;
    return Row{s.m, log_z, none ? 0.0f : fmaf(-s.s, __builtin_amdgcn_rcpf(s.z), log_z), !(s.z < __builtin_inff())};
}
__device__ __forceinline__ void put_alternative(const ProbsArgs &p, long r, int t, u64 k, const Row &w) {
    p.top_ids[r * p.top + t] = w.bad ? t : (int)(0xffffffffu - (unsigned)k);
    p.top_logp[r * p.top + t] = w.bad ? __builtin_nanf("") : log_prob(of_order((unsigned)(k >> 32)), w.m, w.log_z);
}
// place of a key among list[0 .. n), cleared up to the next multiple of 8
__device__ __forceinline__ int place_in(const u64 *list, int n, u64 k) {
    int rank = 0;
    for (int o = 0; o < n; o += 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) rank += list[o + i] > k;
    }
    return rank;
}

template <int DT, int STEP>
__global__ __launch_bounds__(STEP) __attribute__((amdgpu_waves_per_eu(8))) void probs_chunk_kernel(const ProbsArgs p) {
    constexpr int VE = DT == Y3_F32 ? 4 : 8, ES = DT == Y3_F32 ? 4 : 2, NV = 32 / VE, W = STEP / 64, GROUP = STEP / 64;         // GROUP lanes have one maximum
    __shared__ __attribute__((aligned(16))) u64 list[LIST];
    __shared__ u64 red[W];
    __shared__ float part[W][3], groups[STEP / GROUP], bound_s;
    __shared__ int list_n;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float ninf = -__builtin_inff();
    const long i = p.first + blockIdx.x;                         // (no loop: what it hoists costs a third of the registers)
    const long r = p.chunks == 1 ? i : i / p.chunks;
    const int chunk = (int)(i - r * p.chunks);
    const long at = row_start(p, r);
    if (at < 0) {
        if (at == -2 && chunk == 0) put_row_outside(p, r, tid, STEP);
        return;
    }
    const char *z = p.z + at * ES;
    const int C = p.classes, top = p.top, whole = C / VE;
    const int v0 = chunk * p.chunk_vecs + min(chunk, p.chunk_more), vecs = p.chunk_vecs + (chunk < p.chunk_more);
    const int c0 = v0 * VE, c1 = min(C, (v0 + vecs) * VE);       // the chunk's classes
    const auto first_of = [&](int g) { return (v0 + tid + g * STEP) * VE; };
    // What a chunk does not fill holds -1e38: its exponential is 0 beside any logit above -1e37, and no NaN comes of it.
    constexpr unsigned FILL = DT == Y3_F32 ? 0xfe960000u : 0xfe96fe96u;
    u32x4 raw[NV];
#pragma unroll
    for (int g = 0; g < NV; ++g) {
        raw[g] = u32x4{FILL, FILL, FILL, FILL};
        const int w0 = wave * 64 + g * STEP;                     // (wave-uniform: all 64 vectors are there and whole)
        if (w0 + 63 < vecs && v0 + w0 + 63 < whole) __builtin_memcpy(&raw[g], z + (long)(v0 + w0) * 16 + lane * 16, 16);
        else if (w0 < vecs && v0 + w0 <= whole) {
            const int u = v0 + tid + g * STEP;
            if (tid + g * STEP < vecs && u <= whole && u * VE < C) {
                __builtin_memcpy(&raw[g], z + (long)min(u * VE, C - VE) * ES, 16);
                if (u == whole) {                                // the row's last logits, moved to the front
                    const int drop = (VE - (C - whole * VE)) * ES;
                    u64 lo = (u64)raw[g][1] << 32 | raw[g][0], hi = (u64)raw[g][3] << 32 | raw[g][2];
                    const u64 fill = (u64)FILL << 32 | FILL;
                    if (drop >= 8) { lo = hi; hi = fill; }
                    const int bits = drop % 8 * 8;
                    if (bits) {
                        lo = lo >> bits | hi << (64 - bits);
                        hi = hi >> bits | fill << (64 - bits);
                    }
                    raw[g] = u32x4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
                }
            }
        }
    }
    long id = -1;
    float zid = 0.0f;
    if (tid == (p.chunks == 1 ? 0 : STEP - 64)) {                // (by the wave that writes it; of several chunks the one that has it)
        if (p.logp) {
            id = row_id(p, r);
            if (id >= c0 && id < c1) zid = logit<DT>(z, id);
        }
    }
    if (tid == 0) list_n = 0;
    if (top)
#pragma unroll
        for (int q = tid; q < LIST / 2; q += STEP) *(u32x4 *)(list + 2 * q) = u32x4{0, 0, 0, 0};
    const auto value = [&](int g, int j) {
        if constexpr (DT == Y3_F32) return __uint_as_float(raw[g][j]);
        else return __uint_as_float(j % 2 ? raw[g][j / 2] & 0xffff0000u : raw[g][j / 2] << 16);
    };
    const auto unseen = [&]() {                              // (bf16 is unpacked again where it is used: half the registers)
#pragma unroll
        for (int g = 0; g < NV; ++g) asm volatile("" : "+v"(raw[g]));
    };
    float vmax[NV], big = ninf;
#pragma unroll
    for (int g = 0; g < NV; ++g) {
        vmax[g] = value(g, 0);
#pragma unroll
        for (int j = 1; j < VE; ++j) vmax[g] = vmax_raw(vmax[g], value(g, j));
        big = vmax_raw(big, vmax[g]);
    }
    // exp(x - M) as exp2(x log2 e - fl(M log2 e)), one fused operation: the rounding r of M log2 e is in every exponent
    // alike and comes out of the sums behind the loop.  |r| <= 64 keeps every sum (32 terms of at most 2^64 * 64) and the
    // factor 2^-r normal numbers; from |M| = 7e8 on r can be larger.  Magnitudes whose product overflows have no such form,
    // and 0 * -inf makes S a NaN where there are impossible classes: such waves, and those with lanes that got nothing or
    // only logits below -1e37, do it the long way.
    Sums s = {big, 0.0f, 0.0f};
    const float ml = big * LOG2E;
    unseen();
#pragma unroll
    for (int g = 0; g < NV; ++g)
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const float y = fmaf(value(g, j), LOG2E, -ml), e = __builtin_amdgcn_exp2f(y);
            s.z += e;
            s.s = fmaf(e, y, s.s);
        }
    const float off = fmaf(big, LOG2E, -ml);                     // r
    {
        s.s = fmaf(-off, s.z, s.s) * LN2;
        const float f = __builtin_amdgcn_exp2f(-off);
        s.z *= f;
        s.s *= f;
    }
    if (__ballot(!(fabsf(big) < 1e37f) || !(fabsf(off) <= 64.0f) || s.s != s.s)) {
        const auto real = [&](int g, int j) {
            const int c = first_of(g) + j;
            return c >= c0 && c < c1 && tid + g * STEP < vecs ? value(g, j) : ninf;
        };
        unseen();
        big = ninf;
#pragma unroll
        for (int g = 0; g < NV; ++g)
#pragma unroll
            for (int j = 0; j < VE; ++j) big = vmax_raw(big, real(g, j));
        const float m0 = big == ninf ? 0.0f : big;
        unseen();
        s = Sums{big, 0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < NV; ++g)
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const float y = real(g, j) - m0, e = __builtin_amdgcn_exp2f(y * LOG2E);
                s.z += e;
                s.s = fmaf(e, vmax_raw(y, -1e4f), s.s);          // (an e of 0 adds nothing, whatever y is)
            }
    }
    s = wave_join(s);
    const float group = lanes_reduce<GROUP>(big, Max());
    if (lane == 0) { part[wave][0] = s.m; part[wave][1] = s.z; part[wave][2] = s.s; }
    if (lane % GROUP == 0) groups[tid / GROUP] = group;
    __syncthreads();
    Row row = {0.0f, 0.0f, 0.0f, false};
    if (wave == 0) {
        if (top) {                                               // (the lowest bits left at 0: a bound a little below)
            constexpr int BOUND_BITS = DT == Y3_F32 ? 8 : 16;
            unsigned t = 0;
            const unsigned o = order_of(groups[lane]);
#pragma unroll
            for (int b = 31; b >= BOUND_BITS; --b) {
                const unsigned more = t | 1u << b;
                t = __popcll(__ballot(o >= more)) >= top ? more : t;
            }
            if (lane == 0) bound_s = of_order(max(t, 0x007fffffu));     // (-inf: below it there are only NaN's patterns)
        }
    }
    if (wave == (p.chunks == 1 ? 0 : W - 1)) {                   // (the first wave writes a whole row's alternatives: it needs these)
        s = Sums{part[0][0], part[0][1], part[0][2]};
#pragma unroll
        for (int w = 1; w < W; ++w) s = join(s, Sums{part[w][0], part[w][1], part[w][2]});
        if (p.chunks == 1) {
            row = finish(s);
            if (tid == 0) put_scalars(p, r, zid, id, row.m, row.log_z, row.entropy);
        } else if (lane == 0) p.sums[i] = f32x4{s.m, s.z, s.s, zid};
    }
    if (top) {
        __syncthreads();
        const float bound = bound_s;
        if (bound < -1e37f) {
            // from memory, where nothing is filled up; of impossible classes the chunk's first are enough (that is when
            // fewer than `top` groups have a possible one)
            for (int c = c0 + tid; c < c1; c += STEP) {
                const float x = logit<DT>(z, c);
                if (x >= bound && (x != ninf || c < c0 + top)) {
                    const int to = atomicAdd(&list_n, 1);    // (the order of the list does not show)
                    if (to < LIST) list[to] = key_of(x, c);
                }
            }
        } else if (big >= bound) {
            unseen();
#pragma unroll
            for (int g = 0; g < NV; ++g)
                if (vmax[g] >= bound) {
                    int many = 0;
#pragma unroll
                    for (int j = 0; j < VE; ++j) many += value(g, j) >= bound;
                    int to = atomicAdd(&list_n, many);
#pragma unroll
                    for (int j = 0; j < VE; ++j)
                        if (value(g, j) >= bound) {
                            if (to < LIST) list[to] = key_of(value(g, j), first_of(g) + j);
                            ++to;
                        }
                }
        }
        __syncthreads();
        const int n = list_n;
        const auto put = [&](int t, u64 k) {                 // (by the first wave: it has the row's sums)
            if (p.chunks == 1) put_alternative(p, r, t, k, row);
            else p.keys[i * top + t] = k;
        };
        if (n <= LIST) {
            if (wave == 0) {
                if (row.bad) {
                    if (lane < top) put(lane, 0);
                } else {
                    for (int q = lane; q < n; q += 64) {
                        const u64 k = list[q];
                        const int rank = n == 1 ? 0 : place_in(list, n, k);
                        if (rank < top) put(rank, k);
                    }
                    for (int q = n + lane; q < top; q += 64) put(q, 0);        // (NaN in a chunk of several: fewer keys)
                }
            }
        } else {
            u64 last = ~0ull;
            for (int t = 0; t < top; ++t) {
                u64 best = 0;
                for (int c = c0 + tid; c < c1; c += STEP) {
                    const u64 k = key_of(logit<DT>(z, c), c);
                    if (k < last && k > best) best = k;
                }
                best = wave_max_u64(best);
                if (lane == 0) red[wave] = best;
                __syncthreads();
                last = red[0];
#pragma unroll
                for (int w = 1; w < W; ++w) last = red[w] > last ? red[w] : last;
                __syncthreads();
                if (tid == 0) put(t, last);
            }
        }
    }
}

// One workgroup per row: the chunks' sums in order; their keys from the largest `top`-th one on, ranked by counting.
template <int DT>
__global__ __launch_bounds__(CHUNK_THREADS) void probs_join_kernel(const ProbsArgs p) {
    __shared__ __attribute__((aligned(16))) u64 list[LIST];
    __shared__ u64 red[CHUNK_THREADS / 64];
    __shared__ int list_n;
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, wave = tid >> 6, waves = threads / 64;
    for (long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const long at = row_start(p, r);
        if (at < 0) continue;
        const int top = p.top, n_keys = p.chunks * top;
        const u64 *keys = p.keys + r * n_keys;
        u64 bound = 0;                                           // `top` keys of one chunk reach its last one
        if (top)
            for (int c = lane; c < p.chunks; c += 64) {
                const u64 k = keys[c * top + top - 1];
                bound = k > bound ? k : bound;
            }
        Sums s = {-__builtin_inff(), 0.0f, 0.0f};
        float zid = 0.0f;
        for (int c = lane; c < p.chunks; c += 64) {
            const f32x4 v = p.sums[r * p.chunks + c];
            s = join(s, Sums{v[0], v[1], v[2]});
            zid += v[3];                                         // (the id's logit in one chunk, 0 in the others)
        }
        constexpr int AHEAD = 4;                                 // keys of this thread, requested before they are needed
        u64 mine[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) mine[j] = tid + j * threads < n_keys ? keys[tid + j * threads] : 0;
        long id = -1;
        if (tid == 0) {
            list_n = 0;
            if (p.logp) id = row_id(p, r);
        }
        if (top)
            for (int q = tid; q < LIST / 2; q += threads) *(u32x4 *)(list + 2 * q) = u32x4{0, 0, 0, 0};
        const Row row = finish(wave_join(s));
        zid = wave_reduce(zid, 0.0f, Add());
        if (tid == 0) put_scalars(p, r, zid, id, row.m, row.log_z, row.entropy);
        if (top) {
            bound = wave_max_u64(bound);
            __syncthreads();
            if (row.bad) {
                if (tid < top) put_alternative(p, r, tid, 0, row);
            } else {
                const auto take = [&](u64 k) {
                    if (k != 0 && k >= bound) {
                        const int to = atomicAdd(&list_n, 1);
                        if (to < LIST) list[to] = k;
                    }
                };
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) take(mine[j]);
                for (int q = tid + AHEAD * threads; q < n_keys; q += threads) take(keys[q]);
                __syncthreads();
                const int n = list_n;
                if (n <= LIST) {
                    for (int q = tid; q < n; q += threads) {
                        const u64 k = list[q];
                        const int rank = place_in(list, n, k);
                        if (rank < top) put_alternative(p, r, rank, k, row);
                    }
                } else {
                    u64 last = ~0ull;
                    for (int t = 0; t < top; ++t) {
                        u64 best = 0;
                        for (int q = tid; q < n_keys; q += threads) {
                            const u64 k = keys[q];
                            if (k < last && k > best) best = k;
                        }
                        best = wave_max_u64(best);
                        if (lane == 0) red[wave] = best;
                        __syncthreads();
                        last = red[0];
                        for (int w = 1; w < waves; ++w) last = red[w] > last ? red[w] : last;
                        __syncthreads();
                        if (tid == 0) put_alternative(p, r, t, last, row);
                    }
                }
            }
        }
        __syncthreads();
    }
}

// Chunks of at most 32 logits per thread.  Whole rounds of the threads, so that only the
// last chunk has any that are not filled -- unless that one would be left with few: then all are equal but for one vector
// (29 rows of 41221, 20 alternatives, 34 vectors left: 33 us against 8.8).
// Up to 1024 classes are the lanes kernel's, but for many alternatives of many classes, whose rounds cost more than a list
// (20000 rows of 1000 fp32: 5 alternatives 23 us against 25, 20: 54, 31; of 500: 10: 21, 24, 32: 54, 32; 777 bf16: 10: 23,
// 25, 32: 46, 32), where every lane has a vector.
struct Chunks { int n, vecs, more; };
bool in_lanes(const y3_log_probs_desc *d) {
    const bool f32 = d->dtype == Y3_F32;
    return d->classes <= (f32 ? 256 : 512) || (d->classes <= 1024 && d->classes * d->top <= (f32 ? 6400 : 9000));
}
Chunks chunks_of(const y3_log_probs_desc *d) {
    if (in_lanes(d)) return Chunks{0, 0, 0};
    const int ve = d->dtype == Y3_F32 ? 4 : 8, most = CHUNK_THREADS * 32 / ve;
    const int vecs = (d->classes + ve - 1) / ve;
    const int n = (vecs + most - 1) / most, each = (int)(((vecs + n - 1) / n + CHUNK_THREADS - 1) / CHUNK_THREADS * CHUNK_THREADS);
    if (n == 1) return Chunks{1, vecs, 0};
    if (vecs - (n - 1) * each >= 2 * CHUNK_THREADS) return Chunks{n, each, 0};
    return Chunks{n, vecs / n, vecs % n};
}

template <int DT, int L, int E> void launch_lanes(const ProbsArgs &a, hipStream_t st) {
    constexpr long RPB = 4 * (64 / L), MOST = RPB << 23;         // rows of a block, of a grid (fewer than 2^32 threads)
    ProbsArgs b = a;
    for (b.first = 0; b.first < a.rows; b.first += MOST) {
        const long n = a.rows - b.first < MOST ? a.rows - b.first : MOST;
        hipLaunchKernelGGL((probs_lanes_kernel<DT, L, E>), dim3((unsigned)((n + RPB - 1) / RPB)), dim3(256), 0, st, b);
    }
}
// L lanes with E = 2, 4, .. logits each such that all but each lane's last two exist
template <int DT, int L, int E> void launch_even(const ProbsArgs &a, hipStream_t st) {
    if constexpr (E < 16)
        if (a.classes > L * E) return launch_even<DT, L, E + 2>(a, st);
    launch_lanes<DT, L, E>(a, st);
}
template <int DT> int launch_probs(const ProbsArgs &a, hipStream_t st) {
    const int C = a.classes;
    if (a.chunks == 0 && C <= 128) launch_even<DT, 8, 2>(a, st);
    else if (a.chunks == 0 && C <= 256) launch_even<DT, 16, 10>(a, st);
    else if (a.chunks == 0 && C <= 512) launch_even<DT, 32, 10>(a, st);
    else if (a.chunks == 0) launch_even<DT, 64, 10>(a, st);
    else {
        constexpr int VE = DT == Y3_F32 ? 4 : 8;
        ProbsArgs c = a;
        for (c.first = 0; c.first < a.rows * a.chunks; c.first += 1 << 23) {        // (a grid holds fewer than 2^32 threads)
            const long n = a.rows * a.chunks - c.first;
            const dim3 grid((unsigned)(n < (1 << 23) ? n : 1 << 23));
            const int vecs = a.chunk_vecs + (a.chunk_more > 0);
            if (vecs <= 64 * 32 / VE) hipLaunchKernelGGL((probs_chunk_kernel<DT, 64>), grid, dim3(64), 0, st, c);
            else if (vecs <= 128 * 32 / VE) hipLaunchKernelGGL((probs_chunk_kernel<DT, 128>), grid, dim3(128), 0, st, c);
            else hipLaunchKernelGGL((probs_chunk_kernel<DT, CHUNK_THREADS>), grid, dim3(CHUNK_THREADS), 0, st, c);
        }
        if (a.chunks == 1) return y3_check_launch("log_probs");
        const int rc = y3_check_launch("log_probs (chunks)");
        if (rc) return rc;
        // one wave where its lanes hold all keys twice over
        const int threads = a.chunks * a.top <= 128 ? 64 : CHUNK_THREADS;
        hipLaunchKernelGGL(probs_join_kernel<DT>, dim3((unsigned)(a.rows < (1 << 20) ? a.rows : 1 << 20)), dim3(threads), 0, st, a);
    }
    return y3_check_launch("log_probs");
}

// ---- kept boxes -> rows of logits: one workgroup per image ------------------------------------------------------------
constexpr int MAX_CLASSES = 96;        // y3_decode's
struct RowsArgs {
    y3_decode_desc d;
    const int32_t *kept_idx, *kept_count;
    int64_t *row_offsets;
    int32_t *row_classes;
    int max_boxes;
};
__global__ __launch_bounds__(256) void detection_rows_kernel(const RowsArgs p) {
    __shared__ int before[MAX_CLASSES + 1];                      // rows of the classes below
    const int b = blockIdx.x, C = p.d.num_classes, K = p.max_boxes, cap = C * K;
    if (threadIdx.x == 0) {
        int n = 0;
        for (int c = 0; c < C; ++c) {
            before[c] = n;
            n += min(max(p.kept_count[b * C + c], 0), K);
        }
        before[C] = n;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < cap; i += 256) {
        const int c = i / K, k = i - c * K;
        if (k < before[c + 1] - before[c]) {
            const int r = before[c] + k, box = p.kept_idx[((long)b * C + c) * K + k];
            int base = 0;
            for (int l = 0; l < p.d.num_scales; ++l) {
                const int n = p.d.grid_h[l] * p.d.grid_w[l] * p.d.num_anchors, at = box - base;
                long off = -1;
                if (at >= 0 && at < n)
                    off = ((long)b * p.d.grid_h[l] * p.d.grid_w[l] + at / p.d.num_anchors) * p.d.head_ld[l] + at % p.d.num_anchors * (5 + C) + 5;
                p.row_offsets[((long)l * p.d.batch + b) * cap + r] = off;
                base += n;
            }
            p.row_classes[(long)b * cap + r] = c;
        }
        if (i >= before[C]) {                                    // rows behind the last
            for (int l = 0; l < p.d.num_scales; ++l) p.row_offsets[((long)l * p.d.batch + b) * cap + i] = -1;
            p.row_classes[(long)b * cap + i] = -1;
        }
    }
}

int check_desc(const y3_log_probs_desc *d) {
    Y3_REQUIRE(d, Y3_E_INVALID, "log_probs: null descriptor");
    Y3_REQUIRE(d->dtype == Y3_F32 || d->dtype == Y3_BF16, Y3_E_INVALID, "log_probs: dtype %d", d->dtype);
    Y3_REQUIRE(d->classes >= 1 && d->classes <= (1 << 24), Y3_E_INVALID, "log_probs: %d classes", d->classes);
    Y3_REQUIRE(d->rows >= 0 && d->rows <= (1ll << 40), Y3_E_INVALID, "log_probs: %lld rows", (long long)d->rows);
    Y3_REQUIRE(d->top >= 0 && d->top <= MAX_TOP && d->top <= d->classes, Y3_E_INVALID, "log_probs: top = %d of %d classes (at most %d)", d->top, d->classes, MAX_TOP);
    Y3_REQUIRE(d->extent >= 0 && d->extent <= (1ll << 42), Y3_E_INVALID, "log_probs: extent %lld", (long long)d->extent);
    return Y3_OK;
}

}  // namespace

extern "C" int y3_log_probs_workspace_bytes(const y3_log_probs_desc *d, int64_t *bytes) {
    const int rc = check_desc(d);
    if (rc) return rc;
    Y3_REQUIRE(bytes, Y3_E_INVALID, "log_probs: null pointer");
    const Chunks c = chunks_of(d);
    *bytes = c.n > 1 ? d->rows * c.n * (16 + 8 * (int64_t)d->top) : 0;
    return Y3_OK;
}

extern "C" int y3_log_probs(const y3_log_probs_desc *d, const void *logits, const int64_t *row_offsets, const void *ids, float *logp,
                            float *entropy, int32_t *top_ids, float *top_logp, void *workspace, int64_t workspace_bytes, void *stream) {
    int64_t need = 0;
    const int rc = y3_log_probs_workspace_bytes(d, &need);
    if (rc) return rc;
    if (d->rows == 0) return Y3_OK;
    Y3_REQUIRE(logits && (logp || entropy || d->top), Y3_E_INVALID, "log_probs: null pointer");
    Y3_REQUIRE((ids != nullptr) == (logp != nullptr), Y3_E_INVALID, "log_probs: ids and logp go together");
    Y3_REQUIRE(d->top == 0 || (top_ids && top_logp), Y3_E_INVALID, "log_probs: top = %d without top_ids / top_logp", d->top);
    Y3_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), Y3_E_INVALID, "log_probs: workspace of %lld bytes, needs %lld", (long long)workspace_bytes, (long long)need);
    Y3_REQUIRE((uintptr_t)logits % (d->dtype == Y3_F32 ? 4 : 2) == 0 && (uintptr_t)ids % (d->ids_64 ? 8 : 4) == 0 && (uintptr_t)row_offsets % 8 == 0 &&
               ((uintptr_t)logp | (uintptr_t)entropy | (uintptr_t)top_ids | (uintptr_t)top_logp) % 4 == 0 && aligned16(workspace), Y3_E_ALIGN, "log_probs: pointer not aligned");
    int64_t span = d->extent;                                    // logits from the first row's first to the last row's last
    if (!row_offsets) {
        Y3_REQUIRE(d->group >= 1 && d->group_ld >= 0 && d->row_ld >= 0 && d->group_ld <= (1ll << 40) && d->row_ld <= (1ll << 40), Y3_E_INVALID,
                   "log_probs: group %d, group_ld %lld, row_ld %lld", d->group, (long long)d->group_ld, (long long)d->row_ld);
        // the furthest row start: the last row, or the last of the last whole group
        const int64_t g = (d->rows - 1) / d->group, in_last = (d->rows - 1) % d->group;
        const double last = (double)g * d->group_ld + (double)in_last * d->row_ld;
        const double whole = g > 0 ? (double)(g - 1) * d->group_ld + (double)(d->group - 1) * d->row_ld : 0.0;
        Y3_REQUIRE((last > whole ? last : whole) + d->classes <= (double)d->extent, Y3_E_INVALID, "log_probs: %lld rows reach behind the extent of %lld elements", (long long)d->rows, (long long)d->extent);
        span = (int64_t)(last > whole ? last : whole) + d->classes;
    }
    // what is written: the outputs, and with several chunks the workspace (`need`); what is read: the logits, ids and offsets
    const struct Block { const void *p; int64_t bytes; } written[5] = {{logp, d->rows * 4}, {entropy, d->rows * 4}, {top_ids, d->rows * d->top * 4}, {top_logp, d->rows * d->top * 4}, {workspace, need}};
    const Block read[3] = {{logits, span * (d->dtype == Y3_F32 ? 4 : 2)}, {ids, d->rows * (d->ids_64 ? 8 : 4)}, {row_offsets, d->rows * 8}};
    const auto meet = [](const Block &a, const Block &b) {
        return a.p && b.p && a.bytes && b.bytes && (uintptr_t)a.p < (uintptr_t)b.p + b.bytes && (uintptr_t)b.p < (uintptr_t)a.p + a.bytes;
    };
    for (int i = 0; i < 5; ++i) {
        for (int j = 0; j < 3; ++j)
            Y3_REQUIRE(!meet(written[i], read[j]), Y3_E_INVALID, "log_probs: %s overlaps the %s", i < 4 ? "an output" : "the workspace", j == 0 ? "logits" : j == 1 ? "ids" : "row offsets");
        for (int j = 0; j < i; ++j) Y3_REQUIRE(!meet(written[i], written[j]), Y3_E_INVALID, "log_probs: outputs or the workspace overlap each other");
    }
    ProbsArgs a;
    a.z = (const char *)logits; a.row_offsets = row_offsets; a.ids = ids; a.logp = logp; a.entropy = entropy; a.top_ids = top_ids; a.top_logp = top_logp;
    a.rows = d->rows; a.group_ld = d->group_ld; a.row_ld = d->row_ld; a.extent = d->extent;
    a.classes = d->classes; a.group = d->group; a.top = d->top; a.ids_64 = d->ids_64 != 0;
    if (!row_offsets && d->group > 1 && d->rows < 0x7fffffff) a.fd_group = make_fastdiv(d->group);
    a.fast_group = !row_offsets && d->group > 1 && d->rows < 0x7fffffff;
    const Chunks c = chunks_of(d);
    a.chunks = c.n; a.chunk_vecs = c.vecs; a.chunk_more = c.more;
    a.sums = (f32x4 *)workspace;
    a.keys = (unsigned long long *)((char *)workspace + d->rows * c.n * 16);
    return d->dtype == Y3_F32 ? launch_probs<Y3_F32>(a, (hipStream_t)stream) : launch_probs<Y3_BF16>(a, (hipStream_t)stream);
}

extern "C" int y3_detection_rows(const y3_decode_desc *d, const int32_t *kept_idx, const int32_t *kept_count, int max_boxes, int64_t *row_offsets,
                                 int32_t *row_classes, void *stream) {
    Y3_REQUIRE(d && kept_idx && kept_count && row_offsets && row_classes, Y3_E_INVALID, "detection_rows: null pointer");
    Y3_REQUIRE(d->batch >= 1 && d->num_scales >= 1 && d->num_scales <= 3 && d->num_anchors >= 1, Y3_E_INVALID, "detection_rows: batch %d, %d scales, %d anchors", d->batch, d->num_scales, d->num_anchors);
    Y3_REQUIRE(d->num_classes >= 1 && d->num_classes <= MAX_CLASSES, Y3_E_INVALID, "detection_rows: num_classes %d (at most %d)", d->num_classes, MAX_CLASSES);
    Y3_REQUIRE(max_boxes >= 1 && max_boxes <= 256, Y3_E_INVALID, "detection_rows: max_boxes %d", max_boxes);
    for (int l = 0; l < d->num_scales; ++l)
        Y3_REQUIRE(d->grid_h[l] >= 1 && d->grid_w[l] >= 1 && d->head_ld[l] >= d->num_anchors * (5 + d->num_classes), Y3_E_INVALID, "detection_rows: scale %d: grid %d x %d, head_ld %d", l,
                   d->grid_h[l], d->grid_w[l], d->head_ld[l]);
    Y3_REQUIRE(((uintptr_t)kept_idx | (uintptr_t)kept_count | (uintptr_t)row_classes) % 4 == 0 && (uintptr_t)row_offsets % 8 == 0, Y3_E_ALIGN, "detection_rows: pointer not aligned");
    const int64_t pairs = (int64_t)d->batch * d->num_classes, cap = pairs * max_boxes;
    const auto meet = [](const void *a, int64_t na, const void *b, int64_t nb) { return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na; };
    const int64_t offsets = cap * 8 * d->num_scales;
    Y3_REQUIRE(!meet(row_offsets, offsets, row_classes, cap * 4) && !meet(row_offsets, offsets, kept_idx, cap * 4) && !meet(row_offsets, offsets, kept_count, pairs * 4) &&
               !meet(row_classes, cap * 4, kept_idx, cap * 4) && !meet(row_classes, cap * 4, kept_count, pairs * 4), Y3_E_INVALID, "detection_rows: outputs overlap each other or the kept boxes");
    RowsArgs a;
    a.d = *d; a.kept_idx = kept_idx; a.kept_count = kept_count; a.row_offsets = row_offsets; a.row_classes = row_classes; a.max_boxes = max_boxes;
    hipLaunchKernelGGL(detection_rows_kernel, dim3(d->batch), dim3(256), 0, (hipStream_t)stream, a);
    return y3_check_launch("detection_rows");
}
