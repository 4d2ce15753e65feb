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
constexpr int MAX_TOP = 32;

struct ProbsArgs {
    const char *z;
    const int64_t *row_offsets;
    const void *ids;
    float *logp, *entropy, *top_logp;
    int32_t *top_ids;
    long rows, group_ld, row_ld, extent;
    int classes, group, top, ids_64, fast_group;
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
struct MinI { __device__ __forceinline__ int operator()(int a, int b) const { return min(a, b); } };

// ---- few classes: L lanes per row, up to E logits in each lane's registers -------------------------------------------
// One read of the row; each alternative is a maximum over the registers and the lanes, the lowest class that has it, and
// that logit taken out (NaN: no maximum and no comparison sees it).
template <int DT, int L, int E>
__global__ __launch_bounds__(256) void probs_lanes_kernel(const ProbsArgs p) {
    constexpr int RPW = 64 / L;
    const int lane = threadIdx.x & 63, l = lane & (L - 1);
    const long waves = (long)gridDim.x * 4;
    const float nan = __builtin_nanf(""), ninf = -__builtin_inff();
    for (long r0 = ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * RPW; r0 < p.rows; r0 += waves * RPW) {
        const long r = r0 + lane / L;
        const long at = r < p.rows ? row_start(p, r) : -1;
        if (at < 0) {                                           // (the lanes of a row go together)
            if (at == -2) put_row_outside(p, r, l, L);
            continue;
        }
        const char *z = p.z + at * (DT == Y3_F32 ? 4 : 2);
        float x[E];
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = j * L + l < p.classes ? logit<DT>(z, j * L + l) : ninf;
        long id = -1;
        float zid = 0.0f;
        if (p.logp) {
            id = row_id(p, r);
            if (id >= 0 && id < p.classes) zid = logit<DT>(z, id);
        }
        float m = x[0];
#pragma unroll
        for (int j = 1; j < E; ++j) m = vmax_raw(m, x[j]);
        m = lanes_reduce<L>(m, Max());
        const float m0 = m == ninf ? 0.0f : m;
        float zs = 0.0f, ss = 0.0f;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const float d = x[j] - m0, e = __builtin_amdgcn_exp2f(d * LOG2E);
            zs += e;
            ss = fmaf(e, vmax_raw(d, -1e4f), ss);               // (an e of 0 adds nothing, whatever d is)
        }
        zs = lanes_reduce<L>(zs, Add());
        ss = lanes_reduce<L>(ss, Add());
        const bool none = zs == 0.0f, bad = !(zs < __builtin_inff());
        const float log_z = none ? 0.0f : logf(zs);
        if (l == 0) put_scalars(p, r, zid, id, m, log_z, none ? 0.0f : log_z - ss / zs);
        if (p.top) {
#pragma unroll
            for (int j = 0; j < E; ++j) x[j] = j * L + l < p.classes ? x[j] : nan;
            float keep_lp = 0.0f;
            int keep_id = 0;
            for (int t = 0; t < p.top; ++t) {
                float v = m;
                if (t) {
                    v = x[0];
#pragma unroll
                    for (int j = 1; j < E; ++j) v = vmax_raw(v, x[j]);
                    v = lanes_reduce<L>(v, Max());
                }
                int c = 0x7fffffff;
#pragma unroll
                for (int j = E - 1; j >= 0; --j) c = x[j] == v ? j * L + l : c;
                c = lanes_reduce<L>(c, MinI());
#pragma unroll
                for (int j = 0; j < E; ++j) x[j] = c == j * L + l ? nan : x[j];
                if (l == (t & (L - 1))) {                        // lane t keeps alternative t: rows are stored in one piece
                    keep_id = bad ? t : c;
                    keep_lp = bad ? nan : log_prob(v, m, log_z);
                }
                if ((t & (L - 1)) == L - 1 || t == p.top - 1) {
                    const int first = t & ~(L - 1);
                    if (first + l <= t) {
                        p.top_ids[r * p.top + first + l] = keep_id;
                        p.top_logp[r * p.top + first + l] = keep_lp;
                    }
                }
            }
        }
    }
}

// ---- many classes: W waves per row ----------------------------------------------------------------------------------
// One pass with a running maximum per lane (Z and S scaled along with it).  The row is read in 16-byte vectors: vector 0 is
// what lies in front of the first 16-byte border, the last one what lies behind the last; lane t of the row takes vectors
// t, t + 64 W, ...  Each lane remembers its largest logit and the vector that has it.  For `top` alternatives the wave's
// top-th largest of these 64 maxima is a bound T that at least `top` of its logits reach, and only the lanes whose maximum
// reaches T hold such logits: their vectors alone (top of 64) are read again, from cache, and the logits from T on listed.
// The bound is a key with the class in it, so equal logits do not swell the list; should it fill up all the same, it is
// cut to its `top` largest, which raises T.  Waves join through LDS, in a fixed order.
constexpr int LIST = 192;

typedef unsigned long long u64;
__device__ __forceinline__ u64 key_of(float x, int c) { return (u64)order_of(x) << 32 | (0xffffffffu - (unsigned)c); }

// LDS is in order within a wave; this keeps the compiler to it (what another lane wrote is read behind it)
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// the `top` largest of list[0 .. n) to its front, in order, the rest of the first `top` cleared; returns the last one's key
__device__ __forceinline__ u64 cut_list(u64 *list, int n, int top, int lane) {
    u64 k[LIST / 64];
    int rank[LIST / 64];
#pragma unroll
    for (int i = 0; i < LIST / 64; ++i) {
        k[i] = lane + 64 * i < n ? list[lane + 64 * i] : 0;
        rank[i] = 0;
    }
    for (int s = 0; s < n; ++s) {
        const u64 o = list[s];
#pragma unroll
        for (int i = 0; i < LIST / 64; ++i) rank[i] += o > k[i];
    }
    wave_sync();
    if (lane < top) list[lane] = 0;
    wave_sync();
#pragma unroll
    for (int i = 0; i < LIST / 64; ++i)
        if (k[i] && rank[i] < top) list[rank[i]] = k[i];
    wave_sync();
    return list[top - 1];
}

template <int DT, int W>
__global__ __launch_bounds__(64 * W) void probs_row_kernel(const ProbsArgs p) {
    constexpr int VE = DT == Y3_F32 ? 4 : 8, ES = DT == Y3_F32 ? 4 : 2, STEP = 64 * W, G = 4;
    __shared__ u64 lists[W][LIST];
    __shared__ float part[W][3];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float ninf = -__builtin_inff();
    u64 *list = lists[wave];
    for (long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const long at = row_start(p, r);
        if (at < 0) {
            if (at == -2) put_row_outside(p, r, threadIdx.x, STEP);
            continue;
        }
        const char *z = p.z + at * ES;
        const int C = p.classes, head = (int)((16 - ((uintptr_t)z & 15)) & 15) / ES;
        const int vecs = 1 + (C > head ? (C - head + VE - 1) / VE : 0), whole = 1 + (C > head ? (C - head) / VE : 0);
        const auto unpack = [&](const u32x4 &v, float (&x)[VE]) {
            if constexpr (DT == Y3_F32) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) { x[2 * j] = __uint_as_float(v[j] << 16); x[2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u); }
            }
        };
        const auto first_of = [&](int u) { return head + (u - 1) * VE; };
        const auto load = [&](int u, float (&x)[VE]) {           // any vector; -inf where the row has nothing
            const int b = first_of(u);
            if (u >= 1 && u < whole) unpack(*(const u32x4 *)(z + (long)b * ES), x);
            else
#pragma unroll
                for (int j = 0; j < VE; ++j) x[j] = b + j >= 0 && b + j < C ? logit<DT>(z, b + j) : ninf;
        };
        float m = ninf, zs = 0.0f, ss = 0.0f, big = ninf;
        int big_u = threadIdx.x;
        const auto take = [&](int u, float (&x)[G][VE]) {        // G vectors u, u + STEP, ..
            float vm[G], gm = ninf;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                vm[g] = x[g][0];
#pragma unroll
                for (int j = 1; j < VE; ++j) vm[g] = vmax_raw(vm[g], x[g][j]);
                gm = vmax_raw(gm, vm[g]);
                const bool more = vm[g] > big;
                big = more ? vm[g] : big;
                big_u = more ? u + g * STEP : big_u;
            }
            const float nm = vmax_raw(m, gm), n0 = nm == ninf ? 0.0f : nm;
            const float d = vmax_raw(m - nm, -1e4f), f = __builtin_amdgcn_exp2f(d * LOG2E);       // (m = -inf: Z = S = 0, f = 0)
            ss = f * fmaf(d, zs, ss);
            zs *= f;
            m = nm;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    const float y = x[g][j] - n0, e = __builtin_amdgcn_exp2f(y * LOG2E);
                    zs += e;
                    ss = fmaf(e, vmax_raw(y, -1e4f), ss);        // (an e of 0 adds nothing, whatever y is)
                }
        };
        int u = threadIdx.x;
        {                                                        // the first group has the head; the body has whole vectors only
            float x[G][VE];
#pragma unroll
            for (int g = 0; g < G; ++g) load(u + g * STEP, x[g]);
            take(u, x);
            u += G * STEP;
        }
        const int base = wave * 64;                              // (wave-uniform bounds)
        int ub = base + G * STEP;
        for (; ub + 63 + (G - 1) * STEP < whole; ub += G * STEP, u += G * STEP) {
            u32x4 v[G];
#pragma unroll
            for (int g = 0; g < G; ++g) v[g] = *(const u32x4 *)(z + (long)first_of(u + g * STEP) * ES);
            float x[G][VE];
#pragma unroll
            for (int g = 0; g < G; ++g) unpack(v[g], x[g]);
            take(u, x);
        }
        for (; ub < vecs; ub += G * STEP, u += G * STEP) {
            float x[G][VE];
#pragma unroll
            for (int g = 0; g < G; ++g) load(u + g * STEP, x[g]);
            take(u, x);
        }
        // the wave's sums
        {
            const float wm = lanes_reduce<64>(m, Max());
            const float d = vmax_raw(m - wm, -1e4f), f = __builtin_amdgcn_exp2f(d * LOG2E);
            ss = lanes_reduce<64>(f * fmaf(d, zs, ss), Add());
            zs = lanes_reduce<64>(zs * f, Add());
            m = wm;
        }
        const int top = p.top;
        if (top) {
            // this lane's largest logit as a key: the first place in its vector that has it
            u64 mine = 0;
            {
                float x[VE];
                load(big_u, x);
                const int b = first_of(big_u);
#pragma unroll
                for (int j = VE - 1; j >= 0; --j)
                    if (x[j] == big && b + j >= 0 && b + j < C) mine = key_of(big, b + j);
            }
            list[lane] = mine;
            wave_sync();
            int rank = 0;
            for (int s = 0; s < 64; ++s) rank += list[s] > mine;
            wave_sync();
            u64 bound = 0;                                       // 0: fewer than `top` lanes have anything, everything is listed
            {
                const u64 has = __ballot(rank == top - 1 && mine != 0);
                if (has) {
                    const int at_lane = __builtin_ctzll(has);
                    bound = (u64)(unsigned)__shfl((int)(mine >> 32), at_lane) << 32 | (unsigned)__shfl((int)mine, at_lane);
                }
            }
            int n = 0;
            if (top == 1 && bound) {
                if (lane == 0) list[0] = bound;
                n = 1;
            } else {
                // the lanes that reach the bound, packed into the low lanes (a lane without a key has a bound of 0 beside it)
                const u64 reach = __ballot(mine >= bound);
                const int lanes = __popcll(reach);
                const int place = __popcll(reach & ((1ull << lane) - 1));
                wave_sync();
                if (reach >> lane & 1) list[place] = (u64)lane;
                wave_sync();
                const int owner = lane < lanes ? (int)list[lane] : 0;      // (kept in a register: the list is filled next)
                wave_sync();
                const int per = (vecs - 1 - base + STEP) / STEP;           // vectors of the wave's first lane: the most any has
                const int items = vecs > base ? lanes * per : 0;
                for (int q0 = 0; q0 < items; q0 += 64) {
                    const int q = q0 + lane, o = min(q / per, lanes - 1);
                    const int uu = base + __shfl(owner, o) + (q - o * per) * STEP;
                    float x[VE];
                    const bool on = q < items && uu < vecs;
                    if (on) load(uu, x);
                    const int b = first_of(uu);
#pragma unroll
                    for (int j = 0; j < VE; ++j) {
                        const u64 k = on && b + j >= 0 && b + j < C ? key_of(x[j], b + j) : 0;
                        const bool in = k != 0 && k >= bound;
                        const u64 set = __ballot(in);
                        if (set == 0) continue;
                        if (n + __popcll(set) > LIST) {
                            const u64 last = cut_list(list, n, top, lane);
                            n = top;                              // (n > LIST - 64 > 32: there are at least `top`)
                            bound = last > bound ? last : bound;
                        }
                        if (in) list[n + __popcll(set & ((1ull << lane) - 1))] = k;
                        n += __popcll(set);
                        wave_sync();
                    }
                }
            }
            cut_list(list, n, top, lane);
        }
        if constexpr (W > 1) {
            if (lane == 0) { part[wave][0] = m; part[wave][1] = zs; part[wave][2] = ss; }
            __syncthreads();
            if (top || wave == 0) {
                float tm = part[0][0];
#pragma unroll
                for (int w = 1; w < W; ++w) tm = vmax_raw(tm, part[w][0]);
                float tz = 0.0f, ts = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float d = vmax_raw(part[w][0] - tm, -1e4f), f = __builtin_amdgcn_exp2f(d * LOG2E);
                    ts += f * fmaf(d, part[w][1], part[w][2]);
                    tz += f * part[w][1];
                }
                m = tm; zs = tz; ss = ts;
            }
        }
        const bool none = zs == 0.0f, bad = !(zs < __builtin_inff());
        const float log_z = none ? 0.0f : logf(zs);
        if (threadIdx.x == 0) {
            long id = -1;
            float zid = 0.0f;
            if (p.logp) {
                id = row_id(p, r);
                if (id >= 0 && id < C) zid = logit<DT>(z, id);
            }
            put_scalars(p, r, zid, id, m, log_z, none ? 0.0f : log_z - ss / zs);
        }
        if (top) {
            // the place of every wave's keys among all: keys are distinct, so counting the larger ones is enough
            for (int q = threadIdx.x; q < W * top; q += STEP) {
                const u64 k = lists[q / top][q % top];
                int rank = 0;
                if constexpr (W == 1) rank = q;
                else
                    for (int w = 0; w < W; ++w)
                        for (int s = 0; s < top; ++s) rank += lists[w][s] > k;
                if (bad ? q < top : (k != 0 && rank < top)) {
                    const int to = bad ? q : rank;
                    p.top_ids[r * top + to] = bad ? q : (int)(0xffffffffu - (unsigned)k);
                    p.top_logp[r * top + to] = bad ? __builtin_nanf("") : log_prob(of_order((unsigned)(k >> 32)), m, log_z);
                }
            }
        }
        if (W > 1) __syncthreads();                              // (the next row writes the lists and the sums again)
        else wave_sync();
    }
}

template <int DT, int L, int E> void launch_lanes(const ProbsArgs &a, hipStream_t st) {
    const long waves = (a.rows + 64 / L - 1) / (64 / L), blocks = (waves + 3) / 4;
    hipLaunchKernelGGL((probs_lanes_kernel<DT, L, E>), dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st, a);
}
template <int DT, int W> void launch_row(const ProbsArgs &a, hipStream_t st) {
    hipLaunchKernelGGL((probs_row_kernel<DT, W>), dim3((unsigned)(a.rows < 65536 ? a.rows : 65536)), dim3(64 * W), 0, st, a);
}
template <int DT> void launch_probs(const ProbsArgs &a, hipStream_t st) {
    const int C = a.classes;
    if (C <= 32) launch_lanes<DT, 8, 4>(a, st);
    else if (C <= 64) launch_lanes<DT, 8, 8>(a, st);
    else if (C <= 80) launch_lanes<DT, 8, 10>(a, st);
    else if (C <= 128) launch_lanes<DT, 8, 16>(a, st);
    else if (C <= 256) launch_lanes<DT, 16, 16>(a, st);
    else if (C <= 512) launch_lanes<DT, 32, 16>(a, st);
    else if (C <= 1024) launch_lanes<DT, 64, 16>(a, st);
    else if (a.rows <= 256 && C > 8192) launch_row<DT, 16>(a, st);
    else if (a.rows <= 2048 || C > 8192) launch_row<DT, 4>(a, st);
    else launch_row<DT, 1>(a, st);
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
    *bytes = 0;
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
    if (!row_offsets) {
        Y3_REQUIRE(d->group >= 1 && d->group_ld >= 0 && d->row_ld >= 0 && d->group_ld <= (1ll << 40) && d->row_ld <= (1ll << 40), Y3_E_INVALID,
                   "log_probs: group %d, group_ld %lld, row_ld %lld", d->group, (long long)d->group_ld, (long long)d->row_ld);
        // the furthest row start: the last row, or the last of the last whole group
        const int64_t g = (d->rows - 1) / d->group, in_last = (d->rows - 1) % d->group;
        const double last = (double)g * d->group_ld + (double)in_last * d->row_ld;
        const double whole = g > 0 ? (double)(g - 1) * d->group_ld + (double)(d->group - 1) * d->row_ld : 0.0;
        Y3_REQUIRE((last > whole ? last : whole) + d->classes <= (double)d->extent, Y3_E_INVALID, "log_probs: %lld rows reach behind the extent of %lld elements", (long long)d->rows, (long long)d->extent);
    }
    ProbsArgs a;
    a.z = (const char *)logits; a.row_offsets = row_offsets; a.ids = ids; a.logp = logp; a.entropy = entropy; a.top_ids = top_ids; a.top_logp = top_logp;
    a.rows = d->rows; a.group_ld = d->group_ld; a.row_ld = d->row_ld; a.extent = d->extent;
    a.classes = d->classes; a.group = d->group; a.top = d->top; a.ids_64 = d->ids_64 != 0;
    if (!row_offsets && d->group > 1 && d->rows < 0x7fffffff) a.fd_group = make_fastdiv(d->group);
    a.fast_group = !row_offsets && d->group > 1 && d->rows < 0x7fffffff;
    if (d->dtype == Y3_F32) launch_probs<Y3_F32>(a, (hipStream_t)stream);
    else launch_probs<Y3_BF16>(a, (hipStream_t)stream);
    return y3_check_launch("log_probs");
}
