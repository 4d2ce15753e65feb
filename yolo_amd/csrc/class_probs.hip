// Log probabilities of given classes, entropy and the top alternatives of rows of logits, for gfx950 (MI355X): y3_log_probs.
//
//   M = max z    Z = sum exp(z - M)    S = sum exp(z - M) (z - M)    log p_c = (z_c - M) - log Z    H = log Z - S / Z
// Z >= 1 and S <= 0, so the entropy is a sum of two terms that are not negative: nothing cancels.  Everything is fp32.
// The alternatives are the largest 64-bit keys {order of the logit, ~class}: a total order, so ties go to the lowest class
// and no order of arrival shows in the result.
#include "common.h"

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
    int classes, group, top, ids_64;
};

template <int DT> __device__ __forceinline__ float logit(const char *z, long i) {
    if constexpr (DT == Y3_F32) return ((const float *)z)[i];
    else return bf16_to_f32(((const unsigned short *)z)[i]);
}

// element offset of a row; -1: skip it, -2: it does not lie within the extent
__device__ __forceinline__ long row_start(const ProbsArgs &p, long r) {
    if (!p.row_offsets) return (r / p.group) * p.group_ld + (r % p.group) * p.row_ld;
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

template <typename T, typename F> __device__ __forceinline__ T block_reduce(T v, T *red, F f) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = f(v, __shfl_xor(v, o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = f(f(red[0], red[1]), f(red[2], red[3]));
    __syncthreads();
    return v;
}

// One workgroup per row: maximum, sums, then one pass per alternative.
template <int DT>
__global__ __launch_bounds__(256) void log_probs_kernel(const ProbsArgs p) {
    __shared__ float redf[4];
    __shared__ unsigned long long redk[4];
    for (long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const long at = row_start(p, r);
        if (at == -1) continue;
        if (at == -2) {
            if (threadIdx.x == 0) {
                if (p.logp) p.logp[r] = __builtin_nanf("");
                if (p.entropy) p.entropy[r] = __builtin_nanf("");
            }
            for (int j = threadIdx.x; j < p.top; j += 256) { p.top_ids[r * p.top + j] = -1; p.top_logp[r * p.top + j] = __builtin_nanf(""); }
            continue;
        }
        const char *z = p.z + at * (DT == Y3_F32 ? 4 : 2);
        float m = -__builtin_inff();
        for (int c = threadIdx.x; c < p.classes; c += 256) m = fmaxf(m, logit<DT>(z, c));
        m = block_reduce(m, redf, [](float a, float b) { return fmaxf(a, b); });
        const float m0 = m == -__builtin_inff() ? 0.0f : m;
        float zs = 0.f, ss = 0.f;
        for (int c = threadIdx.x; c < p.classes; c += 256) {
            const float d = logit<DT>(z, c) - m0;
            const float e = __builtin_amdgcn_exp2f(d * LOG2E);
            zs += e;
            ss += e * fmaxf(d, -1e4f);                      // (an e of 0 adds nothing, whatever d is)
        }
        zs = block_reduce(zs, redf, [](float a, float b) { return a + b; });
        ss = block_reduce(ss, redf, [](float a, float b) { return a + b; });
        const bool none = zs == 0.0f;                       // every logit is -inf
        const float log_z = none ? 0.0f : logf(zs);
        if (threadIdx.x == 0) {
            if (p.logp) {
                const long id = row_id(p, r);
                p.logp[r] = id < 0 ? 0.0f : id >= p.classes ? __builtin_nanf("") : log_prob(logit<DT>(z, id), m, log_z);
            }
            if (p.entropy) p.entropy[r] = none ? 0.0f : log_z - ss / zs;
        }
        unsigned long long last = ~0ull;
        for (int j = 0; j < p.top; ++j) {
            unsigned long long best = 0;
            for (int c = threadIdx.x; c < p.classes; c += 256) {
                const unsigned long long key = (unsigned long long)order_of(logit<DT>(z, c)) << 32 | (0xffffffffu - (unsigned)c);
                if (key < last && key > best) best = key;
            }
            last = block_reduce(best, redk, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
            if (threadIdx.x == 0) {
                p.top_ids[r * p.top + j] = (int)(0xffffffffu - (unsigned)last);
                p.top_logp[r * p.top + j] = log_prob(of_order((unsigned)(last >> 32)), m, log_z);
            }
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
    const unsigned grid = (unsigned)(d->rows < (1 << 20) ? d->rows : 1 << 20);
    if (d->dtype == Y3_F32) hipLaunchKernelGGL(log_probs_kernel<Y3_F32>, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(log_probs_kernel<Y3_BF16>, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
    return y3_check_launch("log_probs");
}
