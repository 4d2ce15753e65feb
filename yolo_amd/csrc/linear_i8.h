// Shared by the 8-bit products (linear_i8.hip, linear_i8_tile.hip): launch arguments and the store of four channels.
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(4))) int i32x4;

// 16 / 8 bytes at any element's alignment: global memory takes unaligned vector accesses
typedef u32x4 __attribute__((aligned(2))) u32x4_u2;
typedef u32x4 __attribute__((aligned(4))) u32x4_u4;
typedef f32x4 __attribute__((aligned(4))) f32x4_u4;
typedef unsigned long long __attribute__((aligned(2))) u64_u2;

struct LinArgs {
    const char *x;                     // 8-bit rows on 16 bytes, or float rows
    const float *x_scale;              // with 8-bit rows
    const char *w;
    const float *w_scale, *bias;       // bias may be null
    char *out;
    long rows, x_ld, out_ld;
    int k, k16, n, kb;                 // k rounded up to 16 (bytes of an 8-bit row that may be read), channels, 64-deep k-blocks
    float slope;                       // of the leaky-ReLU; 1: none
    int out_f32;
    int flat;                          // resident kernel: output rows end to end that do not start on 16 bytes
    int n_groups, slab;                // panel kernel: workgroups along n, k-blocks of a slab
    FastDiv fd_items;
};

namespace {

// four channels of one row: scaled, activated, stored.  t, b: the channels' scales and biases.
__device__ __forceinline__ void store4(const LinArgs &p, long row, int nl, const i32x4 &acc, float s, const f32x4 &t, const f32x4 &b) {
    if (row >= p.rows || nl >= p.n) return;
    const bool full = nl + 4 <= p.n;
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        y[j] = leaky_max(fmaf((float)acc[j] * t[j], s, b[j]), p.slope);
    }
    if (p.out_f32) {
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

}  // namespace

// linear_i8_tile.hip: 256 x 256 tiles for 8-bit rows (same packed weights, same sums: same bits as the panel kernel)
bool y3_linear_i8_tile_ok(const LinArgs &a, long cus);
int y3_linear_i8_tile_launch(const LinArgs &a, long cus, hipStream_t stream);
