// 8-bit product, 256 rows x 256 channels per workgroup: the main loop of conv_pp.hip (two wave groups half a phase apart,
// operands through LDS by LDS-DMA two k-steps ahead, counted waits) on v_mfma_i32_16x16x64_i8.
//
// A k-step is 128 inputs.  Its operands are four half-tiles of 16 KB: X0 / X1 = the rows of the waves' first / second 64
// rows, W0 / W1 = their first / second 32 channels.  X is read as rows of 128 bytes (16-byte chunks XOR-swizzled by
// (row >> 1) & 7, on the source address and on the fragment read), W as whole packed fragments: a fragment is 1 KB of memory,
// one LDS-DMA instruction, and 64 consecutive 16-byte slots of LDS, so neither its load nor its read needs an address
// beyond a base and an immediate.  Rows and channels past the ends are past the buffer descriptors' extents and read as zero;
// with an odd number of k-steps one more is run on zero weights, so that a k-step's LDS buffer is a compile-time constant.
// The scales and the bias of a tile come by LDS-DMA too (a plain load would make the compiler drain every request in flight)
// and are held twice, for the tile being multiplied and the one being loaded.
//
// Tiles are walked XCD by XCD, within one in blocks of GROUP_M tile rows: the 32 CUs of an XCD then share 8 + 4 slabs of the
// operands at a time instead of 1 + 32.  Bound by the matrix pipe: 8192 x 8192 -> 8192 385 us, 2.86 POP/s, 57 % of its dense
// peak (the panel kernel: 640); 2048 x 4096 -> 4096 with its pass over bf16 rows, on half of the CUs, 52 us.
#include "linear_i8.h"
#include <type_traits>

namespace {

constexpr int TL_XBUF = 32 * 1024;
constexpr int TL_W0 = 2 * TL_XBUF;
constexpr int TL_VEC = 4 * TL_XBUF;                 // [parity][row scales | channel scales | bias] of 256 floats
constexpr int TL_LDS = TL_VEC + 2 * 3 * 1024;
constexpr int GROUP_M = 8;

constexpr int tl_wait_enc(int v) { return (v & 15) | (7 << 4) | (15 << 8) | ((v >> 4) << 14); }    // s_waitcnt vmcnt(v) only

template <int N> using ic = std::integral_constant<int, N>;

// One LDS-DMA instruction: 16 (4) bytes per lane to (wave-uniform LDS address + lane * 16 (4)); zeros past the extent.
__device__ __forceinline__ void bufdma16(__amdgpu_buffer_rsrc_t rs, unsigned off, char *lds_wave_base) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void *)lds_wave_base, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void bufdma4(__amdgpu_buffer_rsrc_t rs, unsigned off, char *lds_wave_base) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void *)lds_wave_base, 4, off, 0, 0, 0);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void *base, long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (unsigned)min(bytes, 0x7ffff000L), 0x00020000);
}

template <int OUT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void linear_i8_tile_kernel(const LinArgs p, int m_tiles, int n_tiles, int total) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    const int nk = p.kb >> 1, nk2 = (nk + 1) & ~1;               // k-steps, and with the one on zero weights
    const long w_tile_bytes = (long)p.kb * 1024;                 // of 16 channels

    const auto place = [&](int tile, int &mt, int &nt) {
        const int id = xcd_remap(tile, total);
        const int g = id / (GROUP_M * n_tiles), r = id - g * GROUP_M * n_tiles;
        const int gm = min(GROUP_M, m_tiles - g * GROUP_M);
        nt = r / gm;
        mt = g * GROUP_M + r - nt * gm;
    };

    // ---- loader ------------------------------------------------------------------------------------------------------
    const int lrow = tid >> 3;
    const unsigned kc = ((tid & 7) ^ ((tid >> 4) & 7)) * 16;     // source chunk of this LDS slot
    unsigned x_off[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) x_off[q] = (unsigned)((lrow + 64 * q) * p.x_ld) + kc;
    unsigned w_off[2];                                           // this wave's two fragments of a half: channels 16 (wave & 1) ..
#pragma unroll
    for (int h = 0; h < 2; ++h) w_off[h] = (unsigned)(((wave >> 1) * 4 + h * 2 + (wave & 1)) * w_tile_bytes) + lane * 16;
    int l_tile = blockIdx.x, l_kt = 0, lb = 0, l_par = 0;        // (wave-uniform) the k-step the loader is on, its buffers
    bool l_live = l_tile < total;
    __amdgpu_buffer_rsrc_t rs_x = rsrc(p.x, 0), rs_w = rsrc(p.w, 0);
    const auto l_tile_begin = [&]() {
        int mt, nt;
        place(l_tile, mt, nt);
        const long m0 = (long)mt * 256, n0 = (long)nt * 256;
        rs_x = rsrc(p.x + m0 * p.x_ld, (min(p.rows - m0, 256L) - 1) * p.x_ld + p.k16);
        rs_w = rsrc(p.w + nt * 16 * w_tile_bytes, min((p.n + 15) / 16 - nt * 16, 16) * w_tile_bytes);
        char *vec = smem + TL_VEC + l_par * (3 * 1024) + wn * 256;
        if (wm == 0) {
            bufdma4(rsrc(p.x_scale + m0, (p.rows - m0) * 4), wn * 256 + lane * 4, vec);
            bufdma4(rsrc(p.bias ? p.bias + n0 : p.w_scale, p.bias ? (p.n - n0) * 4 : 0), wn * 256 + lane * 4, vec + 2048);
        } else {
            bufdma4(rsrc(p.w_scale + n0, (p.n - n0) * 4), wn * 256 + lane * 4, vec + 1024);
        }
    };
    const auto l_advance = [&]() {
        ++l_kt;
        lb ^= 1;
        if (l_kt == nk2) {
            l_kt = 0;
            l_par ^= 1;
            l_tile += (int)gridDim.x;
            l_live = l_tile < total;
            if (l_live) l_tile_begin();
        }
    };
    const auto stage_x = [&](int h) {
        if (!l_live) return;
#pragma unroll
        for (int j = 0; j < 2; ++j) bufdma16(rs_x, x_off[h + 2 * j] + (unsigned)(l_kt * 128), smem + lb * TL_XBUF + (h + 2 * j) * 8192 + wave * 1024);
    };
    const auto stage_w = [&](int h) {
        if (!l_live) return;
        const unsigned off = l_kt < nk ? w_off[h] + (unsigned)(l_kt * 2048) : 0x7ffff000u;        // (past every extent: zeros)
#pragma unroll
        for (int j = 0; j < 2; ++j) bufdma16(rs_w, off + j * 1024, smem + TL_W0 + lb * TL_XBUF + h * 16384 + (wave * 2 + j) * 1024);
    };

    // ---- consumer addressing: per-lane bases, everything else is an immediate ----------------------------------------
    const int frow = lane & 15, fq = lane >> 4, fsw = (lane >> 1) & 7;
    const int xb0 = (wm * 128 + frow) * 128 + ((0 + fq) ^ fsw) * 16, xb1 = (wm * 128 + frow) * 128 + ((4 + fq) ^ fsw) * 16;
    const int wb = TL_W0 + wn * 4096 + lane * 16;

    // ---- prologue: k-step 0 complete, k-step 1's X0, W0 and W1 in flight ----------------------------------------------
    if (l_live) l_tile_begin();
    stage_x(0);
    stage_w(0);
    stage_w(1);
    stage_x(1);
    l_advance();
    stage_x(0);
    stage_w(0);
    stage_w(1);
    __builtin_amdgcn_s_waitcnt(tl_wait_enc(6));
    __builtin_amdgcn_s_barrier();

    int c_par = 0;
    for (int c_tile = blockIdx.x; c_tile < total; c_tile += (int)gridDim.x, c_par ^= 1) {
        i32x4 acc[4][8];
#pragma unroll
        for (int ni = 0; ni < 4; ++ni)
#pragma unroll
            for (int mi = 0; mi < 8; ++mi) acc[ni][mi] = i32x4{0, 0, 0, 0};
        const auto kstep = [&](auto CB) {
            constexpr int cb = decltype(CB)::value;
            i32x4 xf[4][2], wf[4][2];
            const auto read_x = [&](auto XH) {
                constexpr int xh = decltype(XH)::value;
#pragma unroll
                for (int mi = 0; mi < 4; ++mi) {
                    xf[mi][0] = *(const i32x4 *)(smem + xb0 + (cb * TL_XBUF + (xh * 64 + mi * 16) * 128));
                    xf[mi][1] = *(const i32x4 *)(smem + xb1 + (cb * TL_XBUF + (xh * 64 + mi * 16) * 128));
                }
            };
            const auto read_w = [&](auto WH) {
                constexpr int wh = decltype(WH)::value;
#pragma unroll
                for (int ni = 0; ni < 2; ++ni)
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks)
                        wf[2 * wh + ni][ks] = *(const i32x4 *)(smem + wb + (cb * TL_XBUF + wh * 16384 + ni * 2048 + ks * 1024));
            };
            const auto mfmas = [&](auto XH, auto WH) {
                constexpr int xh = decltype(XH)::value, wh = decltype(WH)::value;
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int ni = 0; ni < 2; ++ni)
#pragma unroll
                        for (int mi = 0; mi < 4; ++mi)
                            acc[2 * wh + ni][4 * xh + mi] =
                                __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[2 * wh + ni][ks], xf[mi][ks], acc[2 * wh + ni][4 * xh + mi], 0, 0, 0);
            };
            // group 1 runs half a phase behind group 0: its barrier comes first, group 0's last.  A load segment ends with
            // its own fragment reads retired (lgkmcnt(0) before the barrier): what a phase has read may be overwritten by
            // requests issued in the next one.
            const auto seg_load = [&]() {
                if (wm == 1) __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
            };
            const auto seg_mfma = [&]() {
                __builtin_amdgcn_s_waitcnt(0xC07F);              // lgkmcnt(0) only
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
            };
            const auto seg_end = [&]() {
                __builtin_amdgcn_sched_barrier(0);
                if (wm == 0) __builtin_amdgcn_s_barrier();
            };
            // phase A: X0 x (W0, W1); requests X1 of the loader's k-step (the next one).  X1 of this k-step has landed once
            // only the eight youngest requests remain (the last phase B's six, these two; scales only make it stricter)
            seg_load();
            read_w(ic<0>{});
            read_x(ic<0>{});
            read_w(ic<1>{});
            stage_x(1);
            if (l_live) __builtin_amdgcn_s_waitcnt(tl_wait_enc(8));
            else __builtin_amdgcn_s_waitcnt(tl_wait_enc(0));
            seg_mfma();
            mfmas(ic<0>{}, ic<0>{});
            mfmas(ic<0>{}, ic<1>{});
            seg_end();
            // phase B: X1 x (W1, W0); requests X0, W0, W1 of the k-step after the next
            seg_load();
            read_x(ic<1>{});
            l_advance();
            stage_x(0);
            stage_w(0);
            stage_w(1);
            if (l_live) __builtin_amdgcn_s_waitcnt(tl_wait_enc(8));
            else __builtin_amdgcn_s_waitcnt(tl_wait_enc(0));
            seg_mfma();
            mfmas(ic<1>{}, ic<1>{});
            mfmas(ic<1>{}, ic<0>{});
            seg_end();
        };
        for (int kt = 0; kt < nk2; kt += 2) {
            kstep(ic<0>{});
            kstep(ic<1>{});
        }
        // ---- epilogue: channels fq 4 .. + 3 of each 16, for rows frow of each 16 ----------------------------------------
        int mt, nt;
        place(c_tile, mt, nt);
        const char *vec = smem + TL_VEC + c_par * (3 * 1024);
        float s[8];
#pragma unroll
        for (int mi = 0; mi < 8; ++mi) s[mi] = *(const float *)(vec + (wm * 128 + mi * 16 + frow) * 4);
        const long row0 = (long)mt * 256 + wm * 128 + frow;
        const int col0 = nt * 256 + wn * 64;
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) {
            f32x4 t[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                t[i] = *(const f32x4 *)(vec + 1024 + (wn * 64 + (2 * pr + i) * 16 + fq * 4) * 4);
                b[i] = *(const f32x4 *)(vec + 2048 + (wn * 64 + (2 * pr + i) * 16 + fq * 4) * 4);
            }
#pragma unroll
            for (int mi = 0; mi < 8; ++mi) {
                const long row = row0 + mi * 16;
                if constexpr (OUT == Y3_F32) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) store4(p, row, col0 + (2 * pr + i) * 16 + fq * 4, acc[2 * pr + i][mi], s[mi], t[i], b[i]);
                } else {
                    float y[2][4];
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            y[i][j] = leaky_max(fmaf((float)acc[2 * pr + i][mi][j] * t[i][j], s[mi], b[i][j]), p.slope);
                        }
                    // the two 16-channel blocks change places between neighbouring quarter-waves: eight channels per lane
                    const auto s0 = __builtin_amdgcn_permlane16_swap(pack_bf16x2(y[0][0], y[0][1]), pack_bf16x2(y[1][0], y[1][1]), false, false);
                    const auto s1 = __builtin_amdgcn_permlane16_swap(pack_bf16x2(y[0][2], y[0][3]), pack_bf16x2(y[1][2], y[1][3]), false, false);
                    const u32x4 o = {s0[0], s1[0], s0[1], s1[1]};
                    const int c = col0 + pr * 32 + ((fq & 1) ? 16 + (fq - 1) * 4 : fq * 4);
                    if (row < p.rows) {
                        unsigned short *to = (unsigned short *)p.out + row * p.out_ld + c;
                        if (c + 8 <= p.n) *(u32x4_u2 *)to = o;
                        else
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (c + j < p.n) to[j] = (unsigned short)(o[j / 2] >> (16 * (j & 1)));
                    }
                }
            }
        }
    }
}

}  // namespace

// Worth it where the tiles fill most of the CUs and the loop is long enough to matter.
bool y3_linear_i8_tile_ok(const LinArgs &a, long cus) {
    const long tiles = (a.rows + 255) / 256 * ((a.n + 255) / 256);
    return a.kb >= 8 && tiles >= cus / 2 && tiles <= 0x7fffffffL / 2 && a.x_ld <= (1 << 22);
}

int y3_linear_i8_tile_launch(const LinArgs &a, long cus, hipStream_t stream) {
    static thread_local int attr_dev = -1;
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (attr_dev != dev) {
        if (hipFuncSetAttribute((const void *)linear_i8_tile_kernel<Y3_BF16>, hipFuncAttributeMaxDynamicSharedMemorySize, TL_LDS) != hipSuccess ||
            hipFuncSetAttribute((const void *)linear_i8_tile_kernel<Y3_F32>, hipFuncAttributeMaxDynamicSharedMemorySize, TL_LDS) != hipSuccess) {
            y3_set_error("linear_i8: cannot reserve %d bytes of LDS", TL_LDS);
            return Y3_E_LAUNCH;
        }
        attr_dev = dev;
    }
    const int m_tiles = (int)((a.rows + 255) / 256), n_tiles = (a.n + 255) / 256;
    const long total = (long)m_tiles * n_tiles;
    const unsigned grid = (unsigned)(total < cus ? total : cus);                 // one workgroup per CU (LDS), persistent
    if (a.out_f32) hipLaunchKernelGGL(linear_i8_tile_kernel<Y3_F32>, dim3(grid), dim3(512), TL_LDS, stream, a, m_tiles, n_tiles, (int)total);
    else hipLaunchKernelGGL(linear_i8_tile_kernel<Y3_BF16>, dim3(grid), dim3(512), TL_LDS, stream, a, m_tiles, n_tiles, (int)total);
    return y3_check_launch("linear_i8 (tiles)");
}
