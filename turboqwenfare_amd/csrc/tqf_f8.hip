// tqf_f8.hip -- products of e4m3 matrices with block-128 scales (gfx950).
//
//   f8_matmul   Y[t][n] = sum_b s_x[t][b] s_w[n / 128][b] sum_{k in b} q_x[t][k] q_w[n][k]
//   f8_experts  y[t] = sum_k w[t][k] D_e(silu(G_e x_t) * U_e x_t),  e = ids[t][k]
// with G, U, D products of the first kind, x and h quantised row by row in
// blocks b of 128 (tqf_f8.h has the format and the device layout).
//
// Weights are the A operand (16 or 32 of their rows), activation rows the B
// operand, so a lane's results are consecutive outputs of one activation row
// and a block's scale is one number per lane: d = the block's product from a
// zero start, acc = fma(d, s_x s_w, acc) in f32.
//
// How exact the block's product is.  The fp8 matrix instructions take eight
// products at a time and cut each to 2^-13 of the largest one's power of two
// (measured, tests/test_gpu_f8.py): a block loses less than 7 * 2^-13 of its
// magnitudes; against 64 bits, one of normal values is 1.3e-5 off (relative,
// 2-norm), 3.9e-5 with rows that span 2^8.  Rounding to bf16 costs 1.7e-3, so bf16
// results of large calls are made of these (f8_matmul's, and the down products of
// f8_experts).  f32 results, the experts' gate and up products, whose error the
// quantisation of h would make larger, and every small call widen the values to
// bf16 (exact) for the bf16 instructions, whose products of e4m3 values came out
// exact in the same test.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "tqf_f8.h"

namespace tqf {

namespace {

constexpr int kKB = 4096;  // bytes of a tile's K block

// ---- layout ------------------------------------------------------------------
__global__ __launch_bounds__(256) void f8_repack_kernel(const uint8_t *__restrict__ q, const float *__restrict__ scales,
                                                        F8Shape d, uint8_t *__restrict__ out) {
    const size_t chunks = f8_tile_bytes(d) / 16, i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t ns = (size_t)(d.tiles / 4) * d.kb;
    if (i < ns) reinterpret_cast<float *>(out + f8_tile_bytes(d))[i] = scales[i];
    if (i >= chunks) return;
    const uint32_t in = (uint32_t)(i & 255);  // chunk within the K block: 32 rows to each 16 columns
    const size_t blk = i >> 8, tile = blk / d.kb;
    const uint32_t kb = (uint32_t)(blk - tile * d.kb);
    const size_t row = tile * 32 + (in & 31);
    const uint32_t col = kb * 128 + (in >> 5) * 16;
    u32x4 v = {0, 0, 0, 0};
    if (row < d.rows && col < d.cols) {
        const uint8_t *src = q + row * d.cols + col;
        const uint32_t n = d.cols - col < 16 ? d.cols - col : 16;
        if (n == 16 && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            v = *reinterpret_cast<const u32x4 *>(src);
        } else {
            for (uint32_t j = 0; j < n; ++j) v[j >> 2] |= (uint32_t)src[j] << (8 * (j & 3));
        }
    }
    reinterpret_cast<u32x4 *>(out)[i] = v;
}

// ---- quantisation of rows ------------------------------------------------------
// Largest magnitude over the eight lanes that hold a block of 128.
__device__ __forceinline__ float amax8(float a) {
    a = fmaxf(a, dpp_f<kDppXor1>(a));
    a = fmaxf(a, dpp_f<kDppXor2>(a));
    return fmaxf(a, dpp_f<kDppHalfMirror>(a));
}
// Sixteen values of a block whose eight lanes are neighbours -> their bytes;
// *scale receives the block's.
__device__ __forceinline__ u32x4 quantize16(const float (&v)[16], float *scale) {
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) a = fmaxf(a, fabsf(v[i]));
    const F8Factors f = f8_factors(amax8(a));
    *scale = f.scale;
    u32x4 q;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        q[i] = f8_pack4(v[4 * i] * f.inv, v[4 * i + 1] * f.inv, v[4 * i + 2] * f.inv, v[4 * i + 3] * f.inv);
    return q;
}

// Quantised rows are kept by K block, [kb][t][128]: the tiled product reads many
// rows of one block at a time, which in rows of kb 128 bytes would lie kb 128
// apart, for most widths all in a few of the L2's channels.
// Chunk i of x [t x cols]: 16 columns; eight lanes share a block of a row (so all
// of an aligned group take part or none), a wavefront has eight rows.
__host__ __device__ __forceinline__ uint32_t quantize_chunks(uint32_t t, uint32_t kb) { return (t + 7) / 8 * 64 * kb; }
// TILED: by K block in tiles of 32 rows laid out as the weights', so that a
// wavefront loads an operand of 32 rows as 1 KiB that lies together; scales as
// [kb][tiles 32].
constexpr __host__ __device__ uint32_t pad32(uint32_t t) { return (t + 31) / 32 * 32; }
template <bool TILED, typename XT>
__device__ __forceinline__ void quantize_chunk(const XT *__restrict__ x, uint32_t t, uint32_t cols, uint32_t kb,
                                               uint32_t i, uint8_t *__restrict__ xq, float *__restrict__ xs) {
    const uint32_t rows8 = i / (64 * kb), block = i / 64 - rows8 * kb, row = rows8 * 8 + i / 8 % 8, k = block * 128 + i % 8 * 16;
    if (row >= t) return;
    const int valid = k < cols ? (int)(cols - k) : 0;
    float v[16], s;
    load_row<16>(x + (size_t)row * cols + k, valid, v);
    const u32x4 q = quantize16(v, &s);
    const size_t at = (size_t)block * (TILED ? pad32(t) : t) + row;
    reinterpret_cast<u32x4 *>(xq)[TILED ? (at - row % 32) * 8 + i % 8 * 32 + row % 32 : at * 8 + i % 8] = q;
    if (i % 8 == 0) xs[at] = s;
}
template <bool TILED, typename XT>
__global__ __launch_bounds__(256) void f8_quantize_kernel(const XT *__restrict__ x, uint32_t t, uint32_t cols, uint32_t kb,
                                                          uint8_t *__restrict__ xq, float *__restrict__ xs) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    quantize_chunk<TILED>(x, t, cols, kb, i, xq, xs);
}

// ---- matrix instructions ---------------------------------------------------------
// A policy says how a wavefront takes a K block: M weight rows by M activation
// rows to an accumulator D; `Raw` what a lane loads of an operand, `Op` what
// the instructions take.  a_off(l, sub, j): byte of load j in the K block of
// the tile; b_row / b_chunk: the activation row and the 16-column chunk of load
// j; row(l, g): the first of the four weight rows in D's group g.
struct Fp8x32 {  // v_mfma_f32_32x32x64_f8f6f4: two to a block
    static constexpr int M = 32, kLoads = 4, kGroups = 4;
    typedef f32x16 D;
    struct Raw {
        u32x4 q[4];
    };
    typedef Raw Op;
    static __device__ __forceinline__ uint32_t a_off(int l, int, int j) { return j * 1024 + l * 16; }
    static __device__ __forceinline__ int b_row(int l) { return l & 31; }
    static __device__ __forceinline__ int b_chunk(int l, int j) { return 2 * j + (l >> 5); }
    static __device__ __forceinline__ int row(int l, int g) { return 8 * g + 4 * (l >> 5); }
    static __device__ __forceinline__ const Op &op(const Raw &r) { return r; }
    static __device__ __forceinline__ i32x8 pair(u32x4 a, u32x4 b) {
        return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
    }
    static constexpr int kParts = 2;
    static __device__ __forceinline__ D part(const Op &a, const Op &b, const D &d, int i) {
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(pair(a.q[2 * i], a.q[2 * i + 1]), pair(b.q[2 * i], b.q[2 * i + 1]), d, 0, 0,
                                                               0, 0, 0, 0);
    }
    static __device__ __forceinline__ float across(float a) { return fmaxf(a, __shfl_xor(a, 32)); }
};
struct Bf16x16 {  // widened to bf16: v_mfma_f32_16x16x32_bf16, four to a block
    static constexpr int M = 16, kLoads = 2, kGroups = 1;
    typedef f32x4 D;
    struct Raw {
        u32x4 q[2];
    };
    struct Op {
        bf16x8 v[4];
    };
    static __device__ __forceinline__ uint32_t a_off(int l, int sub, int j) {
        return (4 * j + (l >> 4)) * 512 + sub * 256 + (l & 15) * 16;
    }
    static __device__ __forceinline__ int b_row(int l) { return l & 15; }
    static __device__ __forceinline__ int b_chunk(int l, int j) { return 4 * j + (l >> 4); }
    static __device__ __forceinline__ int row(int l, int) { return 4 * (l >> 4); }
    static __device__ __forceinline__ float across(float a) {
        a = fmaxf(a, __shfl_xor(a, 16));
        return fmaxf(a, __shfl_xor(a, 32));
    }
    static __device__ __forceinline__ Op op(const Raw &r) {
        return Op{{f8_widen(r.q[0][0], r.q[0][1]), f8_widen(r.q[0][2], r.q[0][3]), f8_widen(r.q[1][0], r.q[1][1]),
                   f8_widen(r.q[1][2], r.q[1][3])}};
    }
    static constexpr int kParts = 4;
    static __device__ __forceinline__ D part(const Op &a, const Op &b, const D &d, int i) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], d, 0, 0, 0);
    }
    static __device__ __forceinline__ D mma(const Op &a, const Op &b) {
        D d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i) d = part(a, b, d, i);
        return d;
    }
};

// ---- copies to LDS -----------------------------------------------------------------
typedef __amdgpu_buffer_rsrc_t Desc;  // loads past `bytes` return zero
__device__ __forceinline__ Desc make_desc(const void *p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, (int)bytes, 0x00020000);
}
typedef __attribute__((address_space(3))) void lds_void;
// Matrices found through a table: without the address space the compiler would
// load through flat instructions, which also count as LDS accesses.
typedef __attribute__((address_space(1))) void global_void;
typedef __attribute__((address_space(1))) const uint8_t global_u8;
typedef __attribute__((address_space(1))) const float global_f32;
typedef __attribute__((address_space(1))) const u32x4 global_u32x4;
__device__ __forceinline__ void copy16(Desc d, uint32_t voff, uint32_t soff, void *lds) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (lds_void *)lds, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void copy4(Desc d, uint32_t voff, uint32_t soff, void *lds) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (lds_void *)lds, 4, voff, soff, 0, 0);
}
// This wavefront's loads (those to LDS among them) but the last N, and its LDS
// reads, are done, then the workgroup's.
template <int N>
__device__ __forceinline__ void publish() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// ---- the tiled product -----------------------------------------------------------
// TW sets of four wavefronts: TW CT M activation rows by 4 RT M weight rows, each
// set with CT M of the activation rows and each of its wavefronts with RT M of the
// weight rows.  The activation rows of a K block are copied to LDS by all and read
// by each, [row][8 chunks] with chunk c of row r in slot c ^ swizzle(r): the
// copies read whole 128-byte lines, and both the 8 and the 16 lanes that LDS serves
// together find their chunks in different banks.  Weights go straight to the
// registers of the wavefront that needs them, or (WL) through LDS too, where two
// sets share them.  AHEAD + 1 stages: a block's loads are issued AHEAD blocks
// before it is computed.  Measured: 4096 x 8192, K 4096 (bf16 y, 256 x 256 tiles)
// 124-131 us, 2.1-2.2 PFLOP/s at the clock the power limit leaves, the matrix cores
// busy 52% of it: LDS serves 192 KiB of operands to a K block, about as long as its
// matrix instructions take, and a quarter of the vector units' time goes to the
// block scales; gate_up of 512 tokens (64 x 256 tiles) 97 us, 5.4 TB/s of weights.
__device__ __forceinline__ int swizzle(int r) { return (r ^ (r >> 3 & 1)) & 7; }  // by r % 16

enum Mode { kDense, kGateUp, kDown };
constexpr int kTileWaves = 4;

// Rows of one expert, with its matrices, so that a workgroup finds all it needs
// in one load.  No rows: nothing to do.
struct Tile {
    uint32_t first, rows;  // positions
    const uint8_t *gate, *up, *down;
};

struct TiledArgs {
    const uint8_t *mat;              // kDense
    F8Shape d;                       // of the matrices
    const uint8_t *xq;               // activation rows [kb][xrows][128]
    const float *xs;                 // [kb][xrows]
    uint32_t xrows;
    void *y;                         // kDense: [t x rows]
    const Tile *tiles;               // experts
    uint32_t rblocks;                // experts: workgroups to a tile
    const int32_t *row_of_pos;       // kGateUp: the activation row of a position
    uint8_t *hq;                     // kGateUp: h [hkb][hrows][128] and its scales [hkb][hrows]
    float *hs;
    uint32_t hkb, hrows;
    void *out;                       // kDown: [positions][rows], f32 or Out16
    float *out_scales;               // Out16's: [positions][rows / 64]
};
// The outputs of a pair wait in memory for their weighted sum: as f32, or, where
// there are many and y is bf16, as f16 times a power of two for each 64 columns
// (one wavefront's) that brings the largest of them below 2^15.  That halves the
// bytes written and read again; it rounds by 2^-11 of the value (2^-39 of the
// largest for the smallest ones), where bf16 y itself is rounded by 2^-8.
typedef _Float16 Out16;
constexpr int kOutBlock = 64;
__device__ __forceinline__ uint32_t out16(float a, float b) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
}

template <class P, int RT, int CT, int MODE, typename YT, int TW = 1, bool WL = false, int AHEAD = 1>
__global__ __launch_bounds__(256 * TW, 2) void f8_tiled_kernel(TiledArgs a) {
    constexpr int M = P::M, kRows = TW * CT * M;  // activation rows of the workgroup
    constexpr int kCopies = CT * M / 32;          // copies of 1 KiB each wavefront makes for a block
    constexpr int kG = P::kGroups;
    static_assert(CT * M % 32 == 0 || kRows == 16, "copies are dealt to the wavefronts");
    constexpr int kWBytes = WL ? kTileWaves * RT * kKB : 16;
    static_assert(!WL || M == 32, "a tile in LDS is one of the matrix's");
    constexpr int kScaleRows = (kRows + 63) / 64 * 64;  // a copy fills 64
    // A variable to each stage: a read of one is then known not to wait for the
    // copies that are under way to another.
    __shared__ __attribute__((aligned(16))) uint8_t x0[kRows * 128], x1[kRows * 128], x2[AHEAD == 2 ? kRows * 128 : 16];
    __shared__ __attribute__((aligned(16))) uint8_t w0[kWBytes], w1[kWBytes];
    __shared__ __attribute__((aligned(16))) uint8_t out_lds[MODE != kGateUp && !WL ? TW * kTileWaves * M * 128 : 16];
    __shared__ float s0[kScaleRows], s1[kScaleRows], s2[AHEAD == 2 ? kScaleRows : 1], s_w[2][kF8MaxCols / 128];
    constexpr int kStages = AHEAD + 1;
    auto stage_x = [&](int u) { return u % kStages == 2 ? x2 : u % kStages ? x1 : x0; };
    auto stage_s = [&](int u) { return u % kStages == 2 ? s2 : u % kStages ? s1 : s0; };
    static_assert(!WL || AHEAD == 1, "two stages of weights in LDS");
    auto stage_w = [&](int u) { return u % 2 ? w1 : w0; };
    __shared__ float s_max[kTileWaves][MODE == kGateUp ? kRows : 1];
    const int tid = threadIdx.x, all_wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64;
    const int wave = all_wave % kTileWaves;  // which weight rows
    const uint32_t kb_n = a.d.kb;

    // which activation rows and weights
    uint32_t first, rows, rblock;
    const uint8_t *mat0, *mat1;  // of the first and second half of a wavefront's row tiles
    if constexpr (MODE == kDense) {
        // Neighbouring workgroups run on different XCDs: each XCD is dealt a
        // contiguous share of an order in which four blocks of activation rows
        // take turns, then the next block of weight rows, so that the 32
        // workgroups that an XCD runs at a time share both in its L2.
        const uint32_t rbs = (a.d.tiles * 32 + 4 * RT * M - 1) / (4 * RT * M), tbs = (a.xrows + kRows - 1) / kRows;
        const uint32_t per = gridDim.x / 8, id = (blockIdx.x % 8) * per + blockIdx.x / 8;
        const uint32_t four = id / (4 * rbs) * 4, left = tbs > four ? tbs - four : 0, turn = left < 4 ? left : 4;
        if (turn == 0) return;
        const uint32_t in = id - four * rbs;
        first = (four + in % turn) * kRows;
        rblock = in / turn;
        if (rblock >= rbs) return;
        if (first >= a.xrows) return;
        rows = a.xrows - first < kRows ? a.xrows - first : kRows;
        mat0 = mat1 = a.mat;
    } else {
        // Neighbouring workgroups run on different XCDs: the blocks of weight
        // rows of one tile, which share its activation rows, are given to one,
        // and with them those of a neighbouring tile, which is often the same
        // expert's and finds its weights in that XCD's L2.
        const uint32_t in = blockIdx.x / 8, tile = in / a.rblocks / 2 * 16 + blockIdx.x % 8 * 2 + in % 2;
        const Tile t = a.tiles[tile];
        if (t.rows == 0) return;
        first = t.first;
        rows = t.rows;
        mat0 = MODE == kGateUp ? t.gate : t.down;
        mat1 = MODE == kGateUp ? t.up : t.down;
        rblock = in / 2 % a.rblocks;
    }
    // row tile r of weight wavefront w: its first row, and where it is (a tile
    // never spans two scale blocks; tiles past the matrix read its last and
    // store nothing)
    auto tile_row = [&](int w, int r) -> uint32_t {
        if constexpr (MODE == kGateUp) return ((rblock * kTileWaves + w) * (RT / 2) + r % (RT / 2)) * M;
        else return ((rblock * kTileWaves + w) * RT + r) * M;
    };
    auto tile_mat = [&](int r) { return MODE == kGateUp && r >= RT / 2 ? mat1 : mat0; };
    auto tile_index = [&](uint32_t row) { return row / 32 < a.d.tiles ? row / 32 : a.d.tiles - 1; };
    global_u8 *base[RT];  // of this wavefront's tiles; with WL, of the ones that it copies
    uint32_t wrow[RT];
    int sub[RT];
    constexpr int kWMine = WL ? RT / TW : RT;
    Desc dw[kWMine];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        wrow[r] = tile_row(wave, r);
        sub[r] = (int)(wrow[r] / 16 & 1);
    }
#pragma unroll
    for (int i = 0; i < kWMine; ++i) {
        const int q = WL ? all_wave * kWMine + i : i, w = WL ? q / RT : wave, r = WL ? q % RT : i;
        base[i] = (global_u8 *)tile_mat(r) + (size_t)tile_index(tile_row(w, r)) * kb_n * kKB;
        if constexpr (WL) dw[i] = make_desc(tile_mat(r) + (size_t)tile_index(tile_row(w, r)) * kb_n * kKB, kb_n * kKB);
    }
    // The weights' scales, for the whole of K: gate's and up's, or those of the
    // two scale blocks that the workgroup's rows span.
    constexpr int kSetRows = MODE == kGateUp ? 0 : 128;
    auto scale_set = [&](int r) { return MODE == kGateUp ? (r < RT / 2 ? 0 : 1) : (int)((wave * RT + r) * M / 128); };
    // Asked for here, before the first block's copies, and kept when those are
    // under way.
    constexpr int kScaleLoads = 2 * (kF8MaxCols / 128) / (256 * TW);
    float w_scale[kScaleLoads];
#pragma unroll
    for (int j = 0; j < kScaleLoads; ++j) {
        const uint32_t i = j * 256 * TW + tid, set = i < kb_n ? 0 : 1, block = i - set * kb_n, row = tile_row(0, 0) + set * kSetRows;
        if (i < 2 * kb_n)
            w_scale[j] = ((global_f32 *)((set ? tile_mat(RT - 1) : tile_mat(0)) + f8_tile_bytes(a.d)))[(size_t)(tile_index(row) / 4) * kb_n + block];
    }
    auto keep_scales = [&] {
#pragma unroll
        for (int j = 0; j < kScaleLoads; ++j) {
            const uint32_t i = j * 256 * TW + tid, set = i < kb_n ? 0 : 1;
            if (i < 2 * kb_n) s_w[set][i - set * kb_n] = w_scale[j];
        }
    };
    // this wavefront's activation rows: with two sets of four, each takes half
    uint32_t row0 = 0, mine = rows;
    if constexpr (TW == 2) {
        const uint32_t half = ((rows + 1) / 2 + M - 1) / M * M;
        row0 = all_wave / kTileWaves ? half : 0;
        mine = row0 ? (rows > half ? rows - half : 0) : (rows < half ? rows : half);
    }
    // activation rows: what this lane copies, and whose scale it applies
    auto source_row = [&](uint32_t local) -> uint32_t {
        const uint32_t p = first + (local < rows ? local : rows - 1);
        if constexpr (MODE == kGateUp) return (uint32_t)a.row_of_pos[p];
        else return p;
    };
    uint32_t xbase = 0;
    if constexpr (MODE != kGateUp) xbase = first;
    // (f8_matmul and f8_experts keep the bytes of a call's rows below 2^32)
    const uint32_t xblock = a.xrows * 128;
    const Desc dx = make_desc(a.xq + (size_t)xbase * 128, kb_n * xblock - xbase * 128);
    // (where there are fewer copies than wavefronts, several make the same one:
    // a branch would split the K loop)
    constexpr int kMine = kCopies ? kCopies : 1;
    uint32_t voff[kMine];
    int at[kMine];
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
        at[j] = (all_wave * kMine + j) * 8 % kRows;
        const int local = at[j] + l / 8;
        voff[j] = (source_row((uint32_t)local) - xbase) * 128 + (uint32_t)(((l & 7) ^ swizzle(local)) * 16);
    }
    const int scale0 = all_wave * 64 % kScaleRows;
    const uint32_t srow = source_row((uint32_t)(scale0 + l)) * 4;
    const Desc ds = make_desc(a.xs, 0xFFFFFFFFu);
    uint32_t boff[P::kLoads];
#pragma unroll
    for (int j = 0; j < P::kLoads; ++j) boff[j] = P::b_row(l) * 128 + ((P::b_chunk(l, j) ^ swizzle(P::b_row(l))) * 16);

    typename P::D acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[r][c] = typename P::D{};

    // The K loop over N of the CT tiles of activation rows (an expert's rows may
    // fill fewer).  Blocks are asked for AHEAD steps before they are computed
    // (past the end the last one again, so that no branch splits the loop): two
    // where the registers hold another block of weights, for a step is as long as
    // a trip to memory if nothing else fills it (both kernels of 512 tokens of
    // experts on the fp8 cores: 177 us with one, 162 with two).  Scales go through LDS
    // too: in registers they would have to be waited for with the blocks asked
    // for after them.
    auto k_loop = [&](auto tiles_used) {
        constexpr int N = decltype(tiles_used)::value;
        typename P::Raw b[kStages][WL ? 1 : RT];  // weights in registers
        // kept in a scalar register: a copy whose offset the compiler put in a
        // vector register would be wrapped in a loop over its values
        const uint32_t last = kb_n - 1;
        auto clamped = [&](uint32_t block) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)(block < last ? block : last)); };
        auto issue_x = [&](uint32_t block, int u) {
            const uint32_t kb = clamped(block);
#pragma unroll
            for (int j = 0; j < kMine; ++j) copy16(dx, voff[j], kb * xblock, stage_x(u) + at[j] * 128);
            copy4(ds, srow + kb * a.xrows * 4, 0, stage_s(u) + scale0);
        };
        auto issue_w = [&](uint32_t block, int u) {
            const uint32_t kb = clamped(block);
#pragma unroll
            for (int r = 0; r < kWMine; ++r)
#pragma unroll
                for (int j = 0; j < P::kLoads; ++j) {
                    if constexpr (WL) copy16(dw[r], l * 16, kb * kKB + j * 1024, stage_w(u) + (all_wave * kWMine + r) * kKB + j * 1024);
                    else b[u % kStages][r].q[j] = *reinterpret_cast<const global_u32x4 *>(base[r] + (size_t)kb * kKB + P::a_off(l, sub[r], j));
                }
        };
        // A wavefront issues in order, and an instruction of the matrix cores
        // waits there for the one before it: so the fmas that take a tile are
        // dealt out behind the matrix instructions of the next one.
        auto compute = [&](uint32_t kb, int u) {
            const uint8_t *st = stage_x(u) + row0 * 128;
            typename P::Op aw[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                if constexpr (WL) {
                    typename P::Raw raw;
#pragma unroll
                    for (int j = 0; j < P::kLoads; ++j)
                        raw.q[j] = *reinterpret_cast<const u32x4 *>(stage_w(u) + (wave * RT + r) * kKB + P::a_off(l, 0, j));
                    aw[r] = P::op(raw);
                } else {
                    aw[r] = P::op(b[u % kStages][r]);
                }
            }
            auto load_b = [&](int c) {
                typename P::Raw raw;
#pragma unroll
                for (int j = 0; j < P::kLoads; ++j) raw.q[j] = *reinterpret_cast<const u32x4 *>(st + c * M * 128 + boff[j]);
                return raw;
            };
            constexpr int kD = 4 * kG, kChunk = (kD + P::kParts - 1) / P::kParts;
            // chunk i of tile n's fmas
            auto add = [&](int n, const typename P::D &d, float scale, int i) {
#pragma unroll
                for (int v = i * kChunk; v < (i + 1) * kChunk && v < kD; ++v)
                    acc[n % RT][n / RT][v] = __builtin_fmaf(d[v], scale, acc[n % RT][n / RT][v]);
            };
            typename P::D d = {};
            float scale = 0.0f, sx[N], sw[RT];
            typename P::Raw raw = load_b(0);
#pragma unroll
            for (int c = 0; c < N; ++c) sx[c] = stage_s(u)[row0 + c * M + P::b_row(l)];
#pragma unroll
            for (int r = 0; r < RT; ++r) sw[r] = s_w[scale_set(r)][kb];
#pragma unroll
            for (int c = 0; c < N; ++c) {
                const typename P::Op bx = P::op(raw);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const int n = c * RT + r;
                    typename P::D next = {};
#pragma unroll
                    for (int i = 0; i < P::kParts; ++i) {
                        next = P::part(aw[r], bx, next, i);
                        if (r == RT - 1 && i == 0 && c + 1 < N) raw = load_b(c + 1);
                        if constexpr (P::kParts == 2) __builtin_amdgcn_sched_barrier(0);
                        if (n) add(n - 1, d, scale, i);
                        if constexpr (P::kParts == 2) __builtin_amdgcn_sched_barrier(0);
                    }
                    d = next;
                    scale = sx[c] * sw[r];
                }
            }
#pragma unroll
            for (int i = 0; i < P::kParts; ++i) add(N * RT - 1, d, scale, i);
        };
        // The loads of a block, which may be under way when the one before is
        // needed.  (All are issued: what the loop asks for is used in it or after
        // it.  A count that is too large would let a copy be read too soon.)
        constexpr int kLoads = kMine + 1 + (WL ? kWMine : RT) * P::kLoads;
        auto step = [&](uint32_t kb, int u) {
            publish<(AHEAD - 1) * kLoads>();
            issue_x(kb + AHEAD, u + AHEAD);
            issue_w(kb + AHEAD, u + AHEAD);
            compute(kb, u);
        };
        issue_w(0, 0);  // first, as it needs no row_of_pos
        issue_x(0, 0);
        keep_scales();
        if constexpr (AHEAD == 2) {
            issue_x(1, 1);
            issue_w(1, 1);
        }
        uint32_t kb = 0;
        for (; kb + kStages <= kb_n; kb += kStages) {
#pragma unroll
            for (int u = 0; u < kStages; ++u) step(kb + u, u);
        }
        // the blocks that are left are all under way
        publish<0>();
#pragma unroll
        for (int u = 0; u < kStages - 1; ++u)
            if (kb + u < kb_n) compute(kb + u, u);
        publish<0>();  // no copy is under way when the workgroup's LDS goes to another
    };
    if constexpr (MODE == kDense) {
        k_loop(std::integral_constant<int, CT>{});
    } else {
        const uint32_t n = (uint32_t)__builtin_amdgcn_readfirstlane((int)((mine + M - 1) / M));
        if (CT >= 6 && n >= 6) k_loop(std::integral_constant<int, CT < 6 ? CT : 6>{});
        else if (CT >= 5 && n >= 5) k_loop(std::integral_constant<int, CT < 5 ? CT : 5>{});
        else if (CT >= 4 && n >= 4) k_loop(std::integral_constant<int, CT < 4 ? CT : 4>{});
        else if (CT >= 3 && n >= 3) k_loop(std::integral_constant<int, CT < 3 ? CT : 3>{});
        else if (CT >= 2 && n >= 2) k_loop(std::integral_constant<int, CT < 2 ? CT : 2>{});
        else k_loop(std::integral_constant<int, 1>{});
    }

    // Results go to memory through LDS (the stages are free now): a lane has a
    // few columns of one row, and stored from there every lane's would be a cache
    // access of its own; passed through LDS, neighbouring lanes store neighbouring
    // 16 bytes.  Chunks are permuted by the row as the activations' are.
    if constexpr (MODE == kGateUp) {
        // h = silu(g) u, quantised: the workgroup's 128 columns are one block
        constexpr int HT = RT / 2;
        float h[HT][CT][4 * kG];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            float m = 0.0f;
#pragma unroll
            for (int r = 0; r < HT; ++r)
#pragma unroll
                for (int i = 0; i < 4 * kG; ++i) {
                    const float g = acc[r][c][i];
                    h[r][c][i] = g * __builtin_amdgcn_rcpf(1.0f + __expf(-g)) * acc[r + HT][c][i];
                    m = fmaxf(m, fabsf(h[r][c][i]));
                }
            m = P::across(m);
            if (l < M && (uint32_t)(c * M + l) < mine) s_max[wave][row0 + c * M + l] = m;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const uint32_t in = (uint32_t)(c * M + P::b_row(l)), local = row0 + in;
            if (in >= mine) continue;
            const float m = fmaxf(fmaxf(s_max[0][local], s_max[1][local]), fmaxf(s_max[2][local], s_max[3][local]));
            const F8Factors f = f8_factors(m);
            const uint32_t pos = first + local;
            if (wave == 0 && l < M) a.hs[(size_t)rblock * a.hrows + pos] = f.scale;
#pragma unroll
            for (int r = 0; r < HT; ++r)
#pragma unroll
                for (int g = 0; g < kG; ++g) {
                    const float *v = &h[r][c][4 * g];
                    const uint32_t byte = wrow[r] % 128 + P::row(l, g);
                    *reinterpret_cast<uint32_t *>(x0 + local * 128 + ((byte / 16 ^ (local & 7)) * 16) + byte % 16) =
                        f8_pack4(v[0] * f.inv, v[1] * f.inv, v[2] * f.inv, v[3] * f.inv);
                }
        }
        __syncthreads();
        for (uint32_t i = tid; i < rows * 8; i += 256 * TW)
            reinterpret_cast<u32x4 *>(a.hq + ((size_t)rblock * a.hrows + first) * 128)[i] =
                *reinterpret_cast<const u32x4 *>(x0 + i / 8 * 128 + ((i ^ i / 8) & 7) * 16);
    } else {
        constexpr bool kOut16 = std::is_same<YT, Out16>::value;
        static_assert(!kOut16 || (MODE == kDown && RT * M == kOutBlock), "a wavefront's columns share a scale");
        YT *y = MODE == kDense ? static_cast<YT *>(a.y) : static_cast<YT *>(a.out);
        const uint32_t blocks = (a.d.rows + kOutBlock - 1) / kOutBlock, n = kOut16 ? blocks * kOutBlock : a.d.rows;
        // M rows of this wavefront's at a time, a line (128 bytes, or what the
        // wavefront has) of each
        constexpr int kEach = 16 / sizeof(YT), kFit = 128 / (M * (int)sizeof(YT)), kTiles = RT < kFit ? RT : kFit;
        constexpr int kLine = kTiles * M * (int)sizeof(YT), kChunks = kLine / 16;
        uint8_t *mine_lds = (WL ? w0 : out_lds) + all_wave * M * 128;
        const int row = P::b_row(l);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            if ((uint32_t)(c * M) >= mine) break;
            float inv = 0.0f;
            if constexpr (kOut16) {
                float m = 0.0f;
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int i = 0; i < 4 * kG; ++i) {
                        const float v = fabsf(acc[r][c][i]);
                        m = fmaxf(m, v < __builtin_inff() ? v : 0.0f);
                    }
                m = P::across(m);
                // 2^e <= m, but no less than 2^-100: 2^(14 - e) stays finite, and an
                // infinity beside zeros an infinity
                const uint32_t p = __float_as_uint(fmaxf(m, 0x1p-100f)) & 0x7F800000u;
                inv = __uint_as_float((268u << 23) - p);  // 2^(14 - e)
                const uint32_t in = (uint32_t)(c * M + row);
                if (l < M && in < mine && wrow[0] < n)
                    a.out_scales[(size_t)(first + row0 + in) * blocks + wrow[0] / kOutBlock] = __uint_as_float(p) * 0x1p-14f;
            }
#pragma unroll
            for (int r0 = 0; r0 < RT; r0 += kTiles) {
#pragma unroll
                for (int r = 0; r < kTiles; ++r)
#pragma unroll
                    for (int g = 0; g < kG; ++g) {
                        const int byte = (r * M + P::row(l, g)) * (int)sizeof(YT);
                        const f32x4 v = {acc[r0 + r][c][4 * g], acc[r0 + r][c][4 * g + 1], acc[r0 + r][c][4 * g + 2], acc[r0 + r][c][4 * g + 3]};
                        YT *to = reinterpret_cast<YT *>(mine_lds + row * kLine + ((byte / 16 ^ row) & (kChunks - 1)) * 16 + byte % 16);
                        if constexpr (kOut16) *reinterpret_cast<uint2 *>(to) = make_uint2(out16(v[0] * inv, v[1] * inv), out16(v[2] * inv, v[3] * inv));
                        else store4(static_cast<YT *>(__builtin_assume_aligned(to, 4 * sizeof(YT))), 4, v);
                    }
#pragma unroll
                for (int j = 0; j < M * kChunks / 64; ++j) {
                    const int at = (j * 64 + l) / kChunks, chunk = l % kChunks;
                    const u32x4 v = *reinterpret_cast<const u32x4 *>(mine_lds + at * kLine + ((chunk ^ at) & (kChunks - 1)) * 16);
                    const uint32_t in = (uint32_t)(c * M + at), col = wrow[r0] + chunk * kEach;
                    if (in >= mine || col >= n) continue;
                    YT *to = y + (size_t)(first + row0 + in) * n + col;
                    if (col + kEach <= n) {
                        __builtin_memcpy(to, &v, 16);
                    } else {
                        YT each[kEach];
                        __builtin_memcpy(each, &v, 16);
#pragma unroll
                        for (int k = 0; k < kEach; ++k)
                            if (col + k < n) to[k] = each[k];
                    }
                }
            }
        }
    }
}

// ---- few rows: the weight stream ----------------------------------------------
// Up to 16 rows against one matrix in one launch.  Every workgroup quantises
// the rows into LDS (they are few), then its wavefronts walk the weights: with
// SPLIT, the eight wavefronts share a tile's K blocks and add their parts in
// LDS in wavefront order; without, each walks tiles of its own.  SUB: 16-row
// subtiles of a tile that a wavefront takes.
constexpr int kRowsMax = 16;
constexpr int kRowsWaves = 8;
constexpr int kRowsThreads = kRowsWaves * 64;
struct RowsLayout {
    uint32_t stride;  // bytes of a quantised row: 16 more than its values, so that rows start in different banks
    uint32_t scales, red, total;
};
__host__ __device__ inline RowsLayout rows_layout(uint32_t t, uint32_t kb) {
    RowsLayout L;
    L.stride = kb * 128 + 16;
    L.scales = t * L.stride;
    L.red = (L.scales + t * kb * 4 + 15) & ~15u;
    L.total = L.red + kRowsWaves * 2 * 1024;
    return L;
}
constexpr uint32_t kRowsLds = 128u << 10;

template <int SUB, bool SPLIT, typename XT, typename YT>
__global__ __launch_bounds__(kRowsThreads) void f8_rows_kernel(const uint8_t *__restrict__ mat, F8Shape d,
                                                               const XT *__restrict__ x, uint32_t t, YT *__restrict__ y) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    typedef Bf16x16 P;
    const RowsLayout L = rows_layout(t, d.kb);
    float *xs = reinterpret_cast<float *>(lds + L.scales);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64;
    for (uint32_t i = tid; i < t * d.kb * 8; i += kRowsThreads) {
        const uint32_t row = i / (8 * d.kb), c = i - row * 8 * d.kb, k = c * 16;
        float v[16], s;
        load_row<16>(x + (size_t)row * d.cols + k, k < d.cols ? (int)(d.cols - k) : 0, v);
        *reinterpret_cast<u32x4 *>(lds + row * L.stride + k) = quantize16(v, &s);
        if ((c & 7) == 0) xs[row * d.kb + (c >> 3)] = s;
    }
    __syncthreads();

    const uint32_t token = (uint32_t)P::b_row(l) < t ? (uint32_t)P::b_row(l) : t - 1;
    const uint8_t *bx = lds + token * L.stride + (l >> 4) * 16;
    const float *sx = xs + token * d.kb;
    const float *scales = reinterpret_cast<const float *>(mat + f8_tile_bytes(d));
    const uint32_t units = (d.rows + 16 * SUB - 1) / (16 * SUB);
    const uint32_t u0 = SPLIT ? blockIdx.x : blockIdx.x * kRowsWaves + wave, ustep = SPLIT ? gridDim.x : gridDim.x * kRowsWaves;
    for (uint32_t u = u0; u < units; u += ustep) {
        const uint32_t row0 = u * 16 * SUB, tile = row0 / 32;
        const uint8_t *w = mat + (size_t)tile * d.kb * kKB;
        const float *ws = scales + (size_t)(tile / 4) * d.kb;
        const int s0 = (int)(row0 / 16 & 1);
        f32x4 acc[SUB] = {};
        constexpr int kAhead = 4;  // K blocks in flight
        for (uint32_t b0 = SPLIT ? wave : 0; b0 < d.kb; b0 += kAhead * (SPLIT ? kRowsWaves : 1)) {
            typename P::Raw raw[kAhead][SUB];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const uint32_t kb = b0 + i * (SPLIT ? kRowsWaves : 1);
                if (kb >= d.kb) break;
#pragma unroll
                for (int s = 0; s < SUB; ++s)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        raw[i][s].q[j] = *reinterpret_cast<const u32x4 *>(w + (size_t)kb * kKB + P::a_off(l, s0 + s, j));
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const uint32_t kb = b0 + i * (SPLIT ? kRowsWaves : 1);
                if (kb >= d.kb) break;
                typename P::Raw rb;
                rb.q[0] = *reinterpret_cast<const u32x4 *>(bx + kb * 128);
                rb.q[1] = *reinterpret_cast<const u32x4 *>(bx + kb * 128 + 64);
                const typename P::Op b = P::op(rb);
                const float sc = sx[kb] * ws[kb];
#pragma unroll
                for (int s = 0; s < SUB; ++s) {
                    const f32x4 p = P::mma(P::op(raw[i][s]), b);
#pragma unroll
                    for (int v = 0; v < 4; ++v) acc[s][v] = __builtin_fmaf(p[v], sc, acc[s][v]);
                }
            }
        }
        if constexpr (SPLIT) {
            f32x4 *red = reinterpret_cast<f32x4 *>(lds + L.red);
#pragma unroll
            for (int s = 0; s < SUB; ++s) red[(wave * SUB + s) * 64 + l] = acc[s];
            __syncthreads();
            if (wave < SUB) {
                f32x4 v = red[wave * 64 + l];
#pragma unroll
                for (int i = 1; i < kRowsWaves; ++i) v += red[(i * SUB + wave) * 64 + l];
                const uint32_t col = row0 + wave * 16 + P::row(l, 0);
                if ((uint32_t)P::b_row(l) < t && col < d.rows)
                    store4(y + (size_t)P::b_row(l) * d.rows + col, (int)(d.rows - col), v);
            }
            __syncthreads();
        } else {
#pragma unroll
            for (int s = 0; s < SUB; ++s) {
                const uint32_t col = row0 + s * 16 + P::row(l, 0);
                if ((uint32_t)P::b_row(l) < t && col < d.rows)
                    store4(y + (size_t)P::b_row(l) * d.rows + col, (int)(d.rows - col), acc[s]);
            }
        }
    }
}

// Compute units of the current device (asked for once).
int cu_count() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess) return 256;
    if (dev >= 0 && dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) return 256;
    if (dev >= 0 && dev < 64) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

template <typename XT, typename YT>
hipError_t launch_rows(hipStream_t s, const uint8_t *mat, const F8Shape &d, const XT *x, uint32_t t, YT *y) {
    const uint32_t lds = rows_layout(t, d.kb).total, cus = (uint32_t)cu_count();
    const uint32_t per_cu = lds <= (72u << 10) ? 2 : 1;  // workgroups that fit a compute unit's LDS
    const uint32_t tiles = (d.rows + 31) / 32, slots = cus * per_cu;
    auto launch = [&](auto kernel, uint32_t grid) {
        // more than 64 KiB of LDS is asked for by name
        if (lds > (64u << 10)) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        kernel<<<grid, kRowsThreads, lds, s>>>(mat, d, x, t, y);
        return hipGetLastError();
    };
    if (tiles >= slots * kRowsWaves) return launch(f8_rows_kernel<2, false, XT, YT>, slots);
    if (tiles >= cus) return launch(f8_rows_kernel<2, true, XT, YT>, tiles < slots ? tiles : slots);
    const uint32_t units = (d.rows + 15) / 16;
    return launch(f8_rows_kernel<1, true, XT, YT>, units < slots ? units : slots);
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
bool rows_path(const F8Shape &d, uint32_t t) { return t <= kRowsMax && rows_layout(t, d.kb).total <= kRowsLds; }

// ---- a few hundred rows: K split over the wavefronts -----------------------------
// Where the tiles of the product above would leave most compute units without
// work.  A workgroup takes one tile of 32 weight rows by 32 NT activation rows;
// its eight wavefronts take the K blocks in turn, straight from memory to
// registers (both operands lie as the instructions take them), a block ahead,
// and add their sums in LDS, pairwise.
constexpr int kSplitWaves = 8;

template <class P, int NT, typename YT>
__global__ __launch_bounds__(64 * kSplitWaves) void f8_split_kernel(const uint8_t *__restrict__ mat, F8Shape d,
                                                                    const uint8_t *__restrict__ xq, const float *__restrict__ xs,
                                                                    uint32_t t, YT *__restrict__ y) {
    constexpr int M = P::M, RT = 32 / M, CT = 32 * NT / M, kG = P::kGroups, kQuads = RT * CT * kG;
    __shared__ f32x4 red[kSplitWaves][kQuads][64];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64;
    // neighbouring workgroups run on different XCDs: those of one tile of weights
    // are given to one
    const uint32_t chunks = (t + 32 * NT - 1) / (32 * NT), in = blockIdx.x / 8, tile = in / chunks * 8 + blockIdx.x % 8;
    const uint32_t t0 = in % chunks * 32 * NT, t_tiles = pad32(t) / 32;
    if (tile * 32 >= d.rows) return;
    const uint8_t *w = mat + (size_t)tile * d.kb * kKB;
    const float *ws = reinterpret_cast<const float *>(mat + f8_tile_bytes(d)) + (size_t)(tile / 4) * d.kb;
    uint32_t x_tile[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) x_tile[n] = t0 / 32 + n < t_tiles ? t0 / 32 + n : t_tiles - 1;

    typename P::D acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[r][c] = typename P::D{};
    typename P::Raw a[2][RT], b[2][CT];
    float sx[2][CT], sw[2];
    auto ask = [&](uint32_t block, int u) {
        const uint32_t kb = block < d.kb ? block : d.kb - 1;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int j = 0; j < P::kLoads; ++j) a[u][r].q[j] = *reinterpret_cast<const u32x4 *>(w + (size_t)kb * kKB + P::a_off(l, r, j));
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const size_t at = (size_t)kb * t_tiles + x_tile[c * M / 32];
#pragma unroll
            for (int j = 0; j < P::kLoads; ++j) b[u][c].q[j] = *reinterpret_cast<const u32x4 *>(xq + at * kKB + P::a_off(l, c % RT, j));
            sx[u][c] = xs[at * 32 + c % RT * M + P::b_row(l)];
        }
        sw[u] = ws[kb];
    };
    auto compute = [&](int u) {
        typename P::Op aw[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) aw[r] = P::op(a[u][r]);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const typename P::Op bx = P::op(b[u][c]);
            const float scale = sx[u][c] * sw[u];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                typename P::D p = {};
#pragma unroll
                for (int i = 0; i < P::kParts; ++i) p = P::part(aw[r], bx, p, i);
#pragma unroll
                for (int v = 0; v < 4 * kG; ++v) acc[r][c][v] = __builtin_fmaf(p[v], scale, acc[r][c][v]);
            }
        }
    };
    ask(wave, 0);
    for (uint32_t kb = wave; kb < d.kb; kb += 2 * kSplitWaves) {
        ask(kb + kSplitWaves, 1);
        __builtin_amdgcn_sched_barrier(0);
        compute(0);
        ask(kb + 2 * kSplitWaves, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (kb + kSplitWaves < d.kb) compute(1);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int g = 0; g < kG; ++g)
                red[wave][(r * CT + c) * kG + g][l] = f32x4{acc[r][c][4 * g], acc[r][c][4 * g + 1], acc[r][c][4 * g + 2], acc[r][c][4 * g + 3]};
    __syncthreads();
    for (int q = wave; q < kQuads; q += kSplitWaves) {
        const int g = q % kG, c = q / kG % CT, r = q / kG / CT;
        auto two = [&](int i) { return red[i][q][l] + red[i + 4][q][l]; };
        const f32x4 v = (two(0) + two(2)) + (two(1) + two(3));
        const uint32_t row = t0 + c * M + P::b_row(l), col = tile * 32 + r * M + P::row(l, g);
        if (row < t && col < d.rows) store4(y + (size_t)row * d.rows + col, (int)(d.rows - col), v);
    }
}

template <bool TILED, typename XT>
hipError_t quantize(hipStream_t s, const XT *x, uint32_t t, uint32_t cols, uint32_t kb, uint8_t *xq, float *xs) {
    f8_quantize_kernel<TILED><<<(quantize_chunks(t, kb) + 255) / 256, 256, 0, s>>>(x, t, cols, kb, xq, xs);
    return hipGetLastError();
}

template <class P, int RT, int CT, int AHEAD, typename YT, int TW = 1, bool WL = false>
hipError_t launch_dense(hipStream_t s, const TiledArgs &a) {
    constexpr uint32_t kM = P::M;
    const uint32_t rbs = (a.d.tiles * 32 + 4 * RT * kM - 1) / (4 * RT * kM), tbs = (a.xrows + TW * CT * kM - 1) / (TW * CT * kM);
    f8_tiled_kernel<P, RT, CT, kDense, YT, TW, WL, AHEAD><<<(rbs * tbs + 7) / 8 * 8, 256 * TW, 0, s>>>(a);
    return hipGetLastError();
}

template <class P, int NT, typename YT>
hipError_t launch_split(hipStream_t s, const uint8_t *mat, const F8Shape &d, const uint8_t *xq, const float *xs, uint32_t t, YT *y) {
    const uint32_t tiles = (d.rows + 31) / 32, chunks = (t + 32 * NT - 1) / (32 * NT);
    f8_split_kernel<P, NT, YT><<<(tiles + 7) / 8 * 8 * chunks, 64 * kSplitWaves, 0, s>>>(mat, d, xq, xs, t, y);
    return hipGetLastError();
}

// A workgroup's activation rows where K is split; 0: the tiled product is faster,
// as it is once its larger tiles (which load less for a product) fill the card.
// us, split / tiled: 64 bf16 rows of 4096 by 8192 12.2 / 26, 256 26.5 / 50, 512
// (1024 workgroups, four to a compute unit) 45 / 45, 1024 88 / 45, 256 by 20000
// (1250) 59 / 53; f32 rows of the same by 8192, 64 rows 13 / 32, 512 56 / 41.  The
// bf16 instructions take 32 rows always (256 rows 31, in steps of 64 33, of 128 40).
uint32_t split_rows(const F8Shape &d, uint32_t t, bool exact) {
    const uint32_t rows = exact || t <= 32 ? 32 : t <= 64 ? 64 : 128;
    return (uint64_t)((d.rows + 31) / 32) * ((t + rows - 1) / rows) <= 4u * (uint32_t)cu_count() ? rows : 0;
}

template <typename XT, typename YT>
hipError_t matmul(hipStream_t s, const uint8_t *mat, const F8Shape &d, const XT *x, uint32_t t, YT *y, void *scratch) {
    if (rows_path(d, t)) return launch_rows(s, mat, d, x, t, y);
    uint8_t *xq = static_cast<uint8_t *>(scratch);
    float *xs = reinterpret_cast<float *>(xq + align256((size_t)pad32(t) * d.kb * 128));
    constexpr bool kF32 = sizeof(YT) == 4;
    // up to 16 rows have exact products, also those that are too wide for a workgroup's LDS
    const bool exact = kF32 || t <= kRowsMax;
    if (const uint32_t rows = split_rows(d, t, exact)) {
        hipError_t e = quantize<true>(s, x, t, d.cols, d.kb, xq, xs);
        if (e != hipSuccess) return e;
        if (exact) return launch_split<Bf16x16, 1, YT>(s, mat, d, xq, xs, t, y);
        if constexpr (!kF32) {
            return rows == 32   ? launch_split<Fp8x32, 1, YT>(s, mat, d, xq, xs, t, y)
                   : rows == 64 ? launch_split<Fp8x32, 2, YT>(s, mat, d, xq, xs, t, y)
                                : launch_split<Fp8x32, 4, YT>(s, mat, d, xq, xs, t, y);
        }
    }
    hipError_t e = quantize<false>(s, x, t, d.cols, d.kb, xq, xs);
    if (e != hipSuccess) return e;
    TiledArgs a{};
    a.mat = mat;
    a.d = d;
    a.xq = xq;
    a.xs = xs;
    a.xrows = t;
    a.y = y;
    if constexpr (kF32) {
        return t <= 32 ? launch_dense<Bf16x16, 2, 2, 2, YT>(s, a) : launch_dense<Bf16x16, 2, 4, 2, YT>(s, a);
    } else {
        if (exact) return launch_dense<Bf16x16, 2, 2, 2, YT>(s, a);
        if (t <= 32) return launch_dense<Fp8x32, 1, 1, 2, YT>(s, a);
        if (t <= 64) return launch_dense<Fp8x32, 2, 2, 2, YT>(s, a);
        // Tiles of 256 rows where they leave little of the card without work in
        // their last round (a compute unit holds one), else of 64 where all run
        // at once (two to a unit), else of 96.  us for tiles of 64 / 96 / 256 rows:
        // 4096 by 8192, K 4096 172 / 160 / 143, 2048 by 6000 (0.73 of a round) 65 /
        // 78 / 60; 2048 by 4096 (0.5) 46 / 50 / 60, 1024 by 8192 45 / 48 / 55; 2560
        // by 8192, K 2048 (0.63 of two) 57 / 56 / 65.
        const uint64_t cus = (uint64_t)cu_count(), rbs = (d.rows + 255) / 256, rounds = (rbs * ((t + 255) / 256) + cus - 1) / cus;
        if ((uint64_t)d.rows * t * 10 >= rounds * 7 * cus * 256 * 256) return launch_dense<Fp8x32, 2, 4, 1, YT, 2, true>(s, a);
        return rbs * ((t + 63) / 64) <= 2 * cus ? launch_dense<Fp8x32, 2, 2, 2, YT>(s, a) : launch_dense<Fp8x32, 2, 3, 1, YT>(s, a);
    }
}

// ---- the routed experts ------------------------------------------------------
// Many pairs: `plan` sorts the (token, k) pairs by expert and cuts them into
// tiles of one expert each (and quantises x in the workgroups after its own);
// gate_up and down are the tiled product over those tiles; combine adds a
// token's weighted outputs in the order of its routes.  Few pairs: two launches
// that take every pair by itself.
struct ExpertsArgs {
    const uint16_t *ids;  // [t x top_k]
    const float *w;
    uint32_t t, top_k, n_experts;
    int32_t *status;
};
constexpr int kPlanThreads = 1024;
constexpr uint32_t kMaxF8Experts = 1024;

// Positions of the pairs p = t top_k + k, by expert.  Every workgroup counts all
// ids (in LDS: those of the pairs before its own 1024, and all of them) and so
// needs nothing from the others; within an expert its own pairs take places in
// the order in which their LDS atomics arrive, which no result depends on: a
// pair's column of a product is computed alike wherever it stands.  A tile is
// at most tile_m rows of one expert, an expert's tiles of equal size; those behind
// the last have no rows.  An id that names no expert makes *n_tiles -1 and leaves
// no tile with rows: the kernels after this one then do nothing.
template <typename XT>
__global__ __launch_bounds__(kPlanThreads) void f8_plan_kernel(ExpertsArgs a, uint32_t tile_m, int32_t *__restrict__ pos_of_pair,
                                                               int32_t *__restrict__ row_of_pos, Tile *__restrict__ tiles,
                                                               uint32_t max_tiles, const uint8_t *const *__restrict__ mats,
                                                               int32_t *__restrict__ n_tiles, const XT *__restrict__ x,
                                                               uint32_t hidden, uint32_t kb, uint8_t *__restrict__ xq,
                                                               float *__restrict__ xs) {
    const uint32_t pairs = a.t * a.top_k, plan_blocks = (pairs + kPlanThreads - 1) / kPlanThreads;
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    if (blockIdx.x >= plan_blocks) {
        const uint32_t i = (blockIdx.x - plan_blocks) * kPlanThreads + tid;
        quantize_chunk<false>(x, a.t, hidden, kb, i, xq, xs);
        return;
    }
    __shared__ int32_t before[kMaxF8Experts], total[kMaxF8Experts], place[kMaxF8Experts];
    __shared__ int32_t s_pairs[kPlanThreads / 64], s_tiles[kPlanThreads / 64];
    __shared__ int32_t s_bad;
    before[tid] = total[tid] = 0;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    const uint32_t b0 = blockIdx.x * kPlanThreads;
    for (uint32_t r = tid; r < pairs; r += 8 * kPlanThreads) {
        uint32_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = r + i * kPlanThreads < pairs ? a.ids[r + i * kPlanThreads] : TQF_HIP_NO_EXPERT;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (e[i] == TQF_HIP_NO_EXPERT) continue;
            if (e[i] >= a.n_experts) {
                s_bad = 1;
                continue;
            }
            atomicAdd(&total[e[i]], 1);
            if (r + i * kPlanThreads < b0) atomicAdd(&before[e[i]], 1);
        }
    }
    __syncthreads();
    if (s_bad) {
        if (blockIdx.x == 0) {
            for (uint32_t i = tid; i < max_tiles; i += kPlanThreads) tiles[i].rows = 0;
            if (tid == 0) {
                *n_tiles = -1;
                if (a.status) *a.status = TQF_HIP_ERR_INVALID;
            }
        }
        return;
    }
    // exclusive scans of pairs and tiles over the experts, one to a thread
    const int c = total[tid], n = (c + (int)tile_m - 1) / (int)tile_m;
    int sc = c, sn = n;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int u = __shfl_up(sc, o), v = __shfl_up(sn, o);
        if (lane >= o) {
            sc += u;
            sn += v;
        }
    }
    if (lane == 63) {
        s_pairs[wave] = sc;
        s_tiles[wave] = sn;
    }
    __syncthreads();
    int base = sc - c, tbase = sn - n;
    for (int i = 0; i < wave; ++i) {
        base += s_pairs[i];
        tbase += s_tiles[i];
    }
    place[tid] = base + before[tid];
    if (blockIdx.x == 0) {
        const int step = n ? (c + n - 1) / n : 0;
        for (int i = 0; i < n; ++i) {
            const int rows = c - i * step < step ? c - i * step : step;
            tiles[tbase + i] = Tile{(uint32_t)(base + i * step), (uint32_t)rows, mats[3 * tid], mats[3 * tid + 1], mats[3 * tid + 2]};
        }
        int all = 0;
#pragma unroll
        for (int i = 0; i < kPlanThreads / 64; ++i) all += s_tiles[i];
        for (uint32_t i = all + tid; i < max_tiles; i += kPlanThreads) tiles[i].rows = 0;
        if (tid == 0) *n_tiles = all;
    }
    __syncthreads();
    const uint32_t p = b0 + tid;
    if (p < pairs) {
        const uint32_t e = a.ids[p];
        int pos = -1;
        if (e != TQF_HIP_NO_EXPERT) {
            pos = atomicAdd(&place[e], 1);
            row_of_pos[pos] = (int32_t)(p / a.top_k);
        }
        pos_of_pair[p] = pos;
    }
}

template <typename YT>
__global__ __launch_bounds__(256) void f8_combine_kernel(ExpertsArgs a, const int32_t *__restrict__ pos_of_pair,
                                                         const int32_t *__restrict__ n_tiles, const float *__restrict__ out,
                                                         uint32_t hidden, YT *__restrict__ y) {
    if (*n_tiles < 0) return;
    const uint32_t t = blockIdx.y, h = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (h >= hidden) return;
    const int valid = (int)(hidden - h);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t k = 0; k < a.top_k; ++k) {
        const int pos = pos_of_pair[t * a.top_k + k];
        if (pos < 0) continue;
        const float w = a.w[t * a.top_k + k];
        float o[4];
        load_row<4>(out + (size_t)pos * hidden + h, valid, o);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(w, o[i], v[i]);
    }
    store4(y + (size_t)t * hidden + h, valid, v);
}

// The same from Out16: eight columns to a thread.
__global__ __launch_bounds__(256) void f8_combine16_kernel(ExpertsArgs a, const int32_t *__restrict__ pos_of_pair,
                                                           const int32_t *__restrict__ n_tiles, const Out16 *__restrict__ out,
                                                           const float *__restrict__ scales, uint32_t hidden,
                                                           uint16_t *__restrict__ y) {
    if (*n_tiles < 0) return;
    const uint32_t t = blockIdx.y, h = (blockIdx.x * 256 + threadIdx.x) * 8, blocks = (hidden + kOutBlock - 1) / kOutBlock;
    if (h >= hidden) return;
    float v[8] = {};
    for (uint32_t k = 0; k < a.top_k; ++k) {
        const int pos = pos_of_pair[t * a.top_k + k];
        if (pos < 0) continue;
        const u32x4 q = *reinterpret_cast<const u32x4 *>(out + (size_t)pos * blocks * kOutBlock + h);
        const float w = a.w[t * a.top_k + k], scale = scales[(size_t)pos * blocks + h / kOutBlock];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float o = (float)__builtin_bit_cast(_Float16, (uint16_t)(q[i / 2] >> i % 2 * 16)) * scale;
            v[i] = __builtin_fmaf(w, o, v[i]);
        }
    }
    const f32x4 lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
    uint16_t *to = y + (size_t)t * hidden + h;
    if (hidden - h >= 8) {
        const u32x4 b = {bf16_bits2(lo[0], lo[1]), bf16_bits2(lo[2], lo[3]), bf16_bits2(hi[0], hi[1]), bf16_bits2(hi[2], hi[3])};
        __builtin_memcpy(to, &b, 16);
    } else {
        store4(to, (int)(hidden - h), lo);
        store4(to + 4, (int)(hidden - h) - 4, hi);
    }
}

// Few pairs.  A pair's row is the only column of its products, so all 16
// columns of the operand are that row (one address for 16 lanes).  Down has a
// workgroup for each token and 16 columns, so many tokens of few routes are left
// to the tiles (us by pairs / by tiles: 16 tokens of 1 route 20.5 / 24.1, of 4
// 42 / 43, 32 of 1 35 / 31, 64 of 1 63 / 43, 8 of 8 39 / 46).
constexpr uint32_t kPairsMax = 64, kPairsTokens = 16;
constexpr uint32_t kPairsHidden = 8192, kPairsWidth = 2048;

// One trip to memory after another is what these two cost: id, table (or pointer),
// weights.  Loads return in the order they are issued, so all that does not wait
// for another load is asked for before the weights, which everything after them
// would have to wait for.

// Whether every id of the call names an expert or none (each wavefront asks; at
// most kPairsMax = 64 of them).
__device__ __forceinline__ uint32_t load_id(const ExpertsArgs &a, int lane) {
    return (uint32_t)lane < a.t * a.top_k ? a.ids[lane] : TQF_HIP_NO_EXPERT;
}
__device__ __forceinline__ bool ids_ok(const ExpertsArgs &a, uint32_t id) {
    return __ballot(id != TQF_HIP_NO_EXPERT && id >= a.n_experts) == 0;
}
// A row of n K blocks, of which this wavefront needs b0, b0 + step, ...: their
// values quantised to bf16 into q [kb][128] and their scales into s [kb].
// Sixteen lanes take a block, eight values each, four blocks at a time; those of
// the first four are asked for by load_blocks.
template <typename XT>
__device__ __forceinline__ void load_blocks(const XT *x, uint32_t cols, uint32_t b, uint32_t step, uint32_t n, int lane, float (&v)[8]) {
    const uint32_t kb = b + (lane / 16) * step, k = kb * 128 + (lane % 16) * 8;
    load_row<8>(x + k, kb < n && k < cols ? (int)(cols - k) : 0, v);
}
template <typename XT>
__device__ __forceinline__ void quantize_blocks(const XT *x, uint32_t cols, uint32_t b0, uint32_t step, uint32_t n, int lane,
                                                float (&v)[8], uint16_t *q, float *s) {
    for (uint32_t b = b0; b < n; b += 4 * step) {
        if (b != b0) load_blocks(x, cols, b, step, n, lane, v);
        const uint32_t kb = b + (lane / 16) * step, k = kb * 128 + (lane % 16) * 8;
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
        m = amax8(m);
        m = fmaxf(m, dpp_f<kDppMirror>(m));
        const F8Factors f = f8_factors(m);
        if (kb < n) {
            const uint32_t lo = f8_pack4(v[0] * f.inv, v[1] * f.inv, v[2] * f.inv, v[3] * f.inv);
            const uint32_t hi = f8_pack4(v[4] * f.inv, v[5] * f.inv, v[6] * f.inv, v[7] * f.inv);
            *reinterpret_cast<bf16x8 *>(q + k) = f8_widen(lo, hi);
            if (lane % 16 == 0) s[kb] = f.scale;
        }
    }
}
// This lane's operand of K block kb of a row in LDS.
__device__ __forceinline__ Bf16x16::Op pair_operand(const uint16_t *q, uint32_t kb, int lane) {
    const bf16x8 *p = reinterpret_cast<const bf16x8 *>(q + kb * 128 + (lane >> 4) * 16);
    return Bf16x16::Op{{p[0], p[1], p[8], p[9]}};
}

// h[pair] = silu(g) u for 16 columns; four wavefronts share the K blocks.
template <typename XT>
__global__ __launch_bounds__(256) void f8_pair_gate_up_kernel(ExpertsArgs a, const uint8_t *const *__restrict__ mats, F8Shape d,
                                                              const XT *__restrict__ x, float *__restrict__ h, uint32_t hstride,
                                                              const uint8_t **__restrict__ downs) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    typedef Bf16x16 P;
    uint16_t *q = reinterpret_cast<uint16_t *>(lds);
    float *s = reinterpret_cast<float *>(lds + (size_t)d.kb * 256);
    float *red = s + ((d.kb + 3) & ~3u);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64;
    const uint32_t pair = blockIdx.y, e = a.ids[pair], row0 = blockIdx.x * 16;
    const XT *row = x + (size_t)(pair / a.top_k) * d.cols;
    const uint32_t id = load_id(a, l);
    float xv[8];
    load_blocks(row, d.cols, wave, 4, d.kb, l, xv);
    __builtin_amdgcn_sched_barrier(0);
    // An id out of range reads expert 0's matrices until all ids are seen; down
    // finds its matrix without the table.
    const bool named = e < a.n_experts;
    const size_t m0 = (size_t)(named ? e : 0) * 3;
    if (blockIdx.x == 0 && tid == 0) downs[pair] = named ? mats[m0 + 2] : nullptr;
    if (e == TQF_HIP_NO_EXPERT) return;  // (a bad id is reported by its own pair among others)
    global_u8 *g = (global_u8 *)mats[m0], *u = (global_u8 *)mats[m0 + 1];
    const uint32_t tile = row0 / 32;
    const int sub = (int)(row0 / 16 & 1);
    const size_t base = (size_t)tile * d.kb * kKB, sbase = f8_tile_bytes(d) + (size_t)(tile / 4) * d.kb * 4;
    global_f32 *gs = (global_f32 *)(g + sbase), *us = (global_f32 *)(u + sbase);
    f32x4 ag = {0.0f, 0.0f, 0.0f, 0.0f}, au = ag;
    constexpr int kAhead = 4;
    typename P::Raw rg[kAhead], ru[kAhead];
    float sg[kAhead], su[kAhead];
    auto issue = [&](uint32_t b0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const uint32_t kb = b0 + 4 * i;
            if (kb >= d.kb) break;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const size_t at = base + (size_t)kb * kKB + P::a_off(l, sub, j);
                rg[i].q[j] = *reinterpret_cast<const global_u32x4 *>(g + at);
                ru[i].q[j] = *reinterpret_cast<const global_u32x4 *>(u + at);
            }
            sg[i] = gs[kb];
            su[i] = us[kb];
        }
    };
    issue(wave);
    if (!ids_ok(a, id)) {
        if (blockIdx.x == 0 && tid == 0 && a.status) *a.status = TQF_HIP_ERR_INVALID;
        return;
    }
    quantize_blocks(row, d.cols, wave, 4, d.kb, l, xv, q, s);
    __syncthreads();
    for (uint32_t b0 = wave; b0 < d.kb; b0 += 4 * kAhead) {
        if (b0 != (uint32_t)wave) issue(b0);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const uint32_t kb = b0 + 4 * i;
            if (kb >= d.kb) break;
            const typename P::Op b = pair_operand(q, kb, l);
            const f32x4 pg = P::mma(P::op(rg[i]), b), pu = P::mma(P::op(ru[i]), b);
            const float gscale = s[kb] * sg[i], uscale = s[kb] * su[i];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                ag[v] = __builtin_fmaf(pg[v], gscale, ag[v]);
                au[v] = __builtin_fmaf(pu[v], uscale, au[v]);
            }
        }
    }
    if ((l & 15) == 0) {
        *reinterpret_cast<f32x4 *>(red + wave * 32 + P::row(l, 0)) = ag;
        *reinterpret_cast<f32x4 *>(red + wave * 32 + 16 + P::row(l, 0)) = au;
    }
    __syncthreads();
    if (tid < 16 && row0 + tid < d.rows) {
        const float gv = (red[tid] + red[32 + tid]) + (red[64 + tid] + red[96 + tid]);
        const float uv = (red[16 + tid] + red[48 + tid]) + (red[80 + tid] + red[112 + tid]);
        h[(size_t)pair * hstride + row0 + tid] = gv / (1.0f + expf(-gv)) * uv;
    }
}

// y[token] for 16 columns: a wavefront takes the routes k = wave, wave + 8, ...
// downs: the matrix of each pair, null for an empty slot.
template <typename YT>
__global__ __launch_bounds__(512) void f8_pair_down_kernel(ExpertsArgs a, const uint8_t *const *__restrict__ downs, F8Shape d,
                                                           const float *__restrict__ h, uint32_t hstride, YT *__restrict__ y) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float weight[TQF_HIP_ROUTE_MAX_TOP_K];
    __shared__ bool used[TQF_HIP_ROUTE_MAX_TOP_K];
    typedef Bf16x16 P;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64;
    uint16_t *q = reinterpret_cast<uint16_t *>(lds + (size_t)wave * d.kb * 256);
    float *s = reinterpret_cast<float *>(lds + (size_t)8 * d.kb * 256) + wave * d.kb;
    float *red = reinterpret_cast<float *>(lds + (size_t)8 * d.kb * 260);  // [top_k][16]
    const uint32_t token = blockIdx.y, row0 = blockIdx.x * 16, tile = row0 / 32;
    const int sub = (int)(row0 / 16 & 1);
    const size_t base = (size_t)tile * d.kb * kKB, sbase = f8_tile_bytes(d) + (size_t)(tile / 4) * d.kb * 4;
    const uint32_t id = load_id(a, l);
    for (uint32_t k = wave; k < a.top_k; k += 8) {
        const uint32_t pair = token * a.top_k + k;
        const float *row = h + (size_t)pair * hstride;
        const float w = a.w[pair];
        float hv[8];
        load_blocks(row, d.cols, 0, 1, d.kb, l, hv);
        __builtin_amdgcn_sched_barrier(0);
        global_u8 *m = (global_u8 *)downs[pair];
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        if (m) {
            global_f32 *ms = (global_f32 *)(m + sbase);
            constexpr int kAhead = 4;
            typename P::Raw raw[kAhead];
            float sm[kAhead];
            auto issue = [&](uint32_t b0) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (b0 + i >= d.kb) break;
                    sm[i] = ms[b0 + i];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        raw[i].q[j] = *reinterpret_cast<const global_u32x4 *>(m + base + (size_t)(b0 + i) * kKB + P::a_off(l, sub, j));
                }
            };
            issue(0);
            quantize_blocks(row, d.cols, 0, 1, d.kb, l, hv, q, s);
            // this wavefront's own writes: LDS serves it in order
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (uint32_t b0 = 0; b0 < d.kb; b0 += kAhead) {
                if (b0) issue(b0);
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (b0 + i >= d.kb) break;
                    const f32x4 p = P::mma(P::op(raw[i]), pair_operand(q, b0 + i, l));
                    const float sc = s[b0 + i] * sm[i];
#pragma unroll
                    for (int v = 0; v < 4; ++v) acc[v] = __builtin_fmaf(p[v], sc, acc[v]);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // before the next route's values
        }
        if ((l & 15) == 0) *reinterpret_cast<f32x4 *>(red + k * 16 + P::row(l, 0)) = acc;
        if (l == 0) {
            weight[k] = w;
            used[k] = m != nullptr;
        }
    }
    const bool ok = ids_ok(a, id);
    __syncthreads();
    if (ok && tid < 16 && row0 + tid < d.rows) {
        float v = 0.0f;
        for (uint32_t k = 0; k < a.top_k; ++k)
            if (used[k]) v = __builtin_fmaf(weight[k], red[k * 16 + tid], v);
        const f32x4 one = {v, 0.0f, 0.0f, 0.0f};
        store4(y + (size_t)token * d.rows + row0 + tid, 1, one);
    }
}

bool pairs_path(const F8ExpertsDev &ex, uint32_t t, uint32_t top_k) {
    return t <= kPairsTokens && t * top_k <= kPairsMax && ex.hidden <= kPairsHidden && ex.width <= kPairsWidth;
}
// Rows of a tile by the pairs an expert has on average: enough to hold most
// experts' in one tile, whose weights are then read once; but no more than 96, so
// that a compute unit has two workgroups, of which one computes while the other
// starts or stores.  Experts that fill several tiles anyway take 64 rows until
// those of 96 would give every compute unit two workgroups of gate_up, and 32
// where those of 64 would give one to fewer than half of them.  us for tiles of 32
// / 64 / 96 rows, bf16 y, hidden 2048, width 512, top 8: 256 experts, 512 tokens
// (mean 16) 175 / 163 / 180, 1100 (34) 220 / 191 / 197, 2048 (64) 282 / 226 / 210,
// 4096 475 / 328 / 305; 60 experts, 300 tokens (40) 65 / 55 / 58, 512 (68) 86 / 76
// / 62, 800 (107) 118 / 82 / 83, 2048 222 / 159 / 146; 8 experts, 16 tokens 28.5 /
// 30.5 / 39, 64 34 / 39 / 43, 128 35 / 40 / 43, 256 41 / 42 / 50, 512 63 / 50 / 57,
// 1000 101 / 78 / 86, 4096 334 / 240 / 237.  Up to 64 pairs stay on the tiles whose
// products are all exact, as the path for few pairs is.
uint32_t tile_rows(const F8ExpertsDev &ex, uint32_t t, uint32_t top_k) {
    const uint32_t pairs = t * top_k, mean = pairs <= kPairsMax ? std::min(pairs / ex.n_experts, 14u) : pairs / ex.n_experts;
    const uint32_t blocks = (ex.width + 127) / 128, cus = (uint32_t)cu_count();
    if (mean <= 14) return mean <= 6 ? 16 : 32;
    if (ex.n_experts * ((mean + 63) / 64) * blocks < cus / 2) return 32;
    if (mean <= 40) return 64;
    return mean > 96 && pairs / 96 * blocks < 2 * cus ? 64 : 96;
}
struct ExpertsScratch {
    int32_t *pos_of_pair, *row_of_pos, *n_tiles;
    Tile *tiles;
    uint8_t *xq, *hq;
    float *xs, *hs, *out_scales;
    void *out;
    bool out16;
    uint32_t max_tiles;
    size_t total;
};
ExpertsScratch experts_scratch(void *scratch, const F8ExpertsDev &ex, uint32_t t, uint32_t top_k, int32_t y_type) {
    const size_t P = (size_t)t * top_k, kbh = (ex.hidden + 127) / 128, kbf = (ex.width + 127) / 128;
    const uint32_t m = tile_rows(ex, t, top_k);
    ExpertsScratch b;
    b.max_tiles = (uint32_t)(P / m + (P < ex.n_experts ? P : ex.n_experts) + 15) / 16 * 16;  // launched by eights
    uint8_t *p = static_cast<uint8_t *>(scratch);
    size_t off = 0;
    auto take = [&](size_t bytes) {
        uint8_t *at = p + off;
        off += align256(bytes);
        return at;
    };
    b.n_tiles = reinterpret_cast<int32_t *>(take(4));
    b.pos_of_pair = reinterpret_cast<int32_t *>(take(P * 4));
    b.row_of_pos = reinterpret_cast<int32_t *>(take(P * 4));
    b.tiles = reinterpret_cast<Tile *>(take((size_t)b.max_tiles * sizeof(Tile)));
    b.xq = take((size_t)t * kbh * 128);
    b.xs = reinterpret_cast<float *>(take((size_t)t * kbh * 4));
    b.hq = take(P * kbf * 128);
    b.hs = reinterpret_cast<float *>(take(P * kbf * 4));
    const size_t blocks = (ex.hidden + kOutBlock - 1) / kOutBlock;
    b.out16 = m >= 64 && y_type == TQF_HIP_TYPE_BF16;
    b.out = take(b.out16 ? P * blocks * kOutBlock * 2 : P * ex.hidden * 4);
    b.out_scales = reinterpret_cast<float *>(take(b.out16 ? P * blocks * 4 : 0));
    b.total = off;
    return b;
}

// How a kernel takes tiles of kRows rows; G: gate_up, D: down.
template <class P_, int RT_, int CT_, int AHEAD_>
struct TileForm {
    typedef P_ P;
    static constexpr int RT = RT_, CT = CT_, AHEAD = AHEAD_, kRows = CT_ * P_::M;
};
template <class G, class D, typename OT>
hipError_t launch_tiles(hipStream_t s, const F8ExpertsDev &ex, const ExpertsScratch &b, uint32_t t, uint32_t pairs) {
    static_assert(G::kRows == D::kRows, "gate_up and down take the same tiles");
    static_assert(G::RT * G::P::M == 64, "a workgroup of gate_up makes one block of h");
    TiledArgs a{};
    a.d = f8_shape(ex.width, ex.hidden);
    a.xq = b.xq;
    a.xs = b.xs;
    a.xrows = t;
    a.tiles = b.tiles;
    a.row_of_pos = b.row_of_pos;
    a.hq = b.hq;
    a.hs = b.hs;
    a.hkb = (ex.width + 127) / 128;
    a.hrows = pairs;
    a.rblocks = a.hkb;
    f8_tiled_kernel<typename G::P, G::RT, G::CT, kGateUp, float, 1, false, G::AHEAD><<<b.max_tiles * a.rblocks, 256, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.d = f8_shape(ex.hidden, ex.width);
    a.xq = b.hq;
    a.xs = b.hs;
    a.xrows = pairs;
    a.out = b.out;
    a.out_scales = b.out_scales;
    a.rblocks = (ex.hidden + 255) / 256;
    f8_tiled_kernel<typename D::P, D::RT, D::CT, kDown, OT, 1, false, D::AHEAD><<<b.max_tiles * a.rblocks, 256, 0, s>>>(a);
    return hipGetLastError();
}

template <typename XT, typename YT>
hipError_t experts(hipStream_t s, const F8ExpertsDev &ex, const XT *x, YT *y, const ExpertsArgs &a, void *scratch) {
    const uint32_t pairs = a.t * a.top_k;
    const F8Shape dg = f8_shape(ex.width, ex.hidden), dd = f8_shape(ex.hidden, ex.width);
    if (pairs_path(ex, a.t, a.top_k)) {
        const uint8_t **downs = static_cast<const uint8_t **>(scratch);
        float *h = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + kPairsMax * sizeof(void *));
        const uint32_t hstride = dd.kb * 128;
        f8_pair_gate_up_kernel<<<dim3((ex.width + 15) / 16, pairs), 256, dg.kb * 260 + 16 + 512, s>>>(a, ex.mats, dg, x, h, hstride, downs);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        f8_pair_down_kernel<<<dim3((ex.hidden + 15) / 16, a.t), 512, 8 * dd.kb * 260 + a.top_k * 64, s>>>(a, downs, dd, h, hstride, y);
        return hipGetLastError();
    }
    const ExpertsScratch b = experts_scratch(scratch, ex, a.t, a.top_k, sizeof(YT) == 2 ? TQF_HIP_TYPE_BF16 : TQF_HIP_TYPE_F32);
    const uint32_t plan = (pairs + kPlanThreads - 1) / kPlanThreads, quant = (quantize_chunks(a.t, dg.kb) + kPlanThreads - 1) / kPlanThreads;
    const uint32_t m = tile_rows(ex, a.t, a.top_k);
    f8_plan_kernel<<<plan + quant, kPlanThreads, 0, s>>>(a, m, b.pos_of_pair, b.row_of_pos, b.tiles, b.max_tiles, ex.mats, b.n_tiles, x, ex.hidden, dg.kb,
                                                        b.xq, b.xs);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // gate_up always takes the bf16 instructions: its error would move values of h
    // across a rounding step (fp8 ones: 2.1e-3 to 2.3e-3 of y instead of the 1.7e-3
    // that bf16 rounding costs, and an f32 y no nearer than a bf16 one).  down takes
    // the fp8 ones where its results are rounded to bf16 next; 4096 tokens take 305
    // us so, and 277 with gate_up on the fp8 ones too.
    typedef TileForm<Bf16x16, 4, 1, 2> T16;
    typedef TileForm<Bf16x16, 4, 2, 2> T32;
    typedef TileForm<Bf16x16, 4, 4, 2> T64;
    typedef TileForm<Bf16x16, 4, 6, 1> T96;
    if (m == 16) {
        e = launch_tiles<T16, T16, float>(s, ex, b, a.t, pairs);
    } else if (m == 32) {
        e = launch_tiles<T32, T32, float>(s, ex, b, a.t, pairs);
    } else if constexpr (sizeof(YT) == 4) {
        e = m == 64 ? launch_tiles<T64, T64, float>(s, ex, b, a.t, pairs) : launch_tiles<T96, T96, float>(s, ex, b, a.t, pairs);
    } else {
        e = m == 64 ? launch_tiles<T64, TileForm<Fp8x32, 2, 2, 2>, Out16>(s, ex, b, a.t, pairs)
                    : launch_tiles<T96, TileForm<Fp8x32, 2, 3, 1>, Out16>(s, ex, b, a.t, pairs);
    }
    if (e != hipSuccess) return e;
    if (sizeof(YT) == 2 && b.out16) {
        f8_combine16_kernel<<<dim3((ex.hidden + 2047) / 2048, a.t), 256, 0, s>>>(a, b.pos_of_pair, b.n_tiles, static_cast<const Out16 *>(b.out),
                                                                                b.out_scales, ex.hidden, reinterpret_cast<uint16_t *>(y));
    } else {
        f8_combine_kernel<<<dim3((ex.hidden + 1023) / 1024, a.t), 256, 0, s>>>(a, b.pos_of_pair, b.n_tiles, static_cast<const float *>(b.out),
                                                                              ex.hidden, y);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_f8_repack(hipStream_t s, const uint8_t *q, const float *scales, const F8Shape &d, uint8_t *out) {
    const size_t chunks = f8_tile_bytes(d) / 16;  // more than there are scales
    f8_repack_kernel<<<(uint32_t)((chunks + 255) / 256), 256, 0, s>>>(q, scales, d, out);
    return hipGetLastError();
}

size_t f8_matmul_scratch_bytes(const F8Shape &d, uint32_t t) {
    if (rows_path(d, t)) return 0;
    return align256((size_t)pad32(t) * d.kb * 128) + align256((size_t)pad32(t) * d.kb * 4);
}

hipError_t launch_f8_matmul(hipStream_t s, const uint8_t *mat, const F8Shape &d, const void *x, int32_t x_type, uint32_t t,
                            void *y, int32_t y_type, void *scratch) {
    const float *xf = static_cast<const float *>(x);
    const uint16_t *xb = static_cast<const uint16_t *>(x);
    float *yf = static_cast<float *>(y);
    uint16_t *yb = static_cast<uint16_t *>(y);
    if (x_type == TQF_HIP_TYPE_F32)
        return y_type == TQF_HIP_TYPE_F32 ? matmul(s, mat, d, xf, t, yf, scratch) : matmul(s, mat, d, xf, t, yb, scratch);
    return y_type == TQF_HIP_TYPE_F32 ? matmul(s, mat, d, xb, t, yf, scratch) : matmul(s, mat, d, xb, t, yb, scratch);
}

size_t f8_experts_scratch_bytes(const F8ExpertsDev &ex, uint32_t t, uint32_t top_k, int32_t y_type) {
    if (pairs_path(ex, t, top_k)) return kPairsMax * sizeof(void *) + (size_t)t * top_k * ((ex.width + 127) / 128 * 128) * 4;
    return experts_scratch(nullptr, ex, t, top_k, y_type).total;
}

hipError_t launch_f8_experts(hipStream_t s, const F8ExpertsDev &ex, const void *x, int32_t x_type, uint32_t t,
                             const uint16_t *ids, const float *w, uint32_t top_k, void *y, int32_t y_type, int32_t *status,
                             void *scratch) {
    const ExpertsArgs a{ids, w, t, top_k, ex.n_experts, status};
    const float *xf = static_cast<const float *>(x);
    const uint16_t *xb = static_cast<const uint16_t *>(x);
    float *yf = static_cast<float *>(y);
    uint16_t *yb = static_cast<uint16_t *>(y);
    if (x_type == TQF_HIP_TYPE_F32)
        return y_type == TQF_HIP_TYPE_F32 ? experts(s, ex, xf, yf, a, scratch) : experts(s, ex, xf, yb, a, scratch);
    return y_type == TQF_HIP_TYPE_F32 ? experts(s, ex, xb, yf, a, scratch) : experts(s, ex, xb, yb, a, scratch);
}

}  // namespace tqf
