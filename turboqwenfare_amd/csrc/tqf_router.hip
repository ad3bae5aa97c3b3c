// tqf_router.hip -- the router for the rows of a batch (gfx950).
//
//   router_logits   L[t][e] = sum_h x[t][h] R[e][h]
//   route_tokens    s = softmax(L[t]) or sigmoid(L[t]);  c = s + bias (for
//                   choosing only);  the best top_groups groups by the sum of
//                   their best one or two c;  the top_k experts of those by c,
//                   ties to the lowest index;  w = s, divided by their sum if
//                   renormalised, times scale.
// The counterpart for many rows of the router inside the MoE layer kernels
// (RouterResult::from_logits, experts/mod.rs:134-197, is softmax, top-8,
// renormalised).
#include <hip/hip_runtime.h>

#include "tqf_f8.h"

namespace tqf {

namespace {

// ---- logits ------------------------------------------------------------------
// Few rows: a workgroup takes one expert, its four wavefronts a quarter of the
// row each, and every product is summed in 64 bits.  Bound by the launch and
// one trip to memory.
constexpr uint32_t kFewRows = 8;
template <typename XT>
__global__ __launch_bounds__(256) void logits_few_kernel(const float *__restrict__ router, const XT *__restrict__ x, uint32_t t,
                                                         uint32_t n_experts, uint32_t hidden, float *__restrict__ logits) {
    __shared__ double red[4][kFewRows];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64;
    const uint32_t e = blockIdx.x;
    const float *r = router + (size_t)e * hidden;
    double acc[kFewRows] = {};
    for (uint32_t k = tid * 8; k < hidden; k += 2048) {
        float w[8];
        load_row<8>(r + k, (int)(hidden - k), w);
#pragma unroll
        for (uint32_t i = 0; i < kFewRows; ++i) {
            if (i >= t) break;
            float v[8];
            load_row<8>(x + (size_t)i * hidden + k, (int)(hidden - k), v);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[i] = __builtin_fma((double)w[j], (double)v[j], acc[i]);
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < kFewRows; ++i) {
        if (i >= t) break;
        double v = acc[i];
#pragma unroll
        for (int o = 32; o >= 1; o /= 2) v += __shfl_xor(v, o);
        if (l == 0) red[wave][i] = v;
    }
    __syncthreads();
    if (tid < (int)t) logits[(size_t)tid * n_experts + e] = (float)((red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]));
}

// Many rows, on the bf16 matrix cores without losing bits: an f32 is the sum of
// three bf16 (8 bits each; exact for magnitudes above 2^-102, below which the
// last pieces vanish), so R = R0 + R1 + R2, and for bf16 x three products give
// every bit of x R; f32 x is split as well, and of the nine products the six
// above 2^-24 of the largest are taken.  A workgroup has 16 ET experts by 16 TT
// rows; its wavefronts split K (8 ways, a step of 32 columns each in turn) and add
// their sums in LDS, pairwise, in the same order for every tile size.  4096 rows of
// 2048 by 256 experts: 19 us with bf16 x and 35 with f32, where the products alone
// would take 8.6 and 17 at the rate of a large library product; the vector units,
// which split the router's rows anew in every workgroup, and the matrix cores take
// turns.  The f32 instructions (157 TFLOP/s from registers) need 27 us for the
// product alone: more than the bf16 form takes, less than the f32 one does; a
// kernel of them was not built.
struct Split3 {
    bf16x8 p[3];
};
__device__ __forceinline__ Split3 split3(const float (&v)[8]) {
    Split3 s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __bf16 a = (__bf16)v[i];
        const float r = v[i] - (float)a;
        const __bf16 b = (__bf16)r;
        s.p[0][i] = a;
        s.p[1][i] = b;
        s.p[2][i] = (__bf16)(r - (float)b);
    }
    return s;
}
constexpr int kLogitWaves = 8;

// A step's 32 columns of 16 N rows on their way to a wavefront.  A lane that
// loaded its own operands (row l % 16) would make every one of them a cache
// access of its own, and the accesses, one a cycle, would bound the kernel: so
// neighbouring lanes load neighbouring 16 bytes of a row, and the wavefront
// passes them through an LDS tile that only it uses.  Chunks of a 128-byte line
// (one f32 row or two bf16 ones) are permuted by the line, so that neither side
// meets a bank twice.
template <typename T, int N>
struct Stage {
    static constexpr int kRowChunks = 2 * (int)sizeof(T), kLoads = N * kRowChunks / 4, kBytes = kLoads * 1024;
    u32x4 q[kLoads];
    const uint8_t *base;   // of the first row
    uint32_t off[kLoads];  // from there
    static __device__ __forceinline__ int slot(int row, int chunk) {
        const int i = row * kRowChunks + chunk, line = i / 8;
        return (line * 8 + ((i ^ line) & 7)) * 16;
    }
    __device__ __forceinline__ void begin(const T *p, uint32_t hidden, uint32_t row0, uint32_t rows, int l) {
        base = reinterpret_cast<const uint8_t *>(p + (size_t)row0 * hidden);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const uint32_t row = (j * 64 + l) / kRowChunks;
            off[j] = (row0 + row < rows ? row : rows - 1 - row0) * hidden * (uint32_t)sizeof(T) + l % kRowChunks * 16;
        }
    }
    // Rows may begin anywhere (an odd number of columns): the loads need no
    // alignment but the type's.  TAIL: the last step is no whole one; its columns
    // are taken one by one.
    template <bool TAIL>
    __device__ __forceinline__ void ask(uint32_t step, uint32_t hidden, int l) {
        const uint8_t *p = base + (size_t)step * 32 * sizeof(T);
        if (!TAIL || (step + 1) * 32 <= hidden) {
#pragma unroll
            for (int j = 0; j < kLoads; ++j) __builtin_memcpy(&q[j], __builtin_assume_aligned(p + off[j], sizeof(T)), 16);
        } else {
            constexpr int kEach = 16 / sizeof(T);
            const uint32_t k = step * 32 + l % kRowChunks * kEach;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                T v[kEach];
#pragma unroll
                for (int i = 0; i < kEach; ++i) v[i] = k + i < hidden ? reinterpret_cast<const T *>(p + off[j])[i] : T{};
                __builtin_memcpy(&q[j], v, 16);
            }
        }
    }
    __device__ __forceinline__ void put(uint8_t *lds, int l) const {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) *reinterpret_cast<u32x4 *>(lds + slot((j * 64 + l) / kRowChunks, l % kRowChunks)) = q[j];
    }
    // the eight columns 8 g of row 16 i + r
    static __device__ __forceinline__ Split3 get(const uint8_t *lds, int i, int r, int g) {
        Split3 s;
        if constexpr (sizeof(T) == 2) {
            s.p[0] = *reinterpret_cast<const bf16x8 *>(lds + slot(16 * i + r, g));
        } else {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(lds + slot(16 * i + r, 2 * g));
            const f32x4 hi = *reinterpret_cast<const f32x4 *>(lds + slot(16 * i + r, 2 * g + 1));
            const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            s = split3(v);
        }
        return s;
    }
};

template <int ET, int TT, bool TAIL, typename XT>
__global__ __launch_bounds__(64 * kLogitWaves) void logits_kernel(const float *__restrict__ router, const XT *__restrict__ x,
                                                                  uint32_t t, uint32_t n_experts, uint32_t hidden,
                                                                  float *__restrict__ logits) {
    // a wavefront's stage, then its sums
    constexpr int kStage = Stage<float, ET>::kBytes + Stage<XT, TT>::kBytes, kSums = ET * TT * 1024;
    constexpr int kMine = kStage > kSums ? kStage : kSums;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kLogitWaves][kMine];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64, r = l & 15, g = l >> 4;
    uint8_t *mine = lds[wave];
    // neighbouring workgroups run on different XCDs: those of the same rows are
    // given to one, whose L2 then loads them once
    const uint32_t ebs = (n_experts + 16 * ET - 1) / (16 * ET), in = blockIdx.x / 8;
    const uint32_t e0 = in % ebs * 16 * ET, t0 = (in / ebs * 8 + blockIdx.x % 8) * 16 * TT;
    if (t0 >= t) return;
    f32x4 acc[ET][TT] = {};
    // a piece of every row tile before the next piece: neighbouring instructions
    // then add to different sums and need not wait for each other
    auto multiply = [&](int e, const Split3 &w, const Split3 (&xs)[TT]) {
        auto add = [&](int wp, int xp) {
#pragma unroll
            for (int i = 0; i < TT; ++i) acc[e][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[wp], xs[i].p[xp], acc[e][i], 0, 0, 0);
        };
        if constexpr (sizeof(XT) == 2) {
            add(2, 0);
            add(1, 0);
            add(0, 0);
        } else {
            add(2, 0);
            add(1, 1);
            add(0, 2);
            add(1, 0);
            add(0, 1);
            add(0, 0);
        }
    };
    const uint32_t steps = (hidden + 31) / 32;
    // a step's operands are asked for while the one before is computed
    Stage<float, ET> ws;
    Stage<XT, TT> xs;
    ws.begin(router, hidden, e0, n_experts, l);
    xs.begin(x, hidden, t0, t, l);
    uint8_t *wt = mine, *xt = mine + ws.kBytes;
    auto ask = [&](uint32_t st) {
        // behind the last step nothing is loaded, or, where the branch costs more
        // than the load (4096 rows 20.5 us, 19 without it; 512 rows 7.1, and 8.1
        // without it), the last step again
        if (TAIL || ET * TT <= 4) {
            if (st >= steps) return;
        } else {
            st = st < steps ? st : steps - 1;
        }
        ws.template ask<TAIL>(st, hidden, l);
        xs.template ask<TAIL>(st, hidden, l);
    };
    ask(wave);
    for (uint32_t st = wave; st < steps; st += kLogitWaves) {
        ws.put(wt, l);
        xs.put(xt, l);
        ask(st + kLogitWaves);
        Split3 xp[TT];
#pragma unroll
        for (int i = 0; i < TT; ++i) xp[i] = xs.get(xt, i, r, g);
#pragma unroll
        for (int e = 0; e < ET; ++e) {
            multiply(e, ws.get(wt, e, r, g), xp);
            if constexpr (sizeof(XT) == 4) __builtin_amdgcn_sched_barrier(0);  // or the next tiles' pieces take all registers
        }
    }
#pragma unroll
    for (int e = 0; e < ET; ++e)
#pragma unroll
        for (int i = 0; i < TT; ++i) reinterpret_cast<f32x4 *>(mine)[(e * TT + i) * 64 + l] = acc[e][i];
    __syncthreads();
    for (int tile = wave; tile < ET * TT; tile += kLogitWaves) {
        auto sum = [&](int w) { return reinterpret_cast<const f32x4 *>(lds[w])[tile * 64 + l]; };
        auto two = [&](int w) { return sum(w) + sum(w + 4); };
        const f32x4 v = (two(0) + two(2)) + (two(1) + two(3));
        const uint32_t row = t0 + tile % TT * 16 + r, col = e0 + tile / TT * 16 + 4 * g;
        if (row < t && col < n_experts) store4(logits + (size_t)row * n_experts + col, (int)(n_experts - col), v);
    }
}

// ---- routes --------------------------------------------------------------------
// A wavefront takes a row.  Its lanes are dealt to the groups, L = 2^n <= 64 /
// groups of them to each (one group: all 64), and lane j of a group holds its
// experts j, j + L, ...: so a group's best scores are a reduction over L
// neighbouring lanes.  Scores, sums and comparisons are in 64 bits, where
// neither a sum's order nor a rounding decides between two experts whose f32
// scores would be equal.
struct RouteArgs64 {
    uint32_t t, n_experts, per, lanes;  // experts in a group, lanes of a group
    const float *bias;
    tqf_hip_route_options o;
    uint16_t *ids;
    float *w;
    int32_t *status;
};

// Order-preserving key of a double that is not NaN; 0 is below all of them.
__device__ __forceinline__ uint64_t key64(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ float logit_of(const float *p, size_t i) { return p[i]; }
__device__ __forceinline__ float logit_of(const uint16_t *p, size_t i) { return __uint_as_float((uint32_t)p[i] << 16); }

template <int N, typename LT>
__global__ __launch_bounds__(256) void pick_routes_kernel(RouteArgs64 a, const LT *__restrict__ logits) {
    const int lane = threadIdx.x % 64;
    const uint32_t row = blockIdx.x * 4 + threadIdx.x / 64;
    if (row >= a.t) return;
    const double none = -__builtin_inf();
    const uint32_t group = (uint32_t)lane / a.lanes, j0 = (uint32_t)lane % a.lanes, e0 = group * a.per + j0;
    const bool mine = group < a.o.n_groups;
    double s[N], c[N];
    bool bad = false;
    float top = -__builtin_inff();
    float lg[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t j = j0 + i * a.lanes;
        lg[i] = -__builtin_inff();
        if (mine && j < a.per) lg[i] = logit_of(logits, (size_t)row * a.n_experts + e0 + i * a.lanes);
        bad |= !(lg[i] < __builtin_inff());  // NaN or +inf
        top = fmaxf(top, lg[i]);
    }
    if (a.o.score == TQF_HIP_SCORE_SOFTMAX) {
        top = key2f(wave_umax(f2key(top)));
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i] = lg[i] > -__builtin_inff() ? exp((double)lg[i] - (double)top) : 0.0;
            sum += s[i];
        }
#pragma unroll
        for (int o = 32; o >= 1; o /= 2) sum += __shfl_xor(sum, o);
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = lg[i] > -__builtin_inff() ? s[i] / sum : 0.0;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = 1.0 / (1.0 + exp(-(double)lg[i]));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        c[i] = none;
        if (lg[i] > -__builtin_inff()) {
            c[i] = s[i];
            if (a.bias) c[i] += (double)a.bias[e0 + i * a.lanes];
            bad |= !(c[i] < __builtin_inf());
        }
    }
    bad = __ballot(bad) != 0;

    if (a.o.n_groups > 1 && a.o.top_groups < a.o.n_groups) {
        double b1 = none, b2 = none;  // the group's best two
#pragma unroll
        for (int i = 0; i < N; ++i) {
            b2 = c[i] > b1 ? b1 : (c[i] > b2 ? c[i] : b2);
            b1 = c[i] > b1 ? c[i] : b1;
        }
        for (uint32_t o = a.lanes / 2; o >= 1; o /= 2) {
            const double p1 = __shfl_xor(b1, (int)o), p2 = __shfl_xor(b2, (int)o);
            const double hi = p1 > b1 ? p1 : b1, lo = p1 > b1 ? b1 : p1, rest = p2 > b2 ? p2 : b2;
            b1 = hi;
            b2 = lo > rest ? lo : rest;
        }
        if (a.o.group_best == 2 && b2 > none) b1 += b2;
        uint32_t rank = 0;
        for (uint32_t g = 0; g < a.o.n_groups; ++g) {
            const double v = __shfl(b1, (int)(g * a.lanes));
            rank += v > b1 || (v == b1 && g < group);
        }
        if (rank >= a.o.top_groups) {
#pragma unroll
            for (int i = 0; i < N; ++i) c[i] = none;
        }
    }

    uint64_t key[N];
#pragma unroll
    for (int i = 0; i < N; ++i) key[i] = c[i] > none && !bad ? key64(c[i]) : 0;
    double my_s = 0.0;
    uint32_t my_id = TQF_HIP_NO_EXPERT;
    for (uint32_t k = 0; k < a.o.top_k; ++k) {
        // the lane's best: the first of equal keys is its lowest expert
        uint64_t best = 0;
        uint32_t at = 0;
        double val = 0.0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool more = key[i] > best;
            best = more ? key[i] : best;
            at = more ? (uint32_t)i : at;
            val = more ? s[i] : val;
        }
        const uint32_t hi = wave_umax((uint32_t)(best >> 32));
        if (hi == 0) break;  // (a key that is not 0 has bits above its 32nd)
        // one lane with the largest upper half has won; several compare the lower
        // halves, and equals their experts
        bool won = (uint32_t)(best >> 32) == hi;
        uint64_t who = __ballot(won);
        const uint32_t e = e0 + at * a.lanes;
        if (who & (who - 1)) {
            const uint32_t lo = wave_umax(won ? (uint32_t)best : 0u);
            won = won && (uint32_t)best == lo;
            const uint32_t first = ~wave_umax(won ? ~e : 0u);
            won = won && e == first;
            who = __ballot(won);
        }
        const int from = (int)__builtin_ctzll(who);
        const uint32_t win = (uint32_t)__builtin_amdgcn_readlane((int)e, from);
        const double sv = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(val), from),
                                           __builtin_amdgcn_readlane(__double2loint(val), from));
        if ((uint32_t)lane == k) {
            my_s = sv;
            my_id = win;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) key[i] = won && at == (uint32_t)i ? 0 : key[i];
    }
    if (a.o.renormalise) {
        double sum = my_s;
#pragma unroll
        for (int o = 8; o >= 1; o /= 2) sum += __shfl_xor(sum, o);
        my_s = sum > 0.0 ? my_s / sum : 0.0;
    }
    if ((uint32_t)lane < a.o.top_k) {
        a.ids[(size_t)row * a.o.top_k + lane] = (uint16_t)my_id;
        a.w[(size_t)row * a.o.top_k + lane] = (float)(my_s * (double)a.o.scale);
    }
    if (bad && lane == 0 && a.status) *a.status = TQF_HIP_ERR_ROUTER;
}

template <int ET, int TT, typename XT>
void logits_many(hipStream_t s, const float *router, const XT *x, uint32_t t, uint32_t n, uint32_t hidden, float *logits) {
    const uint32_t ebs = (n + 16 * ET - 1) / (16 * ET), tbs = (t + 16 * TT - 1) / (16 * TT), grid = (tbs + 7) / 8 * 8 * ebs;
    if (hidden % 32 == 0) logits_kernel<ET, TT, false, XT><<<grid, 64 * kLogitWaves, 0, s>>>(router, x, t, n, hidden, logits);
    else logits_kernel<ET, TT, true, XT><<<grid, 64 * kLogitWaves, 0, s>>>(router, x, t, n, hidden, logits);
}
template <typename XT>
hipError_t logits_launch(hipStream_t s, const float *router, const XT *x, uint32_t t, uint32_t n, uint32_t hidden, float *logits) {
    if (t <= kFewRows) {
        logits_few_kernel<<<n, 256, 0, s>>>(router, x, t, n, hidden, logits);
        return hipGetLastError();
    }
    // The larger a workgroup's tile, the fewer pieces are split and bytes loaded
    // for a product; the smaller, the sooner its eight wavefronts are through
    // their steps.  With 2048 columns and 256 experts, bf16 rows, us:
    //               1 x 2   2 x 2   2 x 4   2 x 8   4 x 4
    //   512 rows      7.1                    16.2    18
    //   1024 rows    10.7    10.5    12.2    16.4    18.1
    //   4096 rows    35.6    30.7    24.6    19.3    21.7
    // and f32 rows (2 x 8 would not fit the registers)
    //   1024 rows    19.8    16.1    22.4            30.5
    //   4096 rows    62.5    47.9    45.7            35.2
    const uint64_t tiles = (uint64_t)((n + 15) / 16) * ((t + 15) / 16);
    if (tiles <= 512) logits_many<1, 2>(s, router, x, t, n, hidden, logits);
    else if (tiles <= 1024) logits_many<2, 2>(s, router, x, t, n, hidden, logits);
    else if (tiles <= 2048) logits_many<2, 4>(s, router, x, t, n, hidden, logits);
    else if constexpr (sizeof(XT) == 2) logits_many<2, 8>(s, router, x, t, n, hidden, logits);
    else logits_many<4, 4>(s, router, x, t, n, hidden, logits);
    return hipGetLastError();
}

template <typename LT>
hipError_t route_launch(hipStream_t s, const RouteArgs64 &a, const LT *logits) {
    const uint32_t n = (a.per + a.lanes - 1) / a.lanes, grid = (a.t + 3) / 4;
    if (n <= 1) pick_routes_kernel<1><<<grid, 256, 0, s>>>(a, logits);
    else if (n <= 2) pick_routes_kernel<2><<<grid, 256, 0, s>>>(a, logits);
    else if (n <= 4) pick_routes_kernel<4><<<grid, 256, 0, s>>>(a, logits);
    else if (n <= 8) pick_routes_kernel<8><<<grid, 256, 0, s>>>(a, logits);
    else if (n <= 16) pick_routes_kernel<16><<<grid, 256, 0, s>>>(a, logits);
    else if (n <= 32) pick_routes_kernel<32><<<grid, 256, 0, s>>>(a, logits);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace

hipError_t launch_router_logits(hipStream_t s, const float *router, const void *x, int32_t x_type, uint32_t t,
                                uint32_t n_experts, uint32_t hidden, float *logits) {
    if (x_type == TQF_HIP_TYPE_F32) return logits_launch(s, router, static_cast<const float *>(x), t, n_experts, hidden, logits);
    return logits_launch(s, router, static_cast<const uint16_t *>(x), t, n_experts, hidden, logits);
}

hipError_t launch_route_tokens(hipStream_t s, const void *logits, int32_t logits_type, uint32_t t, uint32_t n_experts,
                               const float *bias, const tqf_hip_route_options &o, uint16_t *ids, float *w, int32_t *status) {
    uint32_t lanes = 64;
    while (lanes * o.n_groups > 64) lanes /= 2;
    const RouteArgs64 a{t, n_experts, n_experts / o.n_groups, lanes, bias, o, ids, w, status};
    if (logits_type == TQF_HIP_TYPE_F32) return route_launch(s, a, static_cast<const float *>(logits));
    return route_launch(s, a, static_cast<const uint16_t *>(logits));
}

}  // namespace tqf
