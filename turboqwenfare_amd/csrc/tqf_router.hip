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
    const bool wvec = rows_aligned(router, hidden, 4), xvec = rows_aligned(x, hidden, sizeof(XT));
    double acc[kFewRows] = {};
    for (uint32_t k = tid * 8; k < hidden; k += 2048) {
        float w[8];
        load_row<8>(r + k, (int)(hidden - k), wvec, w);
#pragma unroll
        for (uint32_t i = 0; i < kFewRows; ++i) {
            if (i >= t) break;
            float v[8];
            load_row<8>(x + (size_t)i * hidden + k, (int)(hidden - k), xvec, v);
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
// above 2^-24 of the largest are taken.  The f32 instructions would take five
// times as long.  Wavefronts split K (8 ways) and take their operands straight
// from memory: 16 ET experts by 16 TT rows each, no LDS until their sums are
// added, pairwise.
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

template <int ET, int TT, typename XT>
__global__ __launch_bounds__(64 * kLogitWaves) void logits_kernel(const float *__restrict__ router, const XT *__restrict__ x,
                                                                  uint32_t t, uint32_t n_experts, uint32_t hidden,
                                                                  float *__restrict__ logits) {
    __shared__ f32x4 red[kLogitWaves / 2][ET * TT][64];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64, r = l & 15, g = l >> 4;
    const uint32_t e0 = blockIdx.x * 16 * ET, t0 = blockIdx.y * 16 * TT;
    const bool wvec = rows_aligned(router, hidden, 4), xvec = rows_aligned(x, hidden, sizeof(XT));
    const float *wrow[ET];
    const XT *xrow[TT];
#pragma unroll
    for (int i = 0; i < ET; ++i) {
        const uint32_t e = e0 + i * 16 + r;
        wrow[i] = router + (size_t)(e < n_experts ? e : n_experts - 1) * hidden;
    }
#pragma unroll
    for (int i = 0; i < TT; ++i) {
        const uint32_t row = t0 + i * 16 + r;
        xrow[i] = x + (size_t)(row < t ? row : t - 1) * hidden;
    }
    f32x4 acc[ET][TT] = {};
    const uint32_t steps = (hidden + 31) / 32;
    for (uint32_t st = wave; st < steps; st += kLogitWaves) {
        const uint32_t k = st * 32 + g * 8;
        const int valid = k < hidden ? (int)(hidden - k) : 0;
        Split3 xs[TT];
#pragma unroll
        for (int i = 0; i < TT; ++i) {
            float v[8];
            load_row<8>(xrow[i] + k, valid, xvec, v);
            if constexpr (sizeof(XT) == 2) {
#pragma unroll
                for (int j = 0; j < 8; ++j) xs[i].p[0][j] = (__bf16)v[j];
            } else {
                xs[i] = split3(v);
            }
        }
#pragma unroll
        for (int e = 0; e < ET; ++e) {
            float v[8];
            load_row<8>(wrow[e] + k, valid, wvec, v);
            const Split3 w = split3(v);
#pragma unroll
            for (int i = 0; i < TT; ++i) {
                f32x4 a = acc[e][i];
                auto add = [&](int wp, int xp) { a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[wp], xs[i].p[xp], a, 0, 0, 0); };
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
                acc[e][i] = a;
            }
        }
    }
    for (int half = kLogitWaves / 2; half >= 1; half /= 2) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int e = 0; e < ET; ++e)
#pragma unroll
                for (int i = 0; i < TT; ++i) red[wave - half][e * TT + i][l] = acc[e][i];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int e = 0; e < ET; ++e)
#pragma unroll
                for (int i = 0; i < TT; ++i) acc[e][i] += red[wave][e * TT + i][l];
        }
        __syncthreads();
    }
    if (wave) return;
    const bool vec = ((reinterpret_cast<uintptr_t>(logits) | (uint64_t)n_experts * 4) & 15) == 0;
#pragma unroll
    for (int i = 0; i < TT; ++i) {
        const uint32_t row = t0 + i * 16 + r;
        if (row >= t) continue;
#pragma unroll
        for (int e = 0; e < ET; ++e) {
            const uint32_t col = e0 + e * 16 + 4 * g;
            if (col < n_experts) store4(logits + (size_t)row * n_experts + col, (int)(n_experts - col), vec, acc[e][i]);
        }
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
__global__ __launch_bounds__(256) void route_kernel(RouteArgs64 a, const LT *__restrict__ logits) {
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
        const uint32_t lo = wave_umax((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
        if ((hi | lo) == 0) break;
        const uint32_t e = e0 + at * a.lanes;
        const bool cand = best == (((uint64_t)hi << 32) | lo);
        const uint32_t win = ~wave_umax(cand ? ~e : 0u);
        const bool won = cand && e == win;
        const int from = (int)__builtin_ctzll(__ballot(won));
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

template <typename XT>
hipError_t logits_launch(hipStream_t s, const float *router, const XT *x, uint32_t t, uint32_t n, uint32_t hidden, float *logits) {
    if (t <= kFewRows) {
        logits_few_kernel<<<n, 256, 0, s>>>(router, x, t, n, hidden, logits);
    } else if (t <= 512) {
        logits_kernel<1, 2, XT><<<dim3((n + 15) / 16, (t + 31) / 32), 64 * kLogitWaves, 0, s>>>(router, x, t, n, hidden, logits);
    } else {
        logits_kernel<4, 4, XT><<<dim3((n + 63) / 64, (t + 63) / 64), 64 * kLogitWaves, 0, s>>>(router, x, t, n, hidden, logits);
    }
    return hipGetLastError();
}

template <typename LT>
hipError_t route_launch(hipStream_t s, const RouteArgs64 &a, const LT *logits) {
    const uint32_t n = (a.per + a.lanes - 1) / a.lanes, grid = (a.t + 3) / 4;
    if (n <= 1) route_kernel<1><<<grid, 256, 0, s>>>(a, logits);
    else if (n <= 2) route_kernel<2><<<grid, 256, 0, s>>>(a, logits);
    else if (n <= 4) route_kernel<4><<<grid, 256, 0, s>>>(a, logits);
    else if (n <= 8) route_kernel<8><<<grid, 256, 0, s>>>(a, logits);
    else if (n <= 16) route_kernel<16><<<grid, 256, 0, s>>>(a, logits);
    else if (n <= 32) route_kernel<32><<<grid, 256, 0, s>>>(a, logits);
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
