// tqf_prompt.hip -- causal attention of packed prompts with grouped heads (gfx950).
//
//   y[i][h] = sum_j softmax_j(scale q[i][h] . k[j][h / group]) v[j][h / group]
//             (* sigmoid(gate[i][h])),  j <= i + len_k - len_q of i's sequence.
//
// One pass over the keys with the running maximum m and sum l of the softmax: a
// tile's weights are exp(s - m), and what is summed so far is multiplied by
// exp(m_old - m) when m grows.
//
// A wavefront has 32 rows of one head.  It computes S^T = K Q^T with the
// 32 x 32 x 16 bf16 instructions: in their result a lane has one row and 16 keys,
// so a row's maximum and sum stay in two lanes, and the weights, rounded to bf16
// (at most 2^-8 of each, as y is), are an operand of O^T = V^T P^T
// as they stand: the order in which an instruction takes its K elements is free so
// long as both operands have the same.  V^T comes from LDS by transposing reads.
// A workgroup's wavefronts share tiles of K and V, and so, where heads are
// grouped, are heads of one group at the same rows.  Where there are few rows the
// keys are dealt out to several workgroups, and a second kernel joins their sums.
//
// Bound by how a wavefront's products, softmax and LDS reads take turns: the matrix
// cores are busy for 59% of 8192 rows' time (32 heads of 128: 490 us, 1.1 PFLOP/s;
// large library products reach 1.26 on this card).  4096 rows of 16 heads of 256 take
// 158 us, 0.87 PFLOP/s: the last row's workgroup has all 128 tiles, 1.1 us each when
// it is alone on its compute unit, where two together need 0.8 for one.  Dealing out
// such rows' keys too costs more in the join than it saves (167 us), and so do eight
// wavefronts that have every other tile each and wait for one another (178).
//
// Keys that a row does not see have weight 0, but 0 * inf and 0 * NaN are NaN.
// Rows behind a sequence's end read as zeros (the copies' bounds).  Tiles that some
// rows see in part are looked through for infinities and NaN; where there are any,
// the tile's values are added at the end, key by key, to the rows that see them.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "tqf_attn_device.h"

namespace tqf {

namespace {

constexpr int kWaves = 4;
constexpr int kAhead = 4;  // products that LDS reads go ahead of theirs
constexpr uint32_t kMaxParts = 16;

struct Kernel {
    PromptArgs a;
    uint32_t head_waves;  // wavefronts of a workgroup that have heads of their own (of one group)
    uint32_t head_sets;   // q_heads / head_waves
    uint32_t turn;        // workgroups from here on are taken from the end
    float scale_log2;
    float *o, *top_sum;  // of each part: [total_q][q_heads][dim], and [total_q][q_heads][2]
};

// The workgroup's place in the order of work, blockIdx.x of gridDim.x.
__device__ __forceinline__ uint32_t number_of(const Kernel &p) { return blockIdx.x < p.turn ? blockIdx.x : gridDim.x - 1 - (blockIdx.x - p.turn); }

// 8 elements of a row: times their gates' sigmoids, and as they are stored.
__device__ __forceinline__ void apply_gate(float (&v)[8], u32x4 gate) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] *= sigmoid(__uint_as_float(gate[e] << 16));
        v[2 * e + 1] *= sigmoid(__uint_as_float(gate[e] & 0xFFFF0000u));
    }
}
__device__ __forceinline__ u32x4 bf16_row(const float (&v)[8]) {
    return u32x4{bf16_bits2(v[0], v[1]), bf16_bits2(v[2], v[3]), bf16_bits2(v[4], v[5]), bf16_bits2(v[6], v[7])};
}

// The sequence and the tile in it of a workgroup's tile number; false: none.
struct Place {
    int32_t q0, lq, k0, lk;
    uint32_t tile;
};
__device__ __forceinline__ bool find_place(const PromptArgs &a, uint32_t number, uint32_t tokens, Place &p) {
    const uint32_t l = threadIdx.x & 63;
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < a.n_seqs; s0 += 64) {
        const uint32_t s = s0 + l;
        int32_t q0 = 0, q1 = 0, k0 = 0, k1 = 0;
        if (s < a.n_seqs) {
            q0 = a.cu_q[s], q1 = a.cu_q[s + 1], k0 = a.cu_k[s], k1 = a.cu_k[s + 1];
            const bool bad = q0 < 0 || q1 < q0 || (uint32_t)q1 > a.total_q || k0 < 0 || k1 < k0 || (uint32_t)k1 > a.total_k;
            if (bad) {
                if (a.status) *a.status = TQF_HIP_ERR_INVALID;
                q0 = q1 = k0 = k1 = 0;
            }
        }
        const uint32_t mine = ((uint32_t)(q1 - q0) + tokens - 1) / tokens;
        uint32_t upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const uint32_t v = __shfl_up(upto, o);
            if ((int)l >= o) upto += v;
        }
        const uint64_t past = __ballot(before + upto > number);
        if (past) {
            const int who = __builtin_ctzll(past);
            p.q0 = __shfl(q0, who);
            p.lq = __shfl(q1 - q0, who);
            p.k0 = __shfl(k0, who);
            p.lk = __shfl(k1 - k0, who);
            const uint32_t n = __shfl(mine, who), first = before + __shfl(upto, who) - n;
            p.tile = n - 1 - (number - first);  // the longest first
            return true;
        }
        before += __shfl(upto, 63);
    }
    return false;
}

// A tile of K or V in LDS: rows of 2 D bytes, the 16-byte chunk c of row r in slot
// c ^ swizzle(r).  K: 16 lanes that read a chunk of 16 rows find 16 different
// places in the banks.  V: the four rows that 16 lanes read transposed.
template <int D>
__device__ __forceinline__ uint32_t k_swizzle(uint32_t row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
template <int D>
__device__ __forceinline__ uint32_t v_swizzle(uint32_t row) { return D == 64 ? (row >> 1 & 1) << 2 : (row & 3) << 2; }

// D: head dimension, KT: keys of a tile (a multiple of 32).
template <int D, int KT>
__global__ __launch_bounds__(64 * kWaves, 2) void prompt_kernel(Kernel p) {
    constexpr int kRow = 2 * D, kTile = KT * kRow, kCopies = kTile / 1024 / kWaves, kSub = KT / 32, kDims = D / 32, kSteps = D / 16;
    static_assert(kCopies >= 1 && 2 * kCopies <= kSub * kSteps, "every wavefront copies, one after a product");
    __shared__ __attribute__((aligned(1024))) uint8_t s_k0[kTile], s_v0[kTile], s_k1[kTile], s_v1[kTile];
    // Heads of 256: every fourth 16 dimensions of the rows wait in LDS (two workgroups then take all of a compute
    // unit's): with all of them in registers there are too few for anything else.
    constexpr int kWaiting = D == 256 ? 4 : 0;
    __shared__ __attribute__((aligned(16))) uint8_t s_q[kWaiting ? kWaves * kWaiting * 1024 : 16];
    // Two wavefronts of different workgroups share a SIMD, and the older one goes first where both could: priorities in
    // the keys' products, the softmax and the values' products keep them at different ones.  8192 rows and keys, without:
    // 16 heads of 256 526 us, now 484; 32 of 128 509 and 503 (4096: 146 and 137; with those of 256 140); of 64 298, with
    // either of the two 300 and 304.
    constexpr int kPriority[3] = {D == 256 ? 2 : 0, D == 256 ? 1 : 0, D == 128 ? 1 : 0};
    const PromptArgs &a = p.a;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64, r = l % 32, half = l / 32;
    const uint32_t tokens = 32u * kWaves / p.head_waves;  // of the workgroup
    Place at;
    const uint32_t number = number_of(p);
    if (!find_place(a, number / p.head_sets, tokens, at)) return;
    const uint32_t head = number % p.head_sets * p.head_waves + (uint32_t)wave % p.head_waves;
    const uint32_t kv = __builtin_amdgcn_readfirstlane(head / (a.q_heads / a.kv_heads));
    const int q0 = __builtin_amdgcn_readfirstlane(at.q0), lq = __builtin_amdgcn_readfirstlane(at.lq);
    const int k0 = __builtin_amdgcn_readfirstlane(at.k0), lk = __builtin_amdgcn_readfirstlane(at.lk);
    const int first = (int)(__builtin_amdgcn_readfirstlane(at.tile) * tokens), mine = first + 32 * (wave / (int)p.head_waves);
    const int shift = lk - lq;
    // rows past the end are zeros, see what the last one does and are not stored
    auto last_key = [&] {  // that the lane's row sees (with heads of 256 what a lane can make anew has no register)
        const int at = mine + here(l) % 32;
        return (at < lq ? at : lq - 1) + shift;
    };
    const int limit_min = (mine < lq ? mine : lq - 1) + shift;
    const int limit_max = (mine + 31 < lq ? mine + 31 : lq - 1) + shift;
    const int last = (first + (int)tokens < lq ? first + (int)tokens : lq) - 1 + shift;  // of the workgroup
    const bool live = mine < lq;
    // tiles of the part: [begin, end) of those that the workgroup's rows see
    const uint32_t tiles = last >= 0 ? (uint32_t)last / KT + 1 : 0, part = blockIdx.y, parts = gridDim.y;  // at most 2^26, 2^4
    const int begin = __builtin_amdgcn_readfirstlane(tiles * part / parts), end = __builtin_amdgcn_readfirstlane(tiles * (part + 1) / parts);

    f32x16 o[kDims];
#pragma unroll
    for (int i = 0; i < kDims; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    float m = -kInf, sum = 0.0f;
    uint32_t odd = 0;  // tiles, from the last one on, whose values are left to the end

    const uint8_t *const kp = reinterpret_cast<const uint8_t *>(static_cast<const uint16_t *>(a.k.d) + (size_t)k0 * a.k.row + (size_t)kv * a.k.head);
    const uint8_t *const vp = reinterpret_cast<const uint8_t *>(static_cast<const uint16_t *>(a.v.d) + (size_t)k0 * a.v.row + (size_t)kv * a.v.head);
    const uint32_t k_row = (uint32_t)a.k.row * 2, v_row = (uint32_t)a.v.row * 2;

    // Where the lane's operands are in a tile: chunk half of key r, and, transposed, dimensions l % 32 of the first keys
    // that its half's weights have.  Other chunks and dimensions are these with bits flipped (the swizzles depend on the
    // lane alone), other keys a constant further.  Made anew for each tile: no registers hold addresses.
    auto k_at = [&] {
        const uint32_t lane = here(l), row = lane % 32;
        return row * kRow + (lane / 32 ^ k_swizzle<D>(row)) * 16;
    };
    auto v_at = [&] {
        const uint32_t lane = here(l), row = 4 * (lane / 32) + lane % 16 / 4;
        return row * kRow + ((2 * (lane / 16 % 2) + lane % 4 / 2) ^ v_swizzle<D>(row)) * 16 + lane % 2 * 8;
    };

    // Copies of a tile: a wavefront's `i` takes 1 KiB, which is kCopyRows rows.  Its rows' swizzle is that of the first
    // copy's with constant bits flipped, and the rows' distance a scalar, so an offset is one instruction.  Scalar offsets
    // are not held against the descriptor's end: the sequence's last tile, whose rows may end, has whole ones (copy_last).
    constexpr int kCopyRows = 1024 / kRow, kRowLanes = kRow / 16;
    const int copy_rows = wave * kCopies * kCopyRows;  // those of the wavefronts before
    auto copy_last = [&](const uint8_t *from, uint32_t row_bytes, bool of_k, int kt, uint8_t *to) {
        const uint32_t rows = lk - kt * KT < KT ? lk - kt * KT : KT;
        const Desc d = make_desc(from + (size_t)kt * KT * row_bytes, (rows - 1) * row_bytes + kRow);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const uint32_t rr = copy_rows + i * kCopyRows + l / kRowLanes;
            copy16(d, rr * row_bytes + (l % kRowLanes ^ (of_k ? k_swizzle<D>(rr) : v_swizzle<D>(rr))) * 16, to + (wave * kCopies + i) * 1024);
        }
    };
    // A tile all of whose rows are there.  Before the part's first one there are none: nothing is in such a descriptor's
    // bounds, and zeros go to LDS.  No branch, so that the copies can stand among the products, one after each.
    struct Tile {
        Desc d;
        uint32_t step;          // from copy to copy
        uint32_t chunk, first;  // the lane's: 16 bytes of a row, and the row of the first copy
    };
    auto tile_at = [&](const uint8_t *from, uint32_t row_bytes, bool of_k, int kt) {
        const bool any = kt >= begin;
        const uint32_t lane = D == 256 ? here(l) : l, row = copy_rows + lane / kRowLanes;
        return Tile{make_desc(from + (size_t)(any ? kt : 0) * KT * row_bytes, any ? 0xFFFFFFFFu : 0), any ? kCopyRows * row_bytes : 0,
                    (lane % kRowLanes ^ (of_k ? k_swizzle<D>(row) : v_swizzle<D>(row))) * 16, lane / kRowLanes * row_bytes};
    };
    auto k_tile = [&](int kt) { return tile_at(kp, k_row, true, kt); };
    auto v_tile = [&](int kt) { return tile_at(vp, v_row, false, kt); };
    auto copy = [&](const Tile &t, bool of_k, int i, uint8_t *to) {
        const uint32_t n = wave * kCopies + i;
        copy16(t.d, (t.chunk ^ (of_k ? k_swizzle<D>(i * kCopyRows) : v_swizzle<D>(i * kCopyRows)) * 16) + t.first, n * t.step, to + n * 1024);
    };
    // The first tile is asked for before the rows.
    if (begin < end) {
        copy_last(kp, k_row, true, end - 1, s_k0);
        copy_last(vp, v_row, false, end - 1, s_v0);
    }
    bf16x8 q[kSteps];  // those that wait are not kept here
    auto waits = [](int i) { return kWaiting && i % 4 == 3; };
    uint8_t *const waiting = s_q + wave * kWaiting * 1024;
    {
        const uint32_t q_row = (uint32_t)a.q.row * 2, rows = live ? (lq - mine < 32 ? lq - mine : 32) : 0, q_at = r * q_row + half * 16;
        const Desc from = make_desc(static_cast<const uint16_t *>(a.q.d) + (size_t)(q0 + mine) * a.q.row + (size_t)head * a.q.head,
                                    rows ? (rows - 1) * q_row + D * 2 : 0);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            if (waits(i)) copy16(from, q_at + i * 32, waiting + i / 4 * 1024);
            else q[i] = __builtin_bit_cast(bf16x8, read16(from, q_at + i * 32));
        }
    }
    auto values = [&](const uint8_t *sv, uint32_t v0, int j, int st, int d) {
        const uint8_t *at_v = sv + (v0 ^ (d % 4 * 64)) + (d / 4 * 256 + (j * 32 + st * 16) * kRow);
        const uint2 x = read_transposed(at_v), y = read_transposed(at_v + 8 * kRow);
        return u32x4{x.x, x.y, y.x, y.y};
    };
    // Two stages of LDS, each a variable of its own: while a tile is worked on, the one before it comes.  publish(): this
    // wavefront's copies are there and its reads done, then the workgroup's.
    auto publish = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    // A tile at the end of what the workgroup's rows see: some of them may not see all of its keys.  Its stage is chosen
    // at run time, so the compiler cannot tell it from the one that is being copied to, and waits for the tile before
    // in front of the values' reads.
    auto edge_scores = [&](const uint8_t *sk, f32x16 (&s)[kSub]) {
        const uint32_t k0_at = k_at();
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
            f32x16 acc = {};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const bf16x8 k = *reinterpret_cast<const bf16x8 *>(sk + (k0_at ^ (i % 8 * 32)) + (i / 8 * 256 + j * 32 * kRow));
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, waits(i) ? *reinterpret_cast<const bf16x8 *>(waiting + i / 4 * 1024 + l * 16) : q[i], acc, 0, 0, 0);
            }
            s[j] = acc;
        }
    };
    auto edge_step = [&](f32x16 (&s)[kSub], const uint8_t *sv, int kt) {
        const bool part = kt * KT + KT - 1 > limit_min;  // some row of the wavefront
        if (part) {
            const int limit = last_key();
#pragma unroll
            for (int j = 0; j < kSub; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (kt * KT + j * 32 + 8 * (i / 4) + 4 * half + i % 4 > limit) s[j][i] = -kInf;
        }
        float top = s[0][0];
#pragma unroll
        for (int j = 0; j < kSub; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[j][i]);
        top = other_half_max(top) * p.scale_log2;
        if (__any(top > m + kSlack)) {
            const float m_new = fmaxf(m, top), keep = m_new == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            sum *= keep;
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= keep;
        }
        const float m_use = m == -kInf ? 0.0f : m;
        bf16x8 w[kSub][2];
#pragma unroll
        for (int j = 0; j < kSub; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][i], p.scale_log2, -m_use));
                sum += e;
                w[j][i / 8][i % 8] = (__bf16)e;
            }
        if (part) {
            u16x2 most = {0, 0};  // largest magnitudes among values that some rows do not see
#pragma unroll 4
            for (int i = 0; i < kTile / 1024; ++i) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(sv + i * 1024 + l * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, x[e] & 0x7FFF7FFFu));
            }
            if (__any(most[0] >= 0x7F80 || most[1] >= 0x7F80)) {
                odd |= 1u << (last / KT - kt);
                return;
            }
        }
        const uint32_t v0_at = v_at();
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int j = 0; j < kSub; ++j)
#pragma unroll
                for (int st = 0; st < 2; ++st)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, values(sv, v0_at, j, st, d)), w[j][st], o[d], 0, 0, 0);
    };

    // A tile all of whose keys all rows see, and the copies of the one before it.
    auto step = [&](const uint8_t *sk, const uint8_t *sv, uint8_t *other_k, uint8_t *other_v, int kt) {
        // The order of the instructions is set by hand here and below: reads go kAhead products ahead, and the copies'
        // and the exponentials' instructions stand between the products, in their shadow.
        f32x16 s[kSub];
        const uint32_t k0_at = k_at();
        Tile next = k_tile(kt - 1);
        auto keys = [&](int n) {
            const int j = n / kSteps, i = n % kSteps;
            return *reinterpret_cast<const bf16x8 *>(sk + (k0_at ^ (i % 8 * 32)) + (i / 8 * 256 + j * 32 * kRow));
        };
        bf16x8 ahead_k[kAhead], waited = {};
        __builtin_amdgcn_s_setprio(kPriority[0]);
#pragma unroll
        for (int n = 0; n < kAhead; ++n) ahead_k[n] = keys(n);
#pragma unroll
        for (int n = 0; n < kSub * kSteps; ++n) {
            __builtin_amdgcn_sched_barrier(0);
            const f32x16 zero = {};
            s[n / kSteps] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ahead_k[n % kAhead], waits(n % kSteps) ? waited : q[n % kSteps],
                                                                    n % kSteps ? s[n / kSteps] : zero, 0, 0, 0);
            if (kWaiting && n % 4 == 0) waited = *reinterpret_cast<const bf16x8 *>(waiting + n % kSteps / 4 * 1024 + here(l) * 16);
            if (n + kAhead < kSub * kSteps) ahead_k[n % kAhead] = keys(n + kAhead);
            if (n == kCopies) next = v_tile(kt - 1);
            if (n < kCopies) copy(next, true, n, other_k);
            else if (n < 2 * kCopies) copy(next, false, n - kCopies, other_v);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(kPriority[1]);
        float top = s[0][0];
#pragma unroll
        for (int j = 0; j < kSub; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[j][i]);
        top = other_half_max(top) * p.scale_log2;
        if (__any(top > m + kSlack)) {
            const float m_new = fmaxf(m, top), keep = m_new == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            sum *= keep;
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= keep;
        }
        const float m_use = m == -kInf ? 0.0f : m;
        auto weight = [&](int g, int i) {  // of the group's 8 keys
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g / 2][g % 2 * 8 + i], p.scale_log2, -m_use));
            sum += e;
            return (__bf16)e;
        };
        // 16 keys at a time; the next ones' exponentials are between these ones' products
        constexpr int kGroups = kSub * 2, kEach = 8 / kDims;
        const uint32_t v0_at = v_at();
        u32x4 ahead_v[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) ahead_v[n] = values(sv, v0_at, n / kDims / 2, n / kDims % 2, n % kDims);
        bf16x8 w[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[0][i] = weight(0, i);
        __builtin_amdgcn_s_setprio(kPriority[2]);
#pragma unroll
        for (int n = 0; n < kGroups * kDims; ++n) {
            const int g = n / kDims, d = n % kDims, then = n + kAhead;
            __builtin_amdgcn_sched_barrier(0);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, ahead_v[n % kAhead]), w[g % 2], o[d], 0, 0, 0);
            if (then < kGroups * kDims) ahead_v[n % kAhead] = values(sv, v0_at, then / kDims / 2, then / kDims % 2, then % kDims);
            if (g + 1 < kGroups) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) w[(g + 1) % 2][d * kEach + i] = weight(g + 1, d * kEach + i);
            }
        }
    };

    if (begin < end) {
        int kt = end - 1;
        auto copy_before = [&](uint8_t *other_k, uint8_t *other_v) {
            const Tile k = k_tile(kt - 1), v = v_tile(kt - 1);
#pragma unroll
            for (int i = 0; i < kCopies; ++i) copy(k, true, i, other_k), copy(v, false, i, other_v);
        };
        const int edge = (first + shift + 1 > 0 ? first + shift + 1 : 0) / KT;  // all rows see all of the tiles before this
        bool second = false;
        for (; kt >= edge && kt >= begin; --kt) {
            publish();
            copy_before(second ? s_k0 : s_k1, second ? s_v0 : s_v1);
            if (live && kt * KT <= limit_max) {
                f32x16 s[kSub];
                edge_scores(second ? s_k1 : s_k0, s);
                edge_step(s, second ? s_v1 : s_v0, kt);
            }
            second = !second;
        }
        auto whole = [&](const uint8_t *sk, const uint8_t *sv, uint8_t *other_k, uint8_t *other_v) {
            __builtin_amdgcn_s_setprio(0);
            publish();
            if (live) step(sk, sv, other_k, other_v, kt);
            else copy_before(other_k, other_v);
            --kt;
        };
        if (second && kt >= begin) whole(s_k1, s_v1, s_k0, s_v0);
        while (kt >= begin) {
            whole(s_k0, s_v0, s_k1, s_v1);
            if (kt < begin) break;
            whole(s_k1, s_v1, s_k0, s_v0);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // copies to LDS, also where no tile waited for them

    // Tiles with infinities or NaN that only some rows see: key by key.
    while (odd) {
        const int kt = last / KT - __builtin_ctz(odd);
        odd &= odd - 1;
#pragma unroll 1
        for (int key = kt * KT; key < (kt * KT + KT < lk ? kt * KT + KT : lk); ++key) {
            const uint16_t *kr = reinterpret_cast<const uint16_t *>(kp + (size_t)key * k_row) + half * 8;
            float dot = 0.0f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const bf16x8 x = *reinterpret_cast<const bf16x8 *>(kr + i * 16);
                const bf16x8 z = waits(i) ? *reinterpret_cast<const bf16x8 *>(waiting + i / 4 * 1024 + l * 16) : q[i];
#pragma unroll
                for (int e = 0; e < 8; ++e) dot = __builtin_fmaf((float)x[e], (float)z[e], dot);
            }
            dot += __shfl_xor(dot, 32);
            if (key > last_key()) continue;
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(dot, p.scale_log2, m == -kInf ? 0.0f : -m));
            const uint16_t *vr = reinterpret_cast<const uint16_t *>(vp + (size_t)key * v_row) + half * 4;
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    o[d][i] = __builtin_fmaf(e, __uint_as_float((uint32_t)vr[d * 32 + 8 * (i / 4) + i % 4] << 16), o[d][i]);
        }
    }

    // Rows leave through LDS (the tiles' place, a stage for each wavefront), so that neighbouring lanes have
    // neighbouring bytes of a row: [row][chunk of 4 at chunk ^ row], kOut dimensions at a time.
    constexpr int kOut = kTile / 128, kLanes = kOut / 8;  // lanes of a row
    __syncthreads();
    if (!live) return;
    uint8_t *const out = wave == 0 ? s_k0 : wave == 1 ? s_v0 : wave == 2 ? s_k1 : s_v1;
    sum += __shfl_xor(sum, 32);
    const float inv = parts > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint32_t no_keys = (uint32_t)__ballot(sum == 0.0f);  // of 32 rows
    const size_t first_row = (size_t)(q0 + mine);
    const int rows = lq - mine < 32 ? lq - mine : 32, lane = here(l), row_of = lane / kLanes, at_dim = lane % kLanes * 8;
    if (parts > 1 && half == 0 && r < rows) {
        float *const to = p.top_sum + (((size_t)part * a.total_q + first_row + r) * a.q_heads + head) * 2;
        to[0] = m, to[1] = sum;
    }
    // Rows behind the sequence's end are behind the descriptors' too: neither read nor written, and no branches, which
    // would make every row wait for its own reads (heads of 256: 3.2 us instead of 2.2, of 37 rows 12.4 and 11.1).
    auto leave = [&](auto gated, auto whole) {
        const uint32_t y_row = a.q_heads * D * (whole ? 2 : 4), gate_row = (uint32_t)a.gate.row * 2;
        const size_t place = (first_row * a.q_heads + head) * D;
        const uint32_t y_at = row_of * y_row + at_dim * (whole ? 2 : 4), gate_at = row_of * gate_row + at_dim * 2;
#pragma unroll
        for (int piece = 0; piece < D / kOut; ++piece) {
#pragma unroll
            for (int d = 0; d < kOut / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = o[piece * (kOut / 32) + d][i + e] * inv;
                    const int c = d * 8 + 2 * (i / 4) + half;
                    *reinterpret_cast<f32x4 *>(out + r * (kOut * 4) + (c ^ (r & (kOut / 4 - 1))) * 16) = v;
                }
            constexpr int kSets = 32 * kLanes / 64, kSetRows = 64 / kLanes;
            u32x4 g[kSets] = {};
            if constexpr (gated) {
                const Desc from = make_desc(static_cast<const uint16_t *>(a.gate.d) + first_row * a.gate.row + (size_t)head * a.gate.head, (rows - 1) * gate_row + D * 2);
#pragma unroll
                for (int i = 0; i < kSets; ++i) g[i] = read16(from, gate_at + i * kSetRows * gate_row + piece * (kOut * 2));
            }
            const Desc to = whole ? make_desc(a.y + place, (rows - 1) * y_row + D * 2)
                                  : make_desc(p.o + (size_t)part * a.total_q * a.q_heads * D + place, (rows - 1) * y_row + D * 4);
#pragma unroll
            for (int i = 0; i < kSets; ++i) {
                const int rr = i * kSetRows + row_of, c = at_dim / 4;
                f32x4 x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) x[e] = *reinterpret_cast<const f32x4 *>(out + rr * (kOut * 4) + ((c + e) ^ (rr & (kOut / 4 - 1))) * 16);
                const uint32_t at = y_at + i * kSetRows * y_row + piece * (kOut * (whole ? 2 : 4));
                if constexpr (whole) {
                    float v[8] = {x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]};
                    if (gated) apply_gate(v, g[i] & ((no_keys >> rr & 1) - 1));  // a row without keys is 0, also where its gate is NaN
                    write16(to, at, bf16_row(v));
                } else {
                    write16(to, at, __builtin_bit_cast(u32x4, x[0]));
                    write16(to, at + 16, __builtin_bit_cast(u32x4, x[1]));
                }
            }
        }
    };
    if (parts > 1) leave(std::false_type{}, std::false_type{});
    else if (a.gate.d) leave(std::true_type{}, std::true_type{});
    else leave(std::false_type{}, std::true_type{});
}

// Joins the parts: what each summed counts exp2(its maximum - the largest).  A wavefront has as many of the rows of one
// of the parts' as it can read at once, 8 dimensions to a lane.
template <int D>
__global__ __launch_bounds__(64 * kWaves) void prompt_join_kernel(Kernel p, int parts) {
    constexpr int kLanes = D / 8, kRows = 64 / kLanes, kAtOnce = 8;
    const PromptArgs &a = p.a;
    const int wave = threadIdx.x / 64, l = threadIdx.x % 64;
    const uint32_t tokens = 32u * kWaves / p.head_waves, number = number_of(p);
    Place at;
    if (!find_place(a, number / p.head_sets, tokens, at)) return;
    const uint32_t head = number % p.head_sets * p.head_waves + (uint32_t)wave % p.head_waves;
    const int mine = (int)(at.tile * tokens) + 32 * (wave / (int)p.head_waves);
    const int i = blockIdx.y * kRows + l / kLanes;
    if (mine + i < at.lq) {
        const size_t row = ((size_t)(at.q0 + mine + i)) * a.q_heads + head, step = (size_t)a.total_q * a.q_heads;
        const int at_dim = l % kLanes * 8;
        float top = -kInf, sum = 0.0f, v[8] = {};
        for (int n0 = 0; n0 < parts; n0 += kAtOnce) {
            float2 ms[kAtOnce];
            f32x4 x[kAtOnce][2];
            float most = top;
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const size_t n = n0 + u < parts ? n0 + u : parts - 1;
                ms[u] = *reinterpret_cast<const float2 *>(p.top_sum + (n * step + row) * 2);
#pragma unroll
                for (int e = 0; e < 2; ++e) x[u][e] = *reinterpret_cast<const f32x4 *>(p.o + (n * step + row) * D + at_dim + 4 * e);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) most = fmaxf(most, ms[u].x);
            // without a maximum there are zeros, or NaN, which stay
            const float keep = top == -kInf ? 1.0f : __builtin_amdgcn_exp2f(top - most);
            top = most;
            sum *= keep;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= keep;
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                if (n0 + u >= parts) break;
                const float take = ms[u].x == -kInf ? 1.0f : __builtin_amdgcn_exp2f(ms[u].x - top);
                sum = __builtin_fmaf(ms[u].y, take, sum);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(x[u][e / 4][e % 4], take, v[e]);
            }
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= inv;
        if (a.gate.d && sum != 0.0f)
            apply_gate(v, *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.gate.d) + (size_t)(at.q0 + mine + i) * a.gate.row +
                                                            (size_t)head * a.gate.head + at_dim));
        *reinterpret_cast<u32x4 *>(a.y + row * D + at_dim) = bf16_row(v);
    }
}

// How the work is cut: workgroups, and parts that each one's keys are dealt into.
struct Cutting {
    uint32_t head_waves, head_sets, groups, parts;
};
Cutting cutting_of(const PromptArgs &a) {
    Cutting c{1, 0, 0, 1};
    const uint32_t group = a.q_heads / a.kv_heads;
    while (c.head_waves < kWaves && group % (c.head_waves * 2) == 0) c.head_waves *= 2;
    c.head_sets = a.q_heads / c.head_waves;
    // Groups of 1, 3, 7: all wavefronts have rows of one head, 128 of them, and the heads of a group do not share tiles.
    // It costs nothing that is seen: 4096 rows of 28 heads of 128 on 4 131 us, of 32 on 8 142; 32 rows 7.7 and 8.0.
    const uint32_t tokens = 32 * kWaves / c.head_waves;
    c.groups = (uint32_t)(((uint64_t)a.total_q + (uint64_t)a.n_seqs * (tokens - 1)) / tokens) * c.head_sets;  // at least as many as there are
    // Few rows before many keys: a workgroup needs about 1 us for a tile, whatever else runs, the join 5 and what its
    // rows' bytes take.  Sequences (the usual one here: their lengths are the device's) of 12 tiles on average are cut as
    // long as every workgroup has a compute unit to itself, into parts of four tiles at least.  4096 keys, whole and in
    // parts: 32 rows of 16 heads of 256 124 us and 26 (sixteen; thirty-two 31), 512 rows 124 and 56 (four; eight 60), 2048
    // rows 137 (two 138); 32 rows of 32 of 128 67 and 18, 512 rows 69 and 51, 1024 rows 77 (two 81).  As many rows as
    // keys: 1024 of 256 39 and 38, 2048 of 256 71 (two 78), of 128 48 (two 68).
    const uint32_t keys = a.dim == 256 ? 32 : 64, tiles = a.total_k / a.n_seqs / keys, last = a.total_q / a.n_seqs / keys;
    const uint32_t usual = tiles - (last < tiles ? last : tiles) / 2, units = (uint32_t)cu_count() / c.groups;
    if (usual >= 12 && units > 1) {
        c.parts = units < usual / 4 ? units : usual / 4;
        if (c.parts > kMaxParts) c.parts = kMaxParts;
    }
    // A workgroup stops looking at the 64 sequences that have its tile.  The totals may allow for no more tiles than there
    // are, so one more goes through all of the sequences, whose bounds may be wrong behind the last tile too.
    if (a.n_seqs > 64) c.groups += c.head_sets;
    return c;
}

template <int D, int KT>
hipError_t launch_for(hipStream_t s, const Kernel &p, const Cutting &cut) {
    prompt_kernel<D, KT><<<dim3(cut.groups, cut.parts), dim3(64 * kWaves), 0, s>>>(p);
    if (cut.parts > 1) {
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        prompt_join_kernel<D><<<dim3(cut.groups, 32 * D / 512), dim3(64 * kWaves), 0, s>>>(p, (int)cut.parts);
    }
    return hipGetLastError();
}

}  // namespace

size_t attn_prompt_scratch_bytes(const PromptArgs &a) {
    const Cutting cut = cutting_of(a);
    return cut.parts == 1 ? 0 : (size_t)cut.parts * a.total_q * a.q_heads * (a.dim + 2) * 4;
}

hipError_t launch_attn_prompt(hipStream_t s, const PromptArgs &a, void *scratch) {
    const Cutting cut = cutting_of(a);
    Kernel p{a, cut.head_waves, cut.head_sets, 0, a.scale * kLog2e, nullptr, nullptr};
    if (cut.parts > 1) {
        p.o = static_cast<float *>(scratch);
        p.top_sum = p.o + (size_t)cut.parts * a.total_q * a.q_heads * a.dim;
    }
    // Tiles of a prompt begin with the longest, and what is free first takes the next.  Where all run at once, two to
    // a compute unit, the second of each comes from the end, so that their sums are alike.
    const uint32_t cus = (uint32_t)cu_count();
    p.turn = a.n_seqs == 1 && cut.groups > cus && cut.groups <= 2 * cus ? cus : cut.groups;
    if (a.dim == 64) return launch_for<64, 64>(s, p, cut);
    if (a.dim == 128) return launch_for<128, 64>(s, p, cut);
    return launch_for<256, 32>(s, p, cut);
}

}  // namespace tqf
