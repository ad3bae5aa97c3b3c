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
// grouped, are heads of one group at the same rows.
//
// Keys that a row does not see have weight 0, but 0 * inf and 0 * NaN are NaN.
// Rows behind a sequence's end read as zeros (the copies' bounds).  Tiles that some
// rows see in part are looked through for infinities and NaN; where there are any,
// the tile's values are added at the end, key by key, to the rows that see them.
#include <hip/hip_runtime.h>

#include "tqf_attn_device.h"

namespace tqf {

namespace {

constexpr int kWaves = 4;
constexpr int kAhead = 4;  // products that LDS reads go ahead of theirs
struct Kernel {
    PromptArgs a;
    uint32_t head_waves;  // wavefronts of a workgroup that have heads of their own (of one group)
    uint32_t head_sets;   // q_heads / head_waves
    uint32_t turn;        // workgroups from here on are taken from the end
    float scale_log2;
};

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
    const PromptArgs &a = p.a;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64, r = l % 32, half = l / 32;
    const uint32_t tokens = 32u * kWaves / p.head_waves;  // of the workgroup
    Place at;
    const uint32_t number = blockIdx.x < p.turn ? blockIdx.x : gridDim.x - 1 - (blockIdx.x - p.turn);
    if (!find_place(a, number / p.head_sets, tokens, at)) return;
    const uint32_t head = number % p.head_sets * p.head_waves + (uint32_t)wave % p.head_waves;
    const uint32_t kv = __builtin_amdgcn_readfirstlane(head / (a.q_heads / a.kv_heads));
    const int q0 = __builtin_amdgcn_readfirstlane(at.q0), lq = __builtin_amdgcn_readfirstlane(at.lq);
    const int k0 = __builtin_amdgcn_readfirstlane(at.k0), lk = __builtin_amdgcn_readfirstlane(at.lk);
    const int first = (int)(__builtin_amdgcn_readfirstlane(at.tile) * tokens), mine = first + 32 * (wave / (int)p.head_waves);
    const int shift = lk - lq;
    const int row = mine + r < lq ? mine + r : lq - 1;  // rows past the end do as the last one and are not stored
    const int limit = row + shift;                       // the last key that the lane's row sees
    const int limit_min = (mine < lq ? mine : lq - 1) + shift;
    const int limit_max = (mine + 31 < lq ? mine + 31 : lq - 1) + shift;
    const int last = (first + (int)tokens < lq ? first + (int)tokens : lq) - 1 + shift;  // of the workgroup
    const bool live = mine < lq;

    bf16x8 q[kSteps];  // those that wait are not kept here
    auto waits = [](int i) { return kWaiting && i % 4 == 3; };
    uint8_t *const waiting = s_q + wave * kWaiting * 1024;
    const uint16_t *qp = static_cast<const uint16_t *>(a.q.d) + (size_t)(q0 + row) * a.q.row + (size_t)head * a.q.head + half * 8;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const bf16x8 x = *reinterpret_cast<const bf16x8 *>(qp + i * 16);
        if (waits(i)) *reinterpret_cast<bf16x8 *>(waiting + i / 4 * 1024 + l * 16) = x;
        else q[i] = x;
    }
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
    const uint32_t copy_row = l / kRowLanes, copy_tile_row = wave * kCopies * kCopyRows + copy_row;
    const uint32_t k_chunk = (l % kRowLanes ^ k_swizzle<D>(copy_tile_row)) * 16, v_chunk = (l % kRowLanes ^ v_swizzle<D>(copy_tile_row)) * 16;
    const uint32_t k_first = copy_row * k_row, v_first = copy_row * v_row;
    auto copy_last = [&](const uint8_t *from, uint32_t row_bytes, bool of_k, int kt, uint8_t *to) {
        const uint32_t rows = lk - kt * KT < KT ? lk - kt * KT : KT;
        const Desc d = make_desc(from + (size_t)kt * KT * row_bytes, (rows - 1) * row_bytes + kRow);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const uint32_t rr = copy_tile_row + i * kCopyRows;
            copy16(d, rr * row_bytes + (l % kRowLanes ^ (of_k ? k_swizzle<D>(rr) : v_swizzle<D>(rr))) * 16, to + (wave * kCopies + i) * 1024);
        }
    };
    // A tile all of whose rows are there.  Before the first one there are none: nothing is in such a descriptor's bounds,
    // and zeros go to LDS.  No branch, so that the copies can stand among the products, one after each.
    struct Tile {
        Desc d;
        uint32_t step;  // from copy to copy
    };
    auto tile_at = [&](const uint8_t *from, uint32_t row_bytes, int kt) {
        return Tile{make_desc(from + (size_t)(kt < 0 ? 0 : kt) * KT * row_bytes, kt < 0 ? 0 : 0xFFFFFFFFu), kt < 0 ? 0 : kCopyRows * row_bytes};
    };
    auto copy_k = [&](const Tile &t, int i, uint8_t *to) {
        const uint32_t n = wave * kCopies + i;
        copy16(t.d, (here(k_chunk) ^ k_swizzle<D>(i * kCopyRows) * 16) + k_first, n * t.step, to + n * 1024);
    };
    auto copy_v = [&](const Tile &t, int i, uint8_t *to) {
        const uint32_t n = wave * kCopies + i;
        copy16(t.d, (here(v_chunk) ^ v_swizzle<D>(i * kCopyRows) * 16) + v_first, n * t.step, to + n * 1024);
    };
    auto values = [&](const uint8_t *sv, uint32_t v0, int j, int st, int d) {
        const uint8_t *at_v = sv + (v0 ^ (d % 4 * 64)) + (d / 4 * 256 + (j * 32 + st * 16) * kRow);
        const uint2 x = read_transposed(at_v), y = read_transposed(at_v + 8 * kRow);
        return u32x4{x.x, x.y, y.x, y.y};
    };
    // Two stages of LDS, each a variable of its own: while a tile is worked on, the one before it comes.  publish(): this
    // wavefront's copies are there and its reads done, then the workgroup's.
    auto publish = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    // A tile at the end of what the workgroup's rows see: some of them may not see all of its keys.
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
        const Tile next_k = tile_at(kp, k_row, kt - 1), next_v = tile_at(vp, v_row, kt - 1);
        auto keys = [&](int n) {
            const int j = n / kSteps, i = n % kSteps;
            return *reinterpret_cast<const bf16x8 *>(sk + (k0_at ^ (i % 8 * 32)) + (i / 8 * 256 + j * 32 * kRow));
        };
        bf16x8 ahead_k[kAhead], waited = {};
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
            if (n < kCopies) copy_k(next_k, n, other_k);
            else if (n < 2 * kCopies) copy_v(next_v, n - kCopies, other_v);
        }
        __builtin_amdgcn_sched_barrier(0);
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

    if (last >= 0) {
        int kt = last / KT;
        copy_last(kp, k_row, true, kt, s_k0);
        copy_last(vp, v_row, false, kt, s_v0);
        auto copy_before = [&](uint8_t *other_k, uint8_t *other_v) {
            const Tile k = tile_at(kp, k_row, kt - 1), v = tile_at(vp, v_row, kt - 1);
#pragma unroll
            for (int i = 0; i < kCopies; ++i) copy_k(k, i, other_k), copy_v(v, i, other_v);
        };
        const int edge = (first + shift + 1 > 0 ? first + shift + 1 : 0) / KT;  // all rows see all of the tiles before this
        bool second = false;
        for (; kt >= edge; --kt) {
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
            publish();
            if (live) step(sk, sv, other_k, other_v, kt);
            else copy_before(other_k, other_v);
            --kt;
        };
        if (second && kt >= 0) whole(s_k1, s_v1, s_k0, s_v0);
        while (kt >= 0) {
            whole(s_k0, s_v0, s_k1, s_v1);
            if (kt < 0) break;
            whole(s_k1, s_v1, s_k0, s_v0);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }

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
            if (key > limit) continue;
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
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const size_t first_row = (size_t)(q0 + mine);
    const int rows = lq - mine < 32 ? lq - mine : 32, lane = here(l), row_of = lane / kLanes, at_dim = lane % kLanes * 8;
    uint16_t *const y = a.y + (first_row * a.q_heads + head) * D + at_dim;
    const uint16_t *const gate = static_cast<const uint16_t *>(a.gate.d) + first_row * a.gate.row + (size_t)head * a.gate.head + at_dim;
#pragma unroll
    for (int part = 0; part < D / kOut; ++part) {
#pragma unroll
        for (int d = 0; d < kOut / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = o[part * (kOut / 32) + d][i + e] * inv;
                const int c = d * 8 + 2 * (i / 4) + half;
                *reinterpret_cast<f32x4 *>(out + r * (kOut * 4) + (c ^ (r & (kOut / 4 - 1))) * 16) = v;
            }
        u32x4 g[32 * kLanes / 64];
        if (a.gate.d) {
#pragma unroll
            for (int i = 0; i < 32 * kLanes / 64; ++i) {
                const int rr = i * (64 / kLanes) + row_of;
                g[i] = *reinterpret_cast<const u32x4 *>(gate + (size_t)(rr < rows ? rr : 0) * a.gate.row + part * kOut);
            }
        }
#pragma unroll
        for (int i = 0; i < 32 * kLanes / 64; ++i) {
            const int rr = i * (64 / kLanes) + row_of, c = at_dim / 4;
            float v[8];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const f32x4 x = *reinterpret_cast<const f32x4 *>(out + rr * (kOut * 4) + ((c + e) ^ (rr & (kOut / 4 - 1))) * 16);
#pragma unroll
                for (int u = 0; u < 4; ++u) v[4 * e + u] = x[u];
            }
            if (a.gate.d) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[2 * e] *= sigmoid(__uint_as_float(g[i][e] << 16));
                    v[2 * e + 1] *= sigmoid(__uint_as_float(g[i][e] & 0xFFFF0000u));
                }
            }
            if (rr < rows) {
                const u32x4 bits = {bf16_bits2(v[0], v[1]), bf16_bits2(v[2], v[3]), bf16_bits2(v[4], v[5]), bf16_bits2(v[6], v[7])};
                *reinterpret_cast<u32x4 *>(y + (size_t)rr * a.q_heads * D + part * kOut) = bits;
            }
        }
    }
}

}  // namespace

hipError_t launch_attn_prompt(hipStream_t s, const PromptArgs &a) {
    Kernel p{a, 1, 0, 0, a.scale * kLog2e};
    const uint32_t group = a.q_heads / a.kv_heads;
    while (p.head_waves < kWaves && group % (p.head_waves * 2) == 0) p.head_waves *= 2;
    p.head_sets = a.q_heads / p.head_waves;
    const uint32_t tokens = 32 * kWaves / p.head_waves;
    const uint64_t tiles = (uint64_t)a.total_q / tokens + a.n_seqs;  // at least as many as there are
    const dim3 grid((uint32_t)(tiles * p.head_sets)), block(64 * kWaves);
    // Tiles of a prompt begin with the longest, and what is free first takes the next.  Where all run at once, two to
    // a compute unit, the second of each comes from the end, so that their sums are alike.
    const uint32_t cus = (uint32_t)cu_count();
    p.turn = a.n_seqs == 1 && grid.x > cus && grid.x <= 2 * cus + p.head_sets ? cus : grid.x;
    if (a.dim == 64) prompt_kernel<64, 64><<<grid, block, 0, s>>>(p);
    if (a.dim == 128) prompt_kernel<128, 64><<<grid, block, 0, s>>>(p);
    if (a.dim == 256) prompt_kernel<256, 32><<<grid, block, 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace tqf
