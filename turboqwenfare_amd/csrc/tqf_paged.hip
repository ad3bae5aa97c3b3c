// tqf_paged.hip -- attention of a few rows of every sequence (a token, or the verify
// rows of its drafts) over a paged cache in bf16 or e4m3 (gfx950).
//
//   y[i][h] = sum_j softmax_j(scale q[i][h] . k[j][h / group]) v[j][h / group]
//             (* sigmoid(gate[i][h])),  j < len - rows + i + 1.
//
// Bound by the cache's bytes: the rows of a sequence and the heads of a group stand
// side by side as the columns of the matrix instructions, up to 32 to a workgroup, so
// a key is multiplied with all of them when it arrives.  With more columns every 32
// have workgroups of their own, which read the cache again (64 sequences of 50..8192
// tokens, heads of 256, 4 rows of a group of 8: 53 us, 8 rows 75).  The work
// of all sequences, in steps of 128 keys of one (sequence, key head), is one line
// that is cut into equal parts, a part to a workgroup, whatever the lengths; what a
// workgroup has of a (sequence, key head) that it does not have whole goes to
// memory (maximum, sum, sum of values) and a second kernel joins it, in the order of
// the keys.  Wavefronts take 32 keys of a step each, by themselves, and join theirs
// in LDS at the end.
//
// One sequence of 131072 tokens (2 key heads of 256, bf16) takes 59 us, of which the
// join 7: 4.5 TB/s; 256 of 4000 (8 heads of 128) 713 us, 5.9 TB/s, as fast as reads
// go on this card.  Between them stand the join and, with sequences of many lengths,
// what each costs beside its bytes (64 of 50..8192 tokens, 4 rows: 53 us, 3.6 TB/s).
//
// As in tqf_prompt.hip: S^T = K Q^T (here 16 x 16 x 32) leaves a row's weights as an
// operand of O^T = V^T P^T; V^T comes from LDS by transposing reads; infinities and
// NaN among values that only some rows see are added at the end, key by key.
#include <hip/hip_runtime.h>

#include "tqf_attn_device.h"

namespace tqf {

namespace {

// Page numbers are read by scalar loads: a vector load's wait would be one for the copies too.
typedef __attribute__((address_space(4))) int32_t constant_i32;
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

// This wavefront's loads (those to LDS among them) but the last N are done.
template <int N>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Its LDS reads are.
__device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

constexpr int kWaves = 4, kWaveKeys = 32, kStepKeys = kWaves * kWaveKeys;

// What the join needs to know of a (sequence, key head) that several parts have: kept
// by the part that begins it.
struct Cut {
    uint32_t seq, kv, first, parts;  // parts 0: none is cut here
};

struct Kernel {
    PagedArgs a;
    uint32_t group, row_blocks, parts, page_shift;  // parts: workgroups of a row block
    uint32_t of_group;                              // 2^20 / group, and one
    float scale_log2;
    uint32_t extra;  // what a (sequence, key head) costs beside its steps, in steps
    bool by_unit;    // cuts [n_seqs x kv_heads], where those are fewer, else [parts]
    Cut *cuts;
    float *partial;  // [2 parts][row_blocks][rows of a block][dim + 2]: values, maximum, sum
};

// row / group.  Rows are fewer than 2^11 and a group is at most 2^8, so what is too much in row * of_group is below 2^20.
__device__ __forceinline__ uint32_t query_of(const Kernel &p, uint32_t row) { return row * p.of_group >> 20; }

// Steps of a sequence's one key head: at least one, which writes the rows of an empty sequence.
__device__ __forceinline__ uint32_t steps_of(const PagedArgs &a, int32_t len) {
    const bool bad = len < 0 || (uint64_t)len > (uint64_t)a.max_pages * a.cache.page;
    const uint32_t n = bad ? 0 : ((uint32_t)len + kStepKeys - 1) / kStepKeys;
    return n ? n : 1;
}

constexpr uint32_t kMostExtra = 2;
// The line of all steps: sequence by sequence, key head by key head; fewer than 2^31
// (the caller has checked the most there can be).  Before the steps of each stand
// `extra` places for what beginning and ending it costs: without them a part of
// many short sequences takes longer than one of a long one (64 sequences of 50 to
// 8192 tokens, 4 rows of 16 heads of 256: 69 us without, 58 with one place, 54 with
// two, 55 with three; 96 in e4m3, 32 heads of 128: 89, 75 and 76; 64 rows of 16 heads
// of 256: one 55, two 53, but 200 of 20 to 2000 tokens 50 and 52; one long sequence:
// 60 in any case).  All results
// are the same in every lane, and the compiler is told so: descriptors made of them
// stay scalar.
struct Line {
    uint32_t mine, upto;  // of sequence `lane`: places of a key head; places of all heads of the sequences up to it
    uint32_t total;
};
__device__ __forceinline__ uint32_t steps_up_to(uint32_t mine) {
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const uint32_t v = __shfl_up(upto, o);
        if ((int)(threadIdx.x & 63) >= o) upto += v;
    }
    return upto;
}
__device__ __forceinline__ Line line_of(const PagedArgs &a, uint32_t extra) {
    const uint32_t l = threadIdx.x & 63;
    Line line;
    line.mine = l < a.n_seqs ? steps_of(a, a.lens[l]) + extra : 0;
    uint32_t rest = 0;
    for (uint32_t s = l + 64; s < a.n_seqs; s += 64) rest += steps_of(a, a.lens[s]) + extra;
    line.upto = steps_up_to(line.mine * a.cache.kv_heads);
    line.total = __builtin_amdgcn_readlane(line.upto, 63);
    if (a.n_seqs > 64) {
#pragma unroll
        for (int o = 32; o >= 1; o /= 2) rest += __shfl_xor(rest, o);
        line.total += __builtin_amdgcn_readfirstlane(rest) * a.cache.kv_heads;
    }
    return line;
}
struct Place {
    uint32_t seq, places, first;  // a sequence, its places for a key head, its first place
};
__device__ __forceinline__ Place place_of(const PagedArgs &a, const Line &line, uint32_t extra, uint32_t place) {
    const uint32_t l = threadIdx.x & 63;
    uint32_t before = 0, mine = line.mine, upto = line.upto;
    for (uint32_t s0 = 0;;) {
        const uint64_t past = __ballot(before + upto > place);
        if (past) {
            const int who = __builtin_ctzll(past);
            const uint32_t n = __builtin_amdgcn_readlane(mine, who);
            return Place{s0 + who, n, before + __builtin_amdgcn_readlane(upto, who) - n * a.cache.kv_heads};
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        s0 += 64;
        if (s0 >= a.n_seqs) return Place{a.n_seqs, 1, 0};  // no such place
        mine = s0 + l < a.n_seqs ? steps_of(a, a.lens[s0 + l]) + extra : 0;
        upto = steps_up_to(mine * a.cache.kv_heads);
    }
}
// Equal parts, the first ones a place longer.
__device__ __forceinline__ uint32_t part_begin(uint32_t total, uint32_t part, uint32_t parts) {
    const uint32_t each = total / parts, more = total % parts;
    return part * each + (part < more ? part : more);
}
__device__ __forceinline__ uint32_t part_of(uint32_t total, uint32_t place, uint32_t parts) {
    const uint32_t each = total / parts, more = total % parts, longer = more * (each + 1);
    return place < longer ? place / (each + 1) : more + (place - longer) / (each ? each : 1);
}

__device__ __forceinline__ void four_bf16(const uint16_t *p, float (&v)[4]) {
    const uint2 b = *reinterpret_cast<const uint2 *>(p);
    v[0] = __uint_as_float(b.x << 16), v[1] = __uint_as_float(b.x & 0xFFFF0000u);
    v[2] = __uint_as_float(b.y << 16), v[3] = __uint_as_float(b.y & 0xFFFF0000u);
}
__device__ __forceinline__ float gate_of(uint16_t b) { return sigmoid(__uint_as_float((uint32_t)b << 16)); }

// Rows of the cache in LDS as the copies bring them, 16-byte chunk c of row r in slot
// c ^ its swizzle: the copies read whole rows, and both the 16 rows of which 16
// lanes read a chunk of keys and those that 32 lanes read transposed are in
// different places of the banks.  kPitch: bytes of a row.
template <int kPitch>
__device__ __forceinline__ uint32_t k_swizzle(uint32_t row) {
    return kPitch >= 256 ? row & 15 : kPitch == 128 ? row >> 1 & 7 : row >> 2 & 3;
}
template <int kPitch, bool F8>
__device__ __forceinline__ uint32_t v_swizzle(uint32_t row) {
    if (F8) {
        const uint32_t upper = row >> 4 & 1;
        return kPitch == 256 ? (row & 7) | upper << 3 : kPitch == 128 ? (row >> 1 & 3) | upper << 2 : (row >> 2 & 1) | upper << 1;
    }
    return kPitch >= 256 ? (row & 7) << 1 : (row >> 1 & 3) << 1;
}

// Workgroups that a compute unit holds, by their LDS (160 KiB; for 32 keys and values
// of four wavefronts) and registers (the sums of values, the rows).
constexpr int residents(int dim, int row_tiles, bool f8) {
    const int by_lds = 160 / (dim * (f8 ? 1 : 2) / 4 + 2), by_registers = dim * row_tiles >= 512 ? 1 : dim * row_tiles >= 256 ? 2 : dim * row_tiles >= 128 ? 3 : 4;
    return by_lds < by_registers ? by_lds : by_registers;
}

// NR: tiles of 16 rows that a workgroup has.  A wavefront's 32 keys and values come
// by copies to LDS that is its own: the next keys are asked for when these have been
// multiplied, the next values likewise, and no registers wait for them.  The source
// waits for the values alone, but the compiler puts a wait for all copies before their
// first transposing read (whether the next keys were asked for depends on a branch):
// the next keys come during the softmax, not beyond it.
template <int D, int NR, bool F8>
__global__ __launch_bounds__(64 * kWaves, residents(D, NR, F8)) void paged_kernel(Kernel p) {
    constexpr int kRow = F8 ? D : 2 * D, kDims = D / 16, kSteps = D / 32, kRows = 16 * NR, kChunks = D / 8;
    constexpr int kCopies = kRow / 64;  // of 1 KiB for 16 keys
    constexpr int kTile = kWaveKeys * kRow, kOutRows = F8 ? 8 : 16;  // rows joined at a time: as many as fit the values' place
    static_assert(kOutRows * D * 4 == kTile, "shares in the place of values");
    // keys, then values; at the end the rows' sums of values
    __shared__ __attribute__((aligned(1024))) uint8_t s_k[kWaves][kTile], s_v[kWaves][kTile];
    __shared__ float s_m[kWaves][kRows], s_l[kWaves][kRows], s_top[kRows], s_sum[kRows];
    const PagedArgs &a = p.a;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64, r = l % 16, g = l / 16;
    const uint32_t part = blockIdx.x / p.row_blocks, block = blockIdx.x % p.row_blocks;
    const Line line = line_of(a, p.extra);
    const uint32_t total = line.total, begin = part_begin(total, part, p.parts), end = part_begin(total, part + 1, p.parts);
    const uint32_t all_rows = a.rows * p.group;
    const size_t page_size = a.cache.page;
    uint8_t *const kl = s_k[wave], *const vl = s_v[wave];
    // K: chunk of key r (and r + 16) that a lane has of a step of 32 dimensions; V^T: dimension 16 d + l % 16 of the
    // keys that its weights have (4 g and 16 + 4 g on).  Other steps' and dimensions' are these with bits flipped.
    const uint32_t k_at = r * kRow + (g ^ k_swizzle<kRow>(r)) * 16;
    uint32_t v_at, v_at2;
    if constexpr (F8) {
        const uint32_t key = r / 2 < 4 ? 4 * g + r / 2 : 16 + 4 * g + r / 2 - 4;  // of the eight rows
        v_at = key * kRow + v_swizzle<kRow, true>(key) * 16 + r % 2 * 8;
        v_at2 = 0;
    } else {
        const uint32_t key = 4 * g + r / 4;
        v_at = key * kRow + ((r % 4 / 2) ^ v_swizzle<kRow, false>(key)) * 16 + r % 2 * 8;
        v_at2 = v_at + 16 * kRow;  // the swizzle of row + 16 is that of the row
    }

    const bool keeps_cuts = block == 0 && tid == 0;
    const Place place = begin < end ? place_of(a, line, p.extra, begin) : Place{a.n_seqs, 1, 0};
    uint32_t seq = place.seq, steps = place.places - p.extra, kv = __builtin_amdgcn_readfirstlane((begin - place.first) / place.places);
    uint32_t unit = place.first + kv * place.places;  // its first place
    uint32_t from = begin - unit > p.extra ? begin - unit - p.extra : 0;
    if (seq >= a.n_seqs || unit + p.extra >= end) {  // no step
        if (keeps_cuts && !p.by_unit) p.cuts[part].parts = 0;
        return;
    }

    int32_t len = 0;
    bool poison = false;
    const constant_i32 *table = nullptr;
    int first = 0, behind = 0;  // the wavefront's first key, and the end of the workgroup's
    int64_t row0[2] = {0, 0};
    f32x4 ks[2], vs[2];
    bf16x8 q[NR][kSteps];
    int limit[NR];

    // the first of 16 keys in the cache; keys behind the end: -1
    auto find = [&](int key) -> int64_t {
        if (key >= len) return -1;
        int32_t page = table[__builtin_amdgcn_readfirstlane((uint32_t)key >> p.page_shift)];
        if (page < 0 || (uint32_t)page >= a.cache.n_pages) {
            poison = true;
            page = 0;
        }
        return (int64_t)(((size_t)page * a.cache.kv_heads + kv) * page_size + ((uint32_t)key & (uint32_t)(page_size - 1)));
    };
    // copies of 32 keys' rows; those behind the end are zero
    auto copy = [&](const void *from_cache, const int64_t (&row0)[2], int k0, uint8_t *to, bool values) {
        uint32_t lane = l;
        asm volatile("" : "+v"(lane));  // offsets are computed where they are used: they would take registers all along
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int left = len - k0 - 16 * j, rows = left < 0 ? 0 : left < 16 ? left : 16;
            const Desc d = make_desc(static_cast<const uint8_t *>(from_cache) + (row0[j] < 0 ? 0 : (size_t)row0[j]) * kRow, rows * kRow);
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const uint32_t byte = i * 1024 + lane * 16, rr = byte / kRow, c = byte % kRow / 16;
                const uint32_t sw = values ? v_swizzle<kRow, F8>(16 * j + rr) : k_swizzle<kRow>(rr);
                copy16(d, rr * kRow + (c ^ sw) * 16, to + j * 16 * kRow + i * 1024);
            }
        }
    };
    auto scales = [&] {
        if constexpr (F8) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t at_row = row0[j] < 0 ? row0[0] : row0[j];
                ks[j] = *reinterpret_cast<const f32x4 *>(a.cache.k_scales + at_row + 4 * g);
                vs[j] = *reinterpret_cast<const f32x4 *>(a.cache.v_scales + at_row + 4 * g);
            }
        }
    };
    // Asks for the rows and the first keys of steps from..upto of (seq, kv).
    uint32_t upto = 0;
    auto ask = [&] {
        upto = steps < end - unit - p.extra ? steps : end - unit - p.extra;
        len = ((const constant_i32 *)(uintptr_t)a.lens)[seq];
        poison = len < 0 || (uint64_t)len > (uint64_t)a.max_pages * page_size;
        if (poison) len = 0;
        table = (const constant_i32 *)(uintptr_t)(a.pages + (size_t)seq * a.max_pages);
        first = (int)(from * kStepKeys) + wave * kWaveKeys;
        behind = upto * kStepKeys < (uint32_t)len ? (int)(upto * kStepKeys) : len;  // the last step may end at 2^31
        // column r of tile n is row block * kRows + 16 n + r, of query row / group and head row % group
        const uint32_t here_r = here(r), here_g = here(g);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            uint32_t row = block * kRows + n * 16 + here_r;
            if (row >= all_rows) row = all_rows - 1;
            const uint32_t i = query_of(p, row), head = kv * p.group + (row - query_of(p, row) * p.group);
            limit[n] = len - (int)a.rows + (int)i;
            const uint16_t *qp = static_cast<const uint16_t *>(a.q.d) + ((size_t)seq * a.rows + i) * a.q.row + (size_t)head * a.q.head;
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
                q[n][s] = *reinterpret_cast<const bf16x8 *>(qp + (F8 ? s / 2 * 64 + here_g * 16 + s % 2 * 8 : s * 32 + here_g * 8));
        }
        if (first < behind) {
            row0[0] = find(first), row0[1] = find(first + 16);
            copy(a.cache.k, row0, first, kl, false);
            scales();
        }
    };

    ask();
    for (;;) {
        const int limit_min = len - (int)a.rows;
        int odd_at = -1;  // the wavefront's keys from here on are left to the end: only the sequence's last step can be such
        f32x4 o[kDims][NR];
        float m[NR], sum[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            m[n] = -kInf;
            sum[n] = 0.0f;
#pragma unroll
            for (int d = 0; d < kDims; ++d) o[d][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        if (first < behind) {
            copy(a.cache.v, row0, first, vl, true);
            // the rows are waited for here, so that no wait inside the loop is for them
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(q[n][s]));
            for (int k0 = first;;) {
                const bool more = behind - k0 > kStepKeys;
                const int next = more ? k0 + kStepKeys : behind;
                f32x4 s[2][NR];
                int64_t row_next[2] = {0, 0};
                if (more) row_next[0] = find(next), row_next[1] = find(next + 16);
                wait_copies<2 * kCopies>();  // the keys are there, the values' copies may be under way
                {
                    uint32_t at_k = k_at;
                    asm volatile("" : "+v"(at_k));
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
#pragma unroll
                        for (int n = 0; n < NR; ++n) s[j][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int i = 0; i < kSteps; i += F8 ? 2 : 1) {
                            // chunk 4 i + g (of e4m3, two steps' dimensions)
                            const int c = F8 ? i / 2 * 4 : i * 4;
                            const u32x4 x = *reinterpret_cast<const u32x4 *>(kl + (at_k ^ (c % 16 * 16)) + c / 16 * 256 + j * 16 * kRow);
                            if constexpr (F8) {
                                const bf16x8 lo = f8_widen(x[0], x[1]), hi = f8_widen(x[2], x[3]);
#pragma unroll
                                for (int n = 0; n < NR; ++n) {
                                    s[j][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, q[n][i], s[j][n], 0, 0, 0);
                                    s[j][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, q[n][i + 1], s[j][n], 0, 0, 0);
                                }
                            } else {
#pragma unroll
                                for (int n = 0; n < NR; ++n)
                                    s[j][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), q[n][i], s[j][n], 0, 0, 0);
                            }
                        }
                    }
                }
                f32x4 vscale[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if constexpr (F8) {
                        vscale[j] = vs[j];
#pragma unroll
                        for (int n = 0; n < NR; ++n) s[j][n] *= ks[j];
                    }
                }
                reads_done();
                if (more) {
                    row0[0] = row_next[0], row0[1] = row_next[1];
                    copy(a.cache.k, row0, next, kl, false);
                    scales();
                }
                const bool partly = k0 + kWaveKeys - 1 > limit_min;  // some row does not see all keys
                bf16x8 w[NR];
                bool grown = false;
                float top[NR];
#pragma unroll
                for (int n = 0; n < NR; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            s[j][n][i] *= p.scale_log2;
                            if (partly && k0 + 16 * j + 4 * g + i > limit[n]) s[j][n][i] = -kInf;
                        }
                    top[n] = fmaxf(fmaxf(fmaxf(s[0][n][0], s[0][n][1]), fmaxf(s[0][n][2], s[0][n][3])),
                                   fmaxf(fmaxf(s[1][n][0], s[1][n][1]), fmaxf(s[1][n][2], s[1][n][3])));
                    top[n] = other_half_max(other_row_max(top[n]));
                    grown |= top[n] > m[n] + kSlack;
                }
                if (__any(grown)) {
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        const float m_new = fmaxf(m[n], top[n]), keep = m_new == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m[n] - m_new);
                        m[n] = m_new;
                        sum[n] *= keep;
#pragma unroll
                        for (int d = 0; d < kDims; ++d) o[d][n] *= keep;
                    }
                }
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    const float m_use = m[n] == -kInf ? 0.0f : m[n];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float x = __builtin_amdgcn_exp2f(s[e / 4][n][e % 4] - m_use);
                        sum[n] += x;
                        if constexpr (F8) w[n][e] = (__bf16)(partly && k0 + 16 * (e / 4) + 4 * g + e % 4 > limit[n] ? 0.0f : x * vscale[e / 4][e % 4]);
                        else w[n][e] = (__bf16)x;
                    }
                }
                // the values are there; the next keys' copies (and scales) may be under way
                if (more) wait_copies<2 * kCopies + (F8 ? 4 : 0)>();
                else wait_copies<0>();
                if (partly && a.rows > 1) {
                    uint32_t any = 0;
#pragma unroll
                    for (int i = 0; i < kTile / 1024; ++i) {
                        const u32x4 x = *reinterpret_cast<const u32x4 *>(vl + i * 1024 + l * 16);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            // e4m3: all but the sign set; bf16: the exponent's carry
                            if constexpr (F8) any |= ((x[e] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                            else any |= ((x[e] & 0x7FFF7FFFu) + 0x00800080u) & 0x80008000u;
                        }
                    }
                    if (__any(any != 0)) odd_at = k0;
                }
                if (odd_at != k0) {
                    uint32_t at_v = v_at, at_v2 = v_at2;
                    asm volatile("" : "+v"(at_v), "+v"(at_v2));
#pragma unroll
                    for (int d = 0; d < kDims; ++d) {
                        bf16x8 v;
                        if constexpr (F8) {
                            const int c = d;
                            const auto x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2 *)(vl + (at_v ^ (c * 16))));
                            v = f8_widen((uint32_t)x[0], (uint32_t)x[1]);
                        } else {
                            const int c = d * 2;
                            const uint2 x = read_transposed(vl + (at_v ^ (c % 16 * 16)) + c / 16 * 256), y = read_transposed(vl + (at_v2 ^ (c % 16 * 16)) + c / 16 * 256);
                            v = __builtin_bit_cast(bf16x8, u32x4{x.x, x.y, y.x, y.y});
                        }
#pragma unroll
                        for (int n = 0; n < NR; ++n) o[d][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, w[n], o[d][n], 0, 0, 0);
                    }
                }
                reads_done();
                if (!more) break;
                copy(a.cache.v, row0, next, vl, true);
                k0 = next;
            }
        }
        // Infinities or NaN that only some rows see: key by key.
        if (odd_at >= 0) {
#pragma unroll 1
            for (int key = odd_at; key < len && key - odd_at < kWaveKeys; ++key) {
                int32_t page = a.pages[(size_t)seq * a.max_pages + ((uint32_t)key >> p.page_shift)];
                if (page < 0 || (uint32_t)page >= a.cache.n_pages) page = 0;  // noticed before
                const size_t at_row = ((size_t)page * a.cache.kv_heads + kv) * page_size + ((uint32_t)key & (uint32_t)(page_size - 1));
                float dot[NR] = {};
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    const uint32_t e0 = F8 ? s / 2 * 64 + g * 16 + s % 2 * 8 : s * 32 + g * 8;
                    bf16x8 x;
                    if constexpr (F8) {
                        const uint2 b = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.cache.k) + at_row * D + e0);
                        x = f8_widen(b.x, b.y);
                    } else {
                        x = *reinterpret_cast<const bf16x8 *>(static_cast<const uint16_t *>(a.cache.k) + at_row * D + e0);
                    }
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int e = 0; e < 8; ++e) dot[n] = __builtin_fmaf((float)x[e], (float)q[n][s][e], dot[n]);
                }
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    dot[n] += __shfl_xor(dot[n], 16);
                    dot[n] += __shfl_xor(dot[n], 32);
                    if constexpr (F8) dot[n] *= a.cache.k_scales[at_row];
                    float e = __builtin_amdgcn_exp2f(dot[n] * p.scale_log2 - (m[n] == -kInf ? 0.0f : m[n]));
                    if constexpr (F8) e *= a.cache.v_scales[at_row];
                    const bool sees = key <= limit[n];
#pragma unroll
                    for (int d = 0; d < kDims; ++d) {
                        float v[4];
                        if constexpr (F8) {
                            const uint32_t b = *reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(a.cache.v) + at_row * D + d * 16 + 4 * g);
                            const bf16x8 x = f8_widen(b, 0);
                            for (int i = 0; i < 4; ++i) v[i] = (float)x[i];
                        } else {
                            four_bf16(static_cast<const uint16_t *>(a.cache.v) + at_row * D + d * 16 + 4 * g, v);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (sees) o[d][n][i] = __builtin_fmaf(e, v[i], o[d][n][i]);
                    }
                }
            }
        }

        // the next (sequence, key head) of the part is asked for before the wavefronts' shares of this one are joined
        const uint32_t of_seq = seq, of_kv = kv;
        const bool bad = __any(poison), begins = from == 0, whole = begins && upto == steps;
        if (bad && a.status && tid % 64 == 0) *a.status = TQF_HIP_ERR_INVALID;
        if (keeps_cuts && begins && p.by_unit) {
            const uint32_t n = whole ? 0 : part_of(total, unit + p.extra + steps - 1, p.parts) - part + 1;
            p.cuts[seq * a.cache.kv_heads + kv] = Cut{seq, kv, part, n};
        }
        from = 0;
        unit += steps + p.extra;
        const bool again = unit + p.extra < end && (kv + 1 < a.cache.kv_heads || seq + 1 < a.n_seqs);
        if (keeps_cuts && !again && !p.by_unit) {
            const uint32_t n = whole || !begins ? 0 : part_of(total, unit - 1, p.parts) - part + 1;
            p.cuts[part] = Cut{seq, kv, part, n};
        }
        if (again) {
            if (++kv == a.cache.kv_heads) {
                kv = 0;
                ++seq;
                steps = steps_of(a, ((const constant_i32 *)(uintptr_t)a.lens)[seq]);
            }
            ask();
        }
        const int here_l = here(l), here_r = here_l % 16, here_g = here_l / 16;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            sum[n] += __shfl_xor(sum[n], 16);
            sum[n] += __shfl_xor(sum[n], 32);
            if (bad) sum[n] = __builtin_nanf("");
            if (here_g == 0) {
                s_m[wave][n * 16 + here_r] = m[n];
                s_l[wave][n * 16 + here_r] = sum[n];
            }
        }
        __syncthreads();
        float *to = p.partial + ((size_t)(2 * part + (begins ? 1 : 0)) * p.row_blocks + block) * kRows * (D + 2);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int row = n * 16 + here_r;
            float top = s_m[0][row], all = 0.0f;
#pragma unroll
            for (int u = 1; u < kWaves; ++u) top = fmaxf(top, s_m[u][row]);
            const float mine = m[n] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m[n] - top);
#pragma unroll
            for (int u = 0; u < kWaves; ++u)  // a wavefront without keys has sum 0, or NaN where its sequence or a page is bad
                all += s_m[u][row] == -kInf ? s_l[u][row] : s_l[u][row] * __builtin_amdgcn_exp2f(s_m[u][row] - top);
            if (wave == 0 && here_g == 0) s_top[row] = top, s_sum[row] = all;
#pragma unroll
            for (int half = 0; half < 16 / kOutRows; ++half) {
                // gates are asked for before the shares meet: one by one each would be a trip to memory
                constexpr int kOuts = (kOutRows * kChunks * 2 + 64 * kWaves - 1) / (64 * kWaves);
                uint2 gates[kOuts] = {};
                if (whole && a.gate.d) {
#pragma unroll
                    for (int x = 0; x < kOuts; ++x) {
                        const int i = x * 64 * kWaves + wave * 64 + here_l;
                        uint32_t row_of = block * kRows + n * 16 + half * kOutRows + i / (2 * kChunks);
                        if (row_of >= all_rows) row_of = all_rows - 1;
                        gates[x] = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.gate.d) + ((size_t)of_seq * a.rows + query_of(p, row_of)) * a.gate.row +
                                                                    ((size_t)of_kv * p.group + (row_of - query_of(p, row_of) * p.group)) * a.gate.head + i % (2 * kChunks) * 4);
                    }
                }
                // [row][chunk of 4 at chunk ^ row] f32
                if (here_r / kOutRows == half) {
#pragma unroll
                    for (int d = 0; d < kDims; ++d) {
                        const int c = d * 4 + here_g, rr = here_r % kOutRows;
                        *reinterpret_cast<f32x4 *>(s_v[wave] + rr * D * 4 + (c ^ rr) * 16) = o[d][n] * mine;
                    }
                }
                __syncthreads();
#pragma unroll
                for (int x = 0; x < kOutRows * kChunks * 2; x += 64 * kWaves) {
                    const int i = x + wave * 64 + here_l, rr = i / (2 * kChunks), c = i % (2 * kChunks), of_block = n * 16 + half * kOutRows + rr;
                    if (kOutRows * kChunks * 2 < 64 * kWaves && rr >= kOutRows) break;
                    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
                    const float total_l = s_sum[of_block];
#pragma unroll
                    for (int u = 0; u < kWaves; ++u) v += *reinterpret_cast<const f32x4 *>(s_v[u] + rr * D * 4 + (c ^ rr) * 16);
                    const uint32_t out_row = block * kRows + of_block;
                    if (!whole) {
                        float *row_to = to + (size_t)of_block * (D + 2);
                        __builtin_memcpy(row_to + c * 4, &v, 16);
                        if (c == 0) {
                            row_to[D] = s_top[of_block];
                            row_to[D + 1] = total_l;
                        }
                    } else if (out_row < all_rows) {
                        const float inv = total_l == 0.0f ? 0.0f : 1.0f / total_l;
                        const size_t token = (size_t)of_seq * a.rows + query_of(p, out_row), head = (size_t)of_kv * p.group + (out_row - query_of(p, out_row) * p.group);
                        v *= inv;
                        if (a.gate.d && total_l != 0.0f) {  // without a key: 0, also where the gate is NaN
                            const uint2 g2 = gates[x / (64 * kWaves)];
                            v[0] *= sigmoid(__uint_as_float(g2.x << 16)), v[1] *= sigmoid(__uint_as_float(g2.x & 0xFFFF0000u));
                            v[2] *= sigmoid(__uint_as_float(g2.y << 16)), v[3] *= sigmoid(__uint_as_float(g2.y & 0xFFFF0000u));
                        }
                        store4(a.y + (token * a.q_heads + head) * D + c * 4, 4, v);
                    }
                }
                __syncthreads();
            }
        }
        if (!again) break;
    }
}

// Joins what several parts have of one (sequence, key head): a workgroup for each
// cut and `each` rows.  With one row its wavefronts have some of the parts each, with
// several, if the parts are few, a row each.  Sixteen wavefronts for the one (cut into
// 128 parts: 7.4 us, with eight 9.1), eight for the other.  Cuts are kept by unit
// where those are fewer than the parts, so that only as many workgroups look for
// one: one sequence of 131072 tokens 60 us, a cut for each part 111.
constexpr int kJoinWaves = 16, kJoinAhead = 4;
template <int D>
__global__ __launch_bounds__(64 * kJoinWaves) void join_kernel(Kernel p, uint32_t block_rows, uint32_t each) {
    constexpr int kPer = D / 64;
    __shared__ float s_o[kJoinWaves][D], s_m[kJoinWaves], s_l[kJoinWaves];
    const PagedArgs &a = p.a;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), l = tid % 64, waves = blockDim.x / 64;
    const uint32_t all_rows = a.rows * p.group, sets = (all_rows + each - 1) / each;
    const Cut cut = p.cuts[blockIdx.x / sets];
    const uint32_t parts = cut.parts, row0 = blockIdx.x % sets * each;
    if (parts == 0) return;
    const size_t stride = (size_t)2 * p.row_blocks * block_rows * (D + 2);  // of a part
    float m, sum, o[kPer];
    // parts `begin`, begin + step, ... of a row
    auto gather = [&](uint32_t row, uint32_t begin, uint32_t step) {
        m = -kInf, sum = 0.0f;
#pragma unroll
        for (int d = 0; d < kPer; ++d) o[d] = 0.0f;
        for (uint32_t i = begin; i < parts; i += kJoinAhead * step) {
            float pm[kJoinAhead], pl[kJoinAhead], po[kJoinAhead][kPer];
#pragma unroll
            for (int x = 0; x < kJoinAhead; ++x) {
                const uint32_t at = i + x * step < parts ? i + x * step : parts - 1;
                const size_t slot = at == 0 ? 1 : 0;  // a part keeps what begins in it apart from what goes on
                const float *from = p.partial + (cut.first + at) * stride + ((slot * p.row_blocks + row / block_rows) * block_rows + row % block_rows) * (D + 2);
                pm[x] = from[D], pl[x] = from[D + 1];
                if constexpr (kPer == 1) po[x][0] = from[l];
                else __builtin_memcpy(po[x], from + l * kPer, 4 * kPer);
            }
#pragma unroll
            for (int x = 0; x < kJoinAhead; ++x) {
                if (i + x * step >= parts) break;
                const float top = fmaxf(m, pm[x]), keep = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - top);
                const float take = pm[x] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(pm[x] - top);
                m = top;
                // a part without keys has sum 0, or NaN where its sequence or a page is bad: NaN stays
                sum = sum * (m == -kInf ? 1.0f : keep) + (pm[x] == -kInf ? pl[x] : pl[x] * take);
#pragma unroll
                for (int d = 0; d < kPer; ++d) o[d] = o[d] * keep + po[x][d] * take;
            }
        }
    };
    // a row's gates, asked for before its parts: behind them they would be a trip to memory more
    uint16_t gate[kPer];
    auto ask_gate = [&](uint32_t row) {
        if (!a.gate.d) return;
        const size_t token = (size_t)cut.seq * a.rows + query_of(p, row), head = (size_t)cut.kv * p.group + (row - query_of(p, row) * p.group);
        const void *from = static_cast<const uint16_t *>(a.gate.d) + token * a.gate.row + head * a.gate.head + l * kPer;
        __builtin_memcpy(gate, __builtin_assume_aligned(from, 2 * kPer), 2 * kPer);
    };
    auto store = [&](uint32_t row) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const size_t token = (size_t)cut.seq * a.rows + query_of(p, row), head = (size_t)cut.kv * p.group + (row - query_of(p, row) * p.group);
        uint16_t y[kPer];
#pragma unroll
        for (int d = 0; d < kPer; ++d) y[d] = __builtin_bit_cast(uint16_t, (__bf16)(o[d] * inv * (a.gate.d && sum != 0.0f ? gate_of(gate[d]) : 1.0f)));
        __builtin_memcpy(__builtin_assume_aligned(a.y + (token * a.q_heads + head) * D + l * kPer, 2 * kPer), y, 2 * kPer);
    };
    if (each > 1 && parts <= kJoinWaves) {
        for (uint32_t row = row0 + wave; row < row0 + each && row < all_rows; row += waves) {
            ask_gate(row);
            gather(row, 0, 1);
            store(row);
        }
        return;
    }
    for (uint32_t row = row0; row < row0 + each && row < all_rows; ++row) {
        if (wave == 0) ask_gate(row);
        gather(row, wave, waves);
#pragma unroll
        for (int d = 0; d < kPer; ++d) s_o[wave][l * kPer + d] = o[d];
        if (l == 0) {
            s_m[wave] = m;
            s_l[wave] = sum;
        }
        __syncthreads();
        if (wave == 0) {
            float top = -kInf;
            for (int i = 0; i < waves; ++i) top = fmaxf(top, s_m[i]);
            sum = 0.0f;
#pragma unroll
            for (int d = 0; d < kPer; ++d) o[d] = 0.0f;
#pragma unroll 4
            for (int i = 0; i < waves; ++i) {
                const float f = s_m[i] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(s_m[i] - top);
                sum += s_m[i] == -kInf ? s_l[i] : s_l[i] * f;
#pragma unroll
                for (int d = 0; d < kPer; ++d) o[d] += s_o[i][l * kPer + d] * f;
            }
            store(row);
        }
        __syncthreads();
    }
}

uint32_t tiles_of_rows(const PagedArgs &a) { return a.rows * (a.q_heads / a.cache.kv_heads) > 16 ? 2 : 1; }
uint32_t row_blocks(const PagedArgs &a) {
    const uint32_t rows = a.rows * (a.q_heads / a.cache.kv_heads), per = 16 * tiles_of_rows(a);
    return (rows + per - 1) / per;
}
uint64_t units_of(const PagedArgs &a) { return (uint64_t)a.n_seqs * a.cache.kv_heads; }
uint64_t most_steps(const PagedArgs &a) { return units_of(a) * (((uint64_t)a.max_pages * a.cache.page + kStepKeys - 1) / kStepKeys); }
// As many workgroups as the compute units hold at once, for each block of rows (several of them, of more than 32
// columns, take turns); no more than there can be steps.
uint32_t parts_of(const PagedArgs &a) {
    const uint64_t want = (uint64_t)residents(a.cache.dim, tiles_of_rows(a), a.cache.f8) * (uint64_t)cu_count();
    return (uint32_t)(most_steps(a) < want ? most_steps(a) : want);
}

uint32_t cuts_of(const PagedArgs &a) { return (uint32_t)(units_of(a) < parts_of(a) ? units_of(a) : parts_of(a)); }
size_t cuts_bytes(const PagedArgs &a) { return ((size_t)cuts_of(a) * sizeof(Cut) + 255) / 256 * 256; }

template <int D, int NR>
hipError_t launch_for(hipStream_t s, const Kernel &p) {
    const dim3 grid(p.parts * p.row_blocks), block(64 * kWaves);
    if (p.a.cache.f8) paged_kernel<D, NR, true><<<grid, block, 0, s>>>(p);
    else paged_kernel<D, NR, false><<<grid, block, 0, s>>>(p);
    if (p.parts > 1) {
        if (const hipError_t e = hipGetLastError()) return e;
        // A workgroup a row while there are few, else eight rows: more workgroups would wait for one another's places.
        // 64 sequences of 4 rows of 16 heads: 58 us with eight, 84 with one; one sequence of 131072 tokens: 110 and 60.
        const uint32_t rows = p.a.rows * p.group, cuts = cuts_of(p.a), each = cuts * rows <= 1024 ? 1 : 8;
        join_kernel<D><<<dim3(cuts * ((rows + each - 1) / each)), dim3(each == 1 ? 1024 : 512), 0, s>>>(p, 16 * NR, each);
    }
    return hipGetLastError();
}

}  // namespace

size_t attn_paged_scratch_bytes(const PagedArgs &a) {
    return cuts_bytes(a) + (size_t)2 * parts_of(a) * row_blocks(a) * 16 * tiles_of_rows(a) * (a.cache.dim + 2) * 4;
}

hipError_t launch_attn_paged(hipStream_t s, const PagedArgs &a, void *scratch) {
    Kernel p{};
    p.a = a;
    p.group = a.q_heads / a.cache.kv_heads;
    p.of_group = (1u << 20) / p.group + 1;
    p.row_blocks = row_blocks(a);
    p.parts = parts_of(a);
    p.page_shift = (uint32_t)__builtin_ctz(a.cache.page);
    p.scale_log2 = a.scale * kLog2e;
    // with a workgroup for every step there is nothing to balance; two tiles of rows of 256 take longest to leave
    p.extra = most_steps(a) <= p.parts ? 0 : a.cache.dim * tiles_of_rows(a) >= 512 ? kMostExtra : 1;
    p.by_unit = units_of(a) <= p.parts;
    p.cuts = static_cast<Cut *>(scratch);
    p.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + cuts_bytes(a));
    const bool two = tiles_of_rows(a) == 2;
    if (a.cache.dim == 64) return two ? launch_for<64, 2>(s, p) : launch_for<64, 1>(s, p);
    if (a.cache.dim == 128) return two ? launch_for<128, 2>(s, p) : launch_for<128, 1>(s, p);
    return two ? launch_for<256, 2>(s, p) : launch_for<256, 1>(s, p);
}

}  // namespace tqf
