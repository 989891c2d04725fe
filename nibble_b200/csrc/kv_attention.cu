// Attention of a sequence's newest tokens over its 8-bit cache (format: kv_cache.cuh).
//
// Query i of `count` stands at position length - count + i and sees the positions up to its own:
//     out = sum_t p_t v_t / sum_t p_t,   p_t = exp(softmax_scale * q . k_t - max)
// The queries of all heads that share a key/value head are rows of one problem (row = i * group + head in group), 16 of them a
// tile of mma.sync m16n8k16.  Codes enter the products as exact FP16 integers, made of bytes by OR-ing them into 1024.0 (one LOP3 for
// two, then 1152 is subtracted); the key's scale multiplies the FP32 score, the value's goes into the probability before that is
// rounded to FP16, both relative to the block at which the accumulator was last rescaled.  FP16 has its eleven bits for
// probabilities down to 2^-24 of the largest (they are held times 2^10), so a weight is off by 2^-12 of itself at most on average
// over thousands of tokens; scores, maxima, sums and outputs are FP32.
//
// Bound: HBM, one byte a number of the cache.  A warp streams blocks of its own through a ring in shared memory (bulk copies: 4 KB of
// keys and 4 KB of values at D = 128), keeps its own running maximum, sum and output, and meets the others at the end of a run
// only.  All blocks of all sequences and heads are cut into equal runs, one for each CTA, whatever the sequences' lengths; what a
// run has of a sequence and head that other runs share goes to the workspace, and a second kernel adds those parts up in order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "kv_cache.cuh"
#include "per_device.h"
#include "tcgen05.cuh"
#include "unpack.cuh"

namespace w4a16 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMinRun = 2 * kWarps;             // blocks that are worth a CTA
constexpr float kNone = -1.0e30f;               // the maximum of nothing
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHeadroom = 1024.0f;            // probabilities are held in FP16 times this: 2^10,
constexpr float kMaxLag = 3.0f;                 // times 2^3 where the maximum has not been followed yet,
constexpr float kMaxRatio = 4.0f;               // times 4 where the values' scale has not: below 65504 in all

struct AttentionParams {
    KvCache cache;
    const char* q;
    long long q_batch, q_token, q_head;          // strides in numbers
    bool q_wide;                                 // rows can be read 16 bytes at a time
    char* out;                                   // [batch][tokens][q heads][D]
    int tokens, q_heads, group;
    int row_tiles;                               // of 16 * MT rows: as many as `tokens` queries make
    const long long* lengths;
    const long long* counts;                     // null: all `tokens` of every sequence
    float scale;                                 // softmax scale * log2 e
    float* parts;                                // workspace: see part_of()
    int grid;                                    // CTAs of the first kernel
    bool split;                                  // whether runs may cut a sequence and head
};

struct Sequence {
    int length, count, blocks, row_tiles;        // row_tiles: of this sequence's queries, 0 when there is nothing to do
};

__device__ __forceinline__ Sequence sequence_of(const AttentionParams& p, int b, int tile_rows) {
    Sequence s{0, 0, 0, 0};
    const long long length = p.lengths[b], count = p.counts == nullptr ? p.tokens : p.counts[b];
    if (length < 0 || length > p.cache.max_len || count < 0 || count > p.tokens) return s;
    s.length = static_cast<int>(length);
    s.count = static_cast<int>(count);
    s.blocks = (s.length + kKvBlock - 1) / kKvBlock;
    s.row_tiles = s.blocks > 0 ? (s.count * p.group + tile_rows - 1) / tile_rows : 0;
    return s;
}

__device__ __forceinline__ long long work_of(const AttentionParams& p, const Sequence& s) {
    return static_cast<long long>(s.blocks) * s.row_tiles * p.cache.kv_heads;
}

// The part of (sequence, head, tile) that a CTA's run holds: its first segment or its last.
__device__ __forceinline__ float* part_of(const AttentionParams& p, int cta, bool first, int tile_rows, int d) {
    return p.parts + (static_cast<size_t>(cta) * 2 + (first ? 0 : 1)) * tile_rows * (d + 2);
}

// All blocks of all sequences, and CTAs that share them.
__device__ __forceinline__ int active_ctas(const AttentionParams& p, long long total) {
    return static_cast<int>(max(1ll, min(static_cast<long long>(p.grid), total / kMinRun)));
}
__device__ __forceinline__ long long run_begin(long long total, int active, int cta) { return total * cta / active; }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four codes of a word as (c0, c2) and (c1, c3).
__device__ __forceinline__ void codes_to_half(uint32_t word, uint32_t& even, uint32_t& odd) {
    even = hsub2_u32(and_xor(word, 0x00ff00ffu, 0x64806480u), 0x64806480u);
    odd = hsub2_u32(and_xor(word >> 8, 0x00ff00ffu, 0x64806480u), 0x64806480u);
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}

// A power of two that brings `top` to between 2^9 and 2^10 (1 for zero), and its inverse.
__device__ __forceinline__ float power_for(float top, float& inverse) {
    const int exponent = top > 0.0f ? max(-100, min(100, 9 - ilogbf(top))) : 0;
    inverse = __int_as_float((127 - exponent) << 23);
    return __int_as_float((127 + exponent) << 23);
}

__device__ __forceinline__ float finite_magnitude(float x) {
    const float m = fabsf(x);
    return m <= 3.4028235e38f ? m : 0.0f;
}

// A team of MT warps shares a ring; each has a 16-row tile of its own, and the kWarps / MT teams take the blocks in turn.
template <typename T, int D, int MT>
struct AttentionShape {
    static constexpr int kTeams = kWarps / MT;
    static constexpr int kTileRows = 16 * MT;
    static constexpr int kBlockBytes = kKvBlock * D;                   // of keys, and of values
    static constexpr int kStages = 2 * MT * (128 / D);                 // blocks of a ring: 64 KB for a CTA, two of which fit an SM
    static constexpr size_t kRingBytes = static_cast<size_t>(kTeams) * kStages * 2 * kBlockBytes;
    static constexpr size_t kMergeBytes = static_cast<size_t>(kTeams) * kTileRows * (D + 2) * sizeof(float);
    static constexpr size_t kSharedBytes = kRingBytes + (kTeams > 1 ? kMergeBytes : 0);
};

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kThreads, 2)
kv_attention_kernel(const AttentionParams p) {
    using Shape = AttentionShape<T, D, MT>;
    constexpr int kTeams = Shape::kTeams, kStages = Shape::kStages, kTileRows = Shape::kTileRows, kSteps = D / 16, kTiles = D / 8;
    extern __shared__ __align__(128) uint8_t shared[];
    __shared__ __align__(8) unsigned long long bars[kTeams][kStages][2];      // full, empty
    __shared__ long long plan[2];                                              // all blocks; blocks before this CTA's sequence
    __shared__ int plan_b;
    pdl_release_downstream();
    pdl_wait_for_upstream();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int team = warp / MT, member = warp % MT;
    const int g = lane >> 2, c = lane & 3;
    uint8_t* const ring = shared + static_cast<size_t>(team) * kStages * 2 * Shape::kBlockBytes;
    float* const merge = reinterpret_cast<float*>(shared + Shape::kRingBytes);
    if (lane == 0 && member == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&bars[team][s][0]), 1);
            mbar_init(smem_u32(&bars[team][s][1]), MT);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // rows of queries that are not there
    for (long long at = blockIdx.x; at < static_cast<long long>(p.cache.batch) * p.tokens; at += gridDim.x) {
        const int b = static_cast<int>(at / p.tokens), i = static_cast<int>(at % p.tokens);
        const Sequence s = sequence_of(p, b, kTileRows);
        if (i < s.count && s.blocks > 0) continue;
        const long long length = p.lengths[b], count = p.counts == nullptr ? p.tokens : p.counts[b];
        if (tid == 0 && (length < 0 || length > p.cache.max_len || count < 0 || count > p.tokens)) {
            atomicOr(p.cache.status, kKvBadLength);
        }
        uint4* to = reinterpret_cast<uint4*>(p.out + at * p.q_heads * D * 2);
        for (int e = tid; e < p.q_heads * D / 8; e += kThreads) to[e] = make_uint4(0u, 0u, 0u, 0u);
    }
    // this CTA's run: where it begins
    if (warp == 0) {
        long long total = 0;
        for (int b = lane; b < p.cache.batch; b += 32) total += work_of(p, sequence_of(p, b, kTileRows));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        long long mine = -1;
        if (total > 0) {
            if (p.split) {
                const int active = active_ctas(p, total);
                if (static_cast<int>(blockIdx.x) < active) mine = run_begin(total, active, blockIdx.x);
            }
        }
        if (p.split && mine >= 0) {
            long long before = 0;
            for (int base = 0; base < p.cache.batch; base += 32) {
                const long long work = base + lane < p.cache.batch ? work_of(p, sequence_of(p, base + lane, kTileRows)) : 0;
                long long upto = work;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long other = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += other;
                }
                const unsigned past = __ballot_sync(0xffffffffu, before + upto > mine);
                if (past != 0) {
                    const int at = __ffs(past) - 1;
                    if (lane == at) {
                        plan[1] = before + upto - work;
                        plan_b = base + at;
                    }
                    break;
                }
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        if (lane == 0) plan[0] = p.split && mine < 0 ? 0 : total;
    }
    __syncthreads();
    const long long total = plan[0];
    if (total == 0) return;
    int b;
    long long base, position, end;             // blocks before sequence b; this run's next block and end
    if (p.split) {
        const int active = active_ctas(p, total);
        b = plan_b;
        base = plan[1];
        position = run_begin(total, active, blockIdx.x);
        end = run_begin(total, active, blockIdx.x + 1);
    } else {                                     // a whole sequence, head and tile for each CTA
        const int per_sequence = p.cache.kv_heads * p.row_tiles;
        b = blockIdx.x / per_sequence;
        const Sequence s = sequence_of(p, b, kTileRows);
        const int unit = blockIdx.x % per_sequence;
        if (unit >= p.cache.kv_heads * s.row_tiles) return;
        base = 0;
        position = static_cast<long long>(unit) * s.blocks;
        end = position + s.blocks;
    }
    unsigned fill = 0, take = 0;                 // blocks that this team's ring was asked for, and that it has used
    bool healthy = true;
    bool first_segment = true;
    while (position < end) {
        Sequence s = sequence_of(p, b, kTileRows);
        while (b + 1 < p.cache.batch && position >= base + work_of(p, s)) {
            base += work_of(p, s);
            ++b;
            s = sequence_of(p, b, kTileRows);
        }
        const long long local = position - base;
        const int unit = static_cast<int>(local / s.blocks), begin = static_cast<int>(local % s.blocks);
        const int stop = static_cast<int>(min(static_cast<long long>(s.blocks), begin + (end - position)));
        const int head = unit / s.row_tiles, tile = unit % s.row_tiles;
        const int full = min(stop, s.length / kKvBlock);                     // blocks [begin, full) are codes, [full, stop) the tail
        const size_t pair = static_cast<size_t>(b) * p.cache.kv_heads + head;
        const uint8_t* k_codes = p.cache.k_codes + pair * p.cache.blocks * Shape::kBlockBytes;
        const uint8_t* v_codes = p.cache.v_codes + pair * p.cache.blocks * Shape::kBlockBytes;
        const float* k_scales = p.cache.k_scales + pair * p.cache.blocks;
        const float* v_scales = p.cache.v_scales + pair * p.cache.blocks;

        auto request = [&](int block) {           // by one thread of the team
            const unsigned slot = fill % kStages;
            const unsigned full_bar = smem_u32(&bars[team][slot][0]);
            if (fill >= kStages && !mbar_wait(smem_u32(&bars[team][slot][1]), (fill / kStages - 1) & 1, kKvGaveUp, p.cache.status)) {
                healthy = false;
            }
            if (healthy) {
                const unsigned to = smem_u32(ring + slot * 2 * Shape::kBlockBytes);
                mbar_arrive_expect_tx(full_bar, 2 * Shape::kBlockBytes);
                bulk_load(to, k_codes + static_cast<size_t>(block) * Shape::kBlockBytes, Shape::kBlockBytes, full_bar);
                bulk_load(to + Shape::kBlockBytes, v_codes + static_cast<size_t>(block) * Shape::kBlockBytes, Shape::kBlockBytes, full_bar);
            }
        };
        const int first_block = begin + team;
        int asked = first_block;                  // next block to request
        for (int i = 0; i < kStages && asked < full; ++i, asked += kTeams) {
            if (lane == 0 && member == 0) request(asked);
            ++fill;
        }

        // queries as the first operand: rows g and g + 8 of this warp's tile, dims in the order of the codes' bytes
        const int row_lo = tile * kTileRows + member * 16 + g, row_hi = row_lo + 8;
        const int rows = s.count * p.group;
        uint32_t q[kSteps][4];
        float q_scale[2] = {p.scale, p.scale};
        int place[2];                              // position of the row's query; -1: no such row
        {
            uint32_t raw[2][D / 8];                // [row][64-dim run * 8 + word]: sixteen dims of each run
            float top[2] = {0.0f, 0.0f};
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = r == 0 ? row_lo : row_hi;
                place[r] = row < rows ? s.length - s.count + row / p.group : -1;
                const T* from = reinterpret_cast<const T*>(p.q) + b * p.q_batch + (row / p.group) * p.q_token +
                                (head * p.group + row % p.group) * p.q_head;
#pragma unroll
                for (int j = 0; j < D / 64; ++j) {
#pragma unroll
                    for (int w = 0; w < 8; w += 4) {
                        uint4 four = make_uint4(0u, 0u, 0u, 0u);
                        if (row < rows && p.q_wide) {
                            four = *reinterpret_cast<const uint4*>(from + j * 64 + c * 16 + w * 2);
                        } else if (row < rows) {
                            const uint16_t* h = reinterpret_cast<const uint16_t*>(from + j * 64 + c * 16 + w * 2);
                            four = make_uint4(h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16,
                                              h[4] | static_cast<uint32_t>(h[5]) << 16, h[6] | static_cast<uint32_t>(h[7]) << 16);
                        }
                        raw[r][j * 8 + w] = four.x;
                        raw[r][j * 8 + w + 1] = four.y;
                        raw[r][j * 8 + w + 2] = four.z;
                        raw[r][j * 8 + w + 3] = four.w;
                    }
#pragma unroll
                    for (int w = 0; w < 8; ++w) {
                        const float2 f = widen2<T>(raw[r][j * 8 + w]);
                        top[r] = fmaxf(top[r], fmaxf(finite_magnitude(f.x), finite_magnitude(f.y)));
                    }
                }
                // BF16 queries become FP16 by a power of two of their row's own: every number that is not 2^-24 below the
                // row's largest keeps all its bits.  FP16 ones are taken as they are.
                float by = 1.0f;
                if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                    float back;
                    by = power_for(top[r], back);
                    q_scale[r] *= back;
                }
#pragma unroll
                for (int j = 0; j < D / 64; ++j) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const float2 lo = widen2<T>(raw[r][j * 8 + 2 * w]), hi = widen2<T>(raw[r][j * 8 + 2 * w + 1]);
                        q[j * 4 + w][r] = pack_half(lo.x * by, hi.x * by);
                        q[j * 4 + w][2 + r] = pack_half(lo.y * by, hi.y * by);
                    }
                }
            }
        }
        float acc[kTiles][4];
#pragma unroll
        for (int j = 0; j < kTiles; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
        float top[2] = {kNone, kNone}, sum[2] = {0.0f, 0.0f};      // the sum of this lane's columns
        float unit_scale = 1.0e-30f;                              // of the accumulator: values are acc * unit_scale / kHeadroom

        // Scores of a block in place of which come the probabilities, as operands of the second product; tokens of lane c:
        // 16 * group + 4 c + 2 e + parity.
        auto probabilities = [&](float (&score)[4][4], int block, float k_scale, float v_scale, uint32_t (&prob)[2][4]) {
            const float by[2] = {k_scale * q_scale[0], k_scale * q_scale[1]};
            const int token = block * kKvBlock;
            float next[2] = {kNone, kNone};
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const bool all = token + kKvBlock - 1 <= place[r];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = score[t][2 * r + e];
                        x = all || token + (t >> 1) * 16 + 4 * c + 2 * e + (t & 1) <= place[r] ? x * by[r] : -INFINITY;
                        next[r] = fmaxf(next[r], x);
                    }
                }
                next[r] = fmaxf(next[r], __shfl_xor_sync(0xffffffffu, next[r], 1));
                next[r] = fmaxf(next[r], __shfl_xor_sync(0xffffffffu, next[r], 2));
            }
            const bool new_unit = v_scale > kMaxRatio * unit_scale;
            const bool lag = next[0] > top[0] + kMaxLag || next[1] > top[1] + kMaxLag;
            if (new_unit || __any_sync(0xffffffffu, lag)) {
                float shrink[2];
                const float unit_change = new_unit ? unit_scale / v_scale : 1.0f;
                if (new_unit) unit_scale = v_scale;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float now = fmaxf(top[r], next[r]);
                    shrink[r] = exp2_fast(top[r] - now);
                    top[r] = now;
                    sum[r] *= shrink[r];
                    shrink[r] *= unit_change;
                }
#pragma unroll
                for (int j = 0; j < kTiles; ++j) {
                    acc[j][0] *= shrink[0];
                    acc[j][1] *= shrink[0];
                    acc[j][2] *= shrink[1];
                    acc[j][3] *= shrink[1];
                }
            }
            const float weight = v_scale / unit_scale * kHeadroom;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float x = score[t][2 * r + e];
                        const float pr = exp2_fast(x - top[r]);
                        sum[r] += pr;
                        w[e] = x == -INFINITY ? 0.0f : pr * weight;      // (a masked token's scale may be NaN)
                    }
                    prob[t >> 1][(t & 1) * 2 + r] = pack_half(w[0], w[1]);
                }
            }
        };

        float k_scale_set = 0.0f, v_scale_set = 0.0f;              // lane l: of this team's block number l since the last set
        int count = 0;
        for (int block = first_block; block < full; block += kTeams, ++count) {
            if ((count & 31) == 0) {
                const int mine = block + lane * kTeams;
                k_scale_set = mine < full ? k_scales[mine] : 0.0f;
                v_scale_set = mine < full ? v_scales[mine] : 0.0f;
            }
            const float k_scale = __shfl_sync(0xffffffffu, k_scale_set, count & 31);
            const float v_scale = __shfl_sync(0xffffffffu, v_scale_set, count & 31);
            const unsigned slot = take % kStages;
            healthy = mbar_wait(smem_u32(&bars[team][slot][0]), (take / kStages) & 1, kKvGaveUp, p.cache.status) && healthy;
            healthy = __all_sync(0xffffffffu, healthy);
            if (!healthy) break;
            const uint8_t* keys = ring + slot * 2 * Shape::kBlockBytes;
            const uint8_t* values = keys + Shape::kBlockBytes;
            float score[4][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) score[t][0] = score[t][1] = score[t][2] = score[t][3] = 0.0f;
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                uint32_t words[4][4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint4 codes = *reinterpret_cast<const uint4*>(keys + (t * (D / 64) + j) * 512 + lane * 16);
                    words[t][0] = codes.x; words[t][1] = codes.y; words[t][2] = codes.z; words[t][3] = codes.w;
                }
#pragma unroll
                for (int w = 0; w < 4; ++w) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        uint32_t even, odd;
                        codes_to_half(words[t][w], even, odd);
                        mma16816(score[t], q[j * 4 + w], even, odd);
                    }
                }
            }
            uint32_t prob[2][4];
            probabilities(score, block, k_scale, v_scale, prob);
#pragma unroll
            for (int j = 0; j < kTiles / 2; ++j) {
                const uint4 codes = *reinterpret_cast<const uint4*>(values + j * 512 + lane * 16);
                const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {                       // words: [half of the sixteen dims][token group]
                    uint32_t even, odd;
                    codes_to_half(words[w], even, odd);
                    mma16816(acc[2 * j + w / 2], prob[w % 2], even, odd);
                }
            }
            // (the slot was read through the generic proxy and is refilled through the async one: each lane orders its own reads)
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars[team][slot][1]));
            ++take;
            if (asked < full) {
                if (lane == 0 && member == 0) request(asked);
                ++fill;
                asked += kTeams;
            }
        }

        // the block that is being filled, by the team whose turn it is
        if (stop > full && healthy && (full - begin) % kTeams == team) {
            const int token = full * kKvBlock;
            const T* k_tail = reinterpret_cast<const T*>(p.cache.k_tail) + (pair * 2 + (full & 1)) * kKvBlock * D;
            const T* v_tail = reinterpret_cast<const T*>(p.cache.v_tail) + (pair * 2 + (full & 1)) * kKvBlock * D;
            const int held = s.length - token;
            // both in FP16 by one power of two each, which takes the scales' place
            float k_top = 0.0f, v_top = 0.0f;
            bool odd_values = false;                               // an infinity or NaN among the values
            for (int i = lane * 2; i < held * D; i += 64) {
                const float2 kf = widen2<T>(*reinterpret_cast<const uint32_t*>(k_tail + i));
                const float2 vf = widen2<T>(*reinterpret_cast<const uint32_t*>(v_tail + i));
                k_top = fmaxf(k_top, fmaxf(finite_magnitude(kf.x), finite_magnitude(kf.y)));
                v_top = fmaxf(v_top, fmaxf(finite_magnitude(vf.x), finite_magnitude(vf.y)));
                odd_values = odd_values || !(fabsf(vf.x) <= 3.4028235e38f) || !(fabsf(vf.y) <= 3.4028235e38f);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                k_top = fmaxf(k_top, __shfl_xor_sync(0xffffffffu, k_top, o));
                v_top = fmaxf(v_top, __shfl_xor_sync(0xffffffffu, v_top, o));
            }
            odd_values = __any_sync(0xffffffffu, odd_values);
            float k_back, v_back;
            const float k_by = power_for(k_top, k_back), v_by = power_for(v_top, v_back);
            float score[4][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                score[t][0] = score[t][1] = score[t][2] = score[t][3] = 0.0f;
                const int at = (t >> 1) * 16 + 2 * g + (t & 1);
#pragma unroll
                for (int j = 0; j < D / 64; ++j) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        float2 lo = make_float2(0.0f, 0.0f), hi = lo;
                        if (at < held) {
                            const uint2 two = *reinterpret_cast<const uint2*>(k_tail + at * D + j * 64 + c * 16 + w * 4);
                            lo = widen2<T>(two.x);
                            hi = widen2<T>(two.y);
                        }
                        mma16816(score[t], q[j * 4 + w], pack_half(lo.x * k_by, hi.x * k_by), pack_half(lo.y * k_by, hi.y * k_by));
                    }
                }
            }
            uint32_t prob[2][4];
            probabilities(score, full, k_back, v_back, prob);
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int at = half * 16 + 4 * c + e;
                        v[e] = at < held ? widen<T>(v_tail[at * D + j * 8 + g]) : 0.0f;
                        // (a probability of zero times an infinity would be NaN in rows that do not see the token: added below)
                        v[e] = fabsf(v[e]) <= 3.4028235e38f ? v[e] * v_by : 0.0f;
                    }
                    mma16816(acc[j], prob[half], pack_half(v[0], v[2]), pack_half(v[1], v[3]));
                }
            }
            if (odd_values) {
                for (int t = 0; t < held; ++t) {
                    for (int j = 0; j < kTiles; ++j) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float v = widen<T>(v_tail[t * D + j * 8 + c * 2 + (e & 1)]);
                            if (!(fabsf(v) <= 3.4028235e38f) && token + t <= place[e >> 1]) acc[j][e] += v;
                        }
                    }
                }
            }
        }
        if (!healthy) break;

        // rows of this run: sums of a row's four lanes, then the teams'
        const float to_value = unit_scale / kHeadroom;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
        }
        const bool whole = begin == 0 && stop == s.blocks;
        float* part = whole ? nullptr : part_of(p, blockIdx.x, first_segment, kTileRows, D);
        const int tile_rows = min(kTileRows, rows - tile * kTileRows);
        auto row_out = [&](int row) {              // of the tile
            const int at = tile * kTileRows + row;
            return reinterpret_cast<T*>(p.out) +
                   ((static_cast<size_t>(b) * p.tokens + at / p.group) * p.q_heads + head * p.group + at % p.group) * D;
        };
        if constexpr (kTeams == 1) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = member * 16 + g + 8 * r;
                if (row >= tile_rows) continue;
                if (whole) {
                    const float by = sum[r] > 0.0f ? to_value / sum[r] : sum[r] == 0.0f ? 0.0f : sum[r];
                    uint32_t* to = reinterpret_cast<uint32_t*>(row_out(row));
#pragma unroll
                    for (int j = 0; j < kTiles; ++j) to[j * 4 + c] = narrow2<T>(acc[j][2 * r] * by, acc[j][2 * r + 1] * by);
                } else {
                    float* to = part + row * (D + 2);
#pragma unroll
                    for (int j = 0; j < kTiles; ++j) {
                        *reinterpret_cast<float2*>(to + j * 8 + c * 2) = make_float2(acc[j][2 * r] * to_value, acc[j][2 * r + 1] * to_value);
                    }
                    if (c == 0) *reinterpret_cast<float2*>(to + D) = make_float2(top[r], sum[r]);
                }
            }
        } else {
            __syncthreads();                        // an earlier segment's rows have been read
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = member * 16 + g + 8 * r;
                if (row >= tile_rows) continue;
                float* to = merge + (team * kTileRows + row) * (D + 2);
#pragma unroll
                for (int j = 0; j < kTiles; ++j) {
                    *reinterpret_cast<float2*>(to + j * 8 + c * 2) = make_float2(acc[j][2 * r] * to_value, acc[j][2 * r + 1] * to_value);
                }
                if (c == 0) *reinterpret_cast<float2*>(to + D) = make_float2(top[r], sum[r]);
            }
            __syncthreads();
            for (int at = tid; at < tile_rows * (D / 2); at += kThreads) {
                const int row = at / (D / 2), d = at % (D / 2) * 2;
                const float* from = merge + row * (D + 2);
                float best = kNone;
#pragma unroll
                for (int t = 0; t < kTeams; ++t) best = fmaxf(best, from[t * kTileRows * (D + 2) + D]);
                float all = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
                for (int t = 0; t < kTeams; ++t) {
                    const float* of = from + t * kTileRows * (D + 2);
                    const float w = exp2_fast(of[D] - best);
                    const float2 v = *reinterpret_cast<const float2*>(of + d);
                    all += w * of[D + 1];
                    x += w * v.x;
                    y += w * v.y;
                }
                if (whole) {
                    const float by = all > 0.0f ? 1.0f / all : all;
                    *reinterpret_cast<uint32_t*>(row_out(row) + d) = narrow2<T>(x * by, y * by);
                } else {
                    float* to = part + row * (D + 2);
                    *reinterpret_cast<float2*>(to + d) = make_float2(x, y);
                    if (d == 0) *reinterpret_cast<float2*>(to + D) = make_float2(best, all);
                }
            }
        }
        position += stop - begin;
        first_segment = false;
    }
    if (!healthy) {                                 // wait, within limits, for copies that are still on their way
        if (lane == 0 && member == 0) {
            for (unsigned s = take; s < fill; ++s) mbar_wait(smem_u32(&bars[team][s % kStages][0]), (s / kStages) & 1, kKvGaveUp, p.cache.status);
        }
    }
}

// Adds up the parts of the sequences and heads that several runs share; one CTA for each row of each tile.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads)
kv_combine_kernel(const AttentionParams p, int tile_rows) {
    __shared__ float sums[kWarps][D], tops[kWarps], weights[kWarps];
    __shared__ long long plan[2];                    // all blocks; blocks before this sequence
    pdl_release_downstream();
    pdl_wait_for_upstream();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rows_at_most = p.tokens * p.group;
    const int row = blockIdx.x % rows_at_most;
    const int pair = blockIdx.x / rows_at_most, b = pair / p.cache.kv_heads, head = pair % p.cache.kv_heads;
    const Sequence s = sequence_of(p, b, tile_rows);
    if (row >= s.count * p.group || s.blocks == 0) return;
    if (warp == 0) {
        long long total = 0, before = 0;
        for (int i = lane; i < p.cache.batch; i += 32) {
            const long long work = work_of(p, sequence_of(p, i, tile_rows));
            total += work;
            if (i < b) before += work;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            total += __shfl_xor_sync(0xffffffffu, total, o);
            before += __shfl_xor_sync(0xffffffffu, before, o);
        }
        if (lane == 0) {
            plan[0] = total;
            plan[1] = before;
        }
    }
    __syncthreads();
    const long long total = plan[0];
    const int active = active_ctas(p, total);
    const int tile = row / tile_rows;
    const long long begin = plan[1] + (static_cast<long long>(head) * s.row_tiles + tile) * s.blocks, end = begin + s.blocks;
    // the runs that hold its first and its last block: the last whose begin is not behind it
    auto run_of = [&](long long block) {
        int at = static_cast<int>(block * active / total);
        while (at + 1 < active && run_begin(total, active, at + 1) <= block) ++at;
        while (at > 0 && run_begin(total, active, at) > block) --at;
        return at;
    };
    const int first = run_of(begin), last = run_of(end - 1);
    if (first == last) return;                       // one run has it all, and has written the result
    const int in_tile = row % tile_rows;
    float best = kNone, weight = 0.0f, acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
    auto part = [&](int run) {
        return part_of(p, run, run_begin(total, active, run) >= begin, tile_rows, D) + in_tile * (D + 2);
    };
    for (int run = first + warp; run <= last; run += kWarps) best = fmaxf(best, part(run)[D]);
#pragma unroll 4
    for (int run = first + warp; run <= last; run += kWarps) {
        const float* from = part(run);
        const float w = exp2_fast(from[D] - best);
        weight += w * from[D + 1];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] += w * from[i * 32 + lane];
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) sums[warp][i * 32 + lane] = acc[i];
    if (lane == 0) {
        tops[warp] = best;
        weights[warp] = weight;
    }
    __syncthreads();
    if (tid < D) {
        float all = 0.0f, x = 0.0f;
        best = kNone;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) best = fmaxf(best, tops[w]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float by = exp2_fast(tops[w] - best);
            all += by * weights[w];
            x += by * sums[w][tid];
        }
        T* to = reinterpret_cast<T*>(p.out) +
                ((static_cast<size_t>(b) * p.tokens + row / p.group) * p.q_heads + head * p.group + row % p.group) * D;
        to[tid] = narrow<T>(all > 0.0f ? x / all : all);
    }
}

struct DeviceState {
    int sms = 0;
};

template <typename T, int D, int MT>
int allow_shared() {
    return cudaFuncSetAttribute(kv_attention_kernel<T, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(AttentionShape<T, D, MT>::kSharedBytes)) == cudaSuccess
               ? 0
               : W4A16_ERR_LAUNCH;
}

template <typename T>
int allow_all() {
    int status = 0;
    status |= allow_shared<T, 64, 1>() | allow_shared<T, 64, 2>() | allow_shared<T, 64, 4>();
    status |= allow_shared<T, 128, 1>() | allow_shared<T, 128, 2>() | allow_shared<T, 128, 4>();
    return status;
}

int device_state(const DeviceState** state) {
    static PerDevice<DeviceState> devices;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= kMaxDevices) return W4A16_ERR_LAUNCH;
    return devices.get(device, [&](DeviceState& fresh) -> int {
        if (cudaDeviceGetAttribute(&fresh.sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return W4A16_ERR_LAUNCH;
        return allow_all<__half>() != 0 || allow_all<__nv_bfloat16>() != 0 ? W4A16_ERR_LAUNCH : 0;
    }, state);
}

// 16-row tiles of a team: as many as hold the rows, at most four.
int tiles_for(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

struct Shape {
    int mt, row_tiles;
    int64_t units, grid;
    bool split;
};

Shape shape_of(const w4a16_kv8_cache& cache, int q_heads, int64_t tokens, int sms) {
    Shape s{};
    const int64_t rows = tokens * (q_heads / cache.kv_heads);
    s.mt = tiles_for(rows);
    s.row_tiles = static_cast<int>((rows + 16 * s.mt - 1) / (16 * s.mt));
    s.units = static_cast<int64_t>(cache.batch) * cache.kv_heads * s.row_tiles;
    const int64_t blocks = (cache.max_len + kKvBlock - 1) / kKvBlock;
    s.split = blocks > kMinRun;
    s.grid = s.split ? std::min<int64_t>(2 * sms, std::max<int64_t>(1, s.units * blocks / kMinRun)) : s.units;
    return s;
}

template <typename T, int D>
int launch_shape(const AttentionParams& p, const Shape& s, bool programmatic, cudaStream_t stream) {
    auto run = [&](auto tiles) {
        constexpr int kMt = decltype(tiles)::value;
        return kv_launch(kv_attention_kernel<T, D, kMt>, dim3(static_cast<unsigned>(s.grid)), dim3(kThreads),
                         AttentionShape<T, D, kMt>::kSharedBytes, programmatic, stream, p);
    };
    const int status = s.mt == 1   ? run(std::integral_constant<int, 1>{})
                       : s.mt == 2 ? run(std::integral_constant<int, 2>{})
                                   : run(std::integral_constant<int, 4>{});
    if (status != W4A16_OK || !s.split) return status;
    const int64_t rows = static_cast<int64_t>(p.cache.batch) * p.cache.kv_heads * p.tokens * p.group;
    // (always programmatic: it waits for the kernel in front itself, which is the one above)
    return kv_launch(kv_combine_kernel<T, D>, dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, true, stream, p, 16 * s.mt);
}

}  // namespace

size_t kv_attention_workspace_bytes(const w4a16_kv8_cache& cache, int q_heads, int64_t tokens) {
    const DeviceState* state = nullptr;
    const int sms = device_state(&state) == 0 ? state->sms : 148;
    const Shape s = shape_of(cache, q_heads, tokens, sms);
    return s.split ? static_cast<size_t>(s.grid) * 2 * 16 * s.mt * (cache.head_dim + 2) * sizeof(float) : 0;
}

int launch_kv_attention(const w4a16_kv8_cache& cache, const w4a16_rows& q, void* out, int q_heads, int64_t tokens,
                        const long long* lengths, const long long* counts, float softmax_scale, void* workspace, size_t workspace_bytes,
                        bool programmatic, cudaStream_t stream) {
    const DeviceState* state = nullptr;
    if (const int status = device_state(&state); status != 0) return status;
    const Shape s = shape_of(cache, q_heads, tokens, state->sms);
    const int64_t rows = static_cast<int64_t>(cache.batch) * q_heads * tokens;
    if (rows > INT32_MAX || s.units > INT32_MAX) return W4A16_ERR_TOO_LARGE;
    if (s.split && (workspace == nullptr || workspace_bytes < kv_attention_workspace_bytes(cache, q_heads, tokens))) return W4A16_ERR_WORKSPACE;
    AttentionParams p{};
    p.cache = kv_view(cache);
    p.q = static_cast<const char*>(q.data);
    p.q_batch = q.batch_stride;
    p.q_token = q.token_stride;
    p.q_head = q.head_stride;
    p.q_wide = reinterpret_cast<uintptr_t>(q.data) % 16 == 0 && q.batch_stride % 8 == 0 && q.token_stride % 8 == 0 && q.head_stride % 8 == 0;
    p.out = static_cast<char*>(out);
    p.tokens = static_cast<int>(tokens);
    p.q_heads = q_heads;
    p.group = q_heads / cache.kv_heads;
    p.row_tiles = s.row_tiles;
    p.lengths = lengths;
    p.counts = counts;
    p.scale = softmax_scale * kLog2e;
    p.parts = static_cast<float*>(workspace);
    p.grid = static_cast<int>(s.grid);
    p.split = s.split;
    const bool bf16 = cache.type == W4A16_TYPE_BF16;
    if (cache.head_dim == 64) {
        return bf16 ? launch_shape<__nv_bfloat16, 64>(p, s, programmatic, stream) : launch_shape<__half, 64>(p, s, programmatic, stream);
    }
    return bf16 ? launch_shape<__nv_bfloat16, 128>(p, s, programmatic, stream) : launch_shape<__half, 128>(p, s, programmatic, stream);
}

}  // namespace w4a16
