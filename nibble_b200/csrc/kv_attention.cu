// Attention of a sequence's newest tokens over its 8-bit cache (format: kv_cache.cuh).
//
// Query i of `count` stands at position length - count + i and sees the positions up to its own:
//     out = sum_t p_t v_t / sum_t p_t,   p_t = exp(softmax_scale * q . k_t - max)
// The queries of all heads that share a key/value head are rows of one problem (row = i * group + head in group).  They are the
// eight columns of mma.sync m16n8k16, and keys and (transposed) values its sixteen rows: one token of a model with eight query heads
// for each key/value head fills a tile.  (With the queries as the sixteen rows half of every tile was empty.)  Codes enter the
// products as exact FP16 integers, made of bytes by XOR-ing them into 1024 + 128 (one LOP3 for two, then 1152 is subtracted); the key's
// scale multiplies the FP32 score, the value's goes into the probability before that is rounded to FP16.  What is rounded, a probability
// times the scale of its values, is held relative to the largest of those that the row has seen, times 2^10, whatever the largest
// probability: FP16 has its eleven bits down to 2^-24 of that.  Where the results are BF16 that is all; where they are FP16 what the
// rounding left takes part in a second product, so that results are off by their own rounding alone (without it by 1.4 to 1.5 times
// that, root mean square, and one token over 65501 takes 29.7 us instead of 29.9, 8 sequences of 8000 with 32 rows 60 instead of 69).
// Scores, maxima, sums and outputs are FP32.
//
// Bound: HBM, one byte a number of the cache.  A warp streams blocks of its own through a ring in shared memory (bulk copies: 4 KB of
// keys and 4 KB of values at D = 128), keeps its own running maximum, sum and output, and meets the others at the end of a run
// only.  All blocks of all sequences and heads are cut into equal runs, one for each CTA, whatever the sequences' lengths; what a
// run has of a sequence and head goes to the workspace, and a second kernel, which starts beside the first, adds those parts up in
// order and attends over the block that is being filled.
//
// Measured (64 query heads on 8, D = 128, in a graph): one token over 65501 29.9 us = 4.5 TB/s, of a measured 6.5 for a copy, of which
// 5 us go by before the first block has arrived and 4 after the last; 48 sequences of up to 8192 tokens 73.0 us = 5.5 TB/s.  Short
// contexts are latency: 500 tokens of 32 heads on 4, D = 64, 6.7 us, of which two kernels that do nothing would take 4.7.  (A warp that
// went over a block that is not there while the first lengths are on their way, to have the loop's code at hand, made 6.9 of it 8.0.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <limits.h>

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
constexpr int kMinRun = 4;                      // blocks that are worth a CTA: one a warp (500 tokens took 6.9 us, with eight 8.0)
constexpr int kUnitCost = 8;                    // what starting and ending a sequence, head and tile costs, in blocks
constexpr float kHeadroom = 10.0f;              // weights are held in FP16 times 2^10,
constexpr float kMaxLag = 3.0f;                 // times 2^3 where the maximum has not been followed yet,
constexpr float kMaxRise = 2.0f;                // times 2^2 where the values' scale has not: below 65504 in all

struct AttentionParams {
    KvCache cache;
    const char* q;
    long long q_batch, q_token, q_head;          // strides in numbers
    bool q_wide;                                 // rows can be read 16 bytes at a time
    char* out;                                   // [batch][tokens][q heads][D]
    int tokens, q_heads, group;
    float per_group;                             // 1 / group
    int tile_rows, row_tiles;                    // rows of a CTA, and as many tiles as `tokens` queries make
    const long long* lengths;
    const long long* counts;                     // null: all `tokens` of every sequence
    float scale;                                 // softmax scale * log2 e
    float* parts;                                // workspace: see part_of()
    int grid;                                    // CTAs of the first kernel
};

struct Sequence {
    int length, count, blocks, row_tiles;        // full blocks; tiles of this sequence's queries
    bool sound;
};

__device__ __forceinline__ Sequence sequence_of(const AttentionParams& p, int b) {
    Sequence s{0, 0, 0, 0, false};
    const long long length = p.lengths[b], count = p.counts == nullptr ? p.tokens : p.counts[b];
    if (length < 0 || length > p.cache.max_len || count < 0 || count > p.tokens) return s;
    s.length = static_cast<int>(length);
    s.count = static_cast<int>(count);
    s.blocks = s.length / kKvBlock;
    s.row_tiles = (s.count * p.group + p.tile_rows - 1) / p.tile_rows;
    s.sound = true;
    return s;
}

// Work of a sequence's heads and tiles, in blocks: each starts and ends at the cost of some.  (All of it is less than 2^31: the
// launcher sees to that.)
__device__ __forceinline__ int work_of(const AttentionParams& p, const Sequence& s) {
    return s.blocks == 0 ? 0 : (s.blocks + kUnitCost) * s.row_tiles * p.cache.kv_heads;
}

// What a run has of a sequence, head and tile: for each row D sums, their maximum and the sum of the weights.  Along the runs either
// the tile or the run goes up from one piece to the next, so their sum names the piece.
__device__ __forceinline__ float* part_of(const AttentionParams& p, int b, int head, int tile, int run, int d) {
    const size_t piece = (static_cast<size_t>(b) * p.cache.kv_heads + head) * p.row_tiles + tile + run;
    return p.parts + piece * p.tile_rows * (d + 2);
}

// All work in equal runs: the first `longer` are one block longer than the others.
struct Runs {
    int active, length, longer;
    __device__ __forceinline__ Runs(const AttentionParams& p, int total)
        : active(max(1, min(p.grid, total / kMinRun))), length(total / active), longer(total - active * length) {}
    __device__ __forceinline__ int begin(int cta) const { return cta * length + min(cta, longer); }
    __device__ __forceinline__ int of(int block) const {
        const int in_longer = longer * (length + 1);
        return block < in_longer ? block / (length + 1) : longer + (block - in_longer) / length;
    }
};

// A piece of one sequence, head and tile: full blocks [begin, stop).
struct Segment {
    int b, length, count, head, tile, begin, stop;
};

// Where the next segment of a run up to `end` is looked for: sequence b, the work before it, and the run's next piece of work.
struct Place {
    int b, base, position;
};

__device__ __forceinline__ bool next_segment(const AttentionParams& p, int end, Place& at, Segment& seg) {
    while (at.position < end && at.b < p.cache.batch) {
        const Sequence s = sequence_of(p, at.b);
        const int work = work_of(p, s);
        if (at.position >= at.base + work) {
            at.base += work;
            ++at.b;
            continue;
        }
        const int cost = s.blocks + kUnitCost;
        const int unit = (at.position - at.base) / cost, from = at.position - at.base - unit * cost;
        const int to = min(cost, from + end - at.position);
        at.position += to - from;
        seg.begin = max(0, from - kUnitCost);
        seg.stop = max(0, to - kUnitCost);
        if (seg.begin == seg.stop) continue;
        seg.length = s.length;
        seg.count = s.count;
        seg.head = unit / s.row_tiles;
        seg.tile = unit - seg.head * s.row_tiles;
        seg.b = at.b;
        return true;
    }
    return false;
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A matrix of 8 x 8 16-bit numbers, two of a row in each lane, transposed across the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t pair) {
    uint32_t out;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(out) : "r"(pair));
    return out;
}

// A team of MT warps shares a ring; each has 8 * NT rows of its own, and the kWarps / MT teams take the blocks in turn.
template <typename T, int D, int NT, int MT>
struct AttentionShape {
    static constexpr int kTeams = kWarps / MT;
    static constexpr int kTileRows = 8 * NT * MT;
    static constexpr int kSlotBytes = kKvBlock * D;                    // a block's keys, or its values
    static constexpr int kSlots = (NT == 1 ? 3 : MT == 1 ? 4 : MT == 2 ? 6 : 8) * (128 / D);
    static constexpr int kResident = NT == 1 ? 3 : 2;                  // CTAs that fit an SM, beside one of the second kernel
    static constexpr int kRegisters = NT == 1 ? 152 : 224;
    static constexpr size_t kRingBytes = static_cast<size_t>(kTeams) * kSlots * kSlotBytes;
    static constexpr size_t kMergeBytes = static_cast<size_t>(kTeams) * kTileRows * (D + 2) * sizeof(float);
    static constexpr size_t kSharedBytes = kRingBytes + kMergeBytes + static_cast<size_t>(kTileRows) * D * 2;      // and the queries
    static_assert(kResident * (kSharedBytes + 2048) <= 227 * 1024);
};

// 8-row tiles of a warp in the variants for 32 and 64 rows: as many as its registers hold, since they share what makes FP16 of codes.
// (D = 64, 32 query heads on 4, without the second product: eight sequences of 8000 tokens, 40 rows: four tiles and two warps to a ring
// 37.4 us, two and four 46.0; 24 rows 25.7 and 29.2; short sequences the same within 1 us.)
template <int D>
constexpr int kWide = D == 64 ? 4 : 2;

// What one thread of a team asks for next.  It runs ahead of the team by the ring's slots, across the ends of segments.
struct Feed {
    Place at;
    int left;                          // slots of this segment that have not been asked for
    const uint8_t *keys, *values;      // the team's next block
    unsigned fill;
};

template <typename T, int D, int NT, int MT>
__global__ void __maxnreg__((AttentionShape<T, D, NT, MT>::kRegisters))
kv_attention_kernel(const AttentionParams p) {
    using Shape = AttentionShape<T, D, NT, MT>;
    constexpr int kTeams = Shape::kTeams, kSlots = Shape::kSlots, kTileRows = Shape::kTileRows, kSteps = D / 16;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ __align__(128) uint8_t shared[];
    __shared__ __align__(8) unsigned long long bars[kTeams][kSlots][2];        // full; empty, where several warps share a ring
    __shared__ int plan[3];                    // all work; this CTA's sequence; work before it
    __shared__ __align__(8) float row_scales[kTileRows];       // what the scores of a row are multiplied with
    __shared__ __align__(8) int row_places[kTileRows];         // its query's position
    pdl_wait_for_upstream();
    pdl_release_downstream();                  // (behind the wait: what the next kernel reads of ours before its own wait is there)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int team = warp / MT, member = warp % MT;
    const int g = lane >> 2, c = lane & 3;
    uint8_t* const ring = shared + static_cast<size_t>(team) * kSlots * Shape::kSlotBytes;
    float* const merge = reinterpret_cast<float*>(shared + Shape::kRingBytes);
    uint4* const staged = reinterpret_cast<uint4*>(shared + Shape::kRingBytes + Shape::kMergeBytes);
    const bool feeder = lane == 0 && member == 0;
    if (feeder) {
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(smem_u32(&bars[team][s][0]), 1);
            mbar_init(smem_u32(&bars[team][s][1]), MT);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // this CTA's run: where it begins
    if (p.cache.batch > 1 && warp == 0) {
        const int first_work = lane < p.cache.batch ? work_of(p, sequence_of(p, lane)) : 0;
        int total = first_work;
        for (int b = lane + 32; b < p.cache.batch; b += 32) total += work_of(p, sequence_of(p, b));
        total = __reduce_add_sync(0xffffffffu, total);
        int mine = -1;
        if (total > 0) {
            const Runs runs(p, total);
            if (static_cast<int>(blockIdx.x) < runs.active) mine = runs.begin(blockIdx.x);
        }
        int before = 0;
        for (int base = 0; mine >= 0 && base < p.cache.batch; base += 32) {
            const int work = base == 0 ? first_work : base + lane < p.cache.batch ? work_of(p, sequence_of(p, base + lane)) : 0;
            int upto = work;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += other;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + upto > mine);
            if (past != 0) {
                const int at = __ffs(past) - 1;
                if (lane == at) {
                    plan[1] = base + at;
                    plan[2] = before + upto - work;
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) plan[0] = total;
    }
    __syncthreads();
    const int total = p.cache.batch > 1 ? plan[0] : work_of(p, sequence_of(p, 0));
    if (total == 0) return;
    const Runs runs(p, total);
    if (static_cast<int>(blockIdx.x) >= runs.active) return;
    Place at{0, 0, runs.begin(blockIdx.x)};
    if (p.cache.batch > 1) {
        at.b = plan[1];
        at.base = plan[2];
    }
    const int end = runs.begin(blockIdx.x + 1);

    bool healthy = true;
    Feed feed{at, 0, nullptr, nullptr, 0};           // (the feeder's; others' stays as it is)
    // Asks for what the team needs next, if there is anything left: by the feeder, into the slot that has just become free.
    auto ask = [&]() {
        while (feed.left == 0) {
            Segment seg;
            if (!next_segment(p, end, feed.at, seg)) return;
            const size_t from = ((static_cast<size_t>(seg.b) * p.cache.kv_heads + seg.head) * p.cache.blocks + seg.begin + team) * Shape::kSlotBytes;
            feed.left = 2 * max(0, (seg.stop - seg.begin - team + kTeams - 1) / kTeams);
            feed.keys = p.cache.k_codes + from;
            feed.values = p.cache.v_codes + from;
        }
        const unsigned slot = feed.fill % kSlots;
        if (MT > 1 && feed.fill >= kSlots &&
            !mbar_wait<false, true>(smem_u32(&bars[team][slot][1]), (feed.fill / kSlots - 1) & 1, kKvGaveUp, p.cache.status)) {
            healthy = false;
            return;
        }
        const unsigned full_bar = smem_u32(&bars[team][slot][0]);
        mbar_arrive_expect_tx(full_bar, Shape::kSlotBytes);
        bulk_load(smem_u32(ring + slot * Shape::kSlotBytes), feed.left & 1 ? feed.values : feed.keys, Shape::kSlotBytes, full_bar);
        (feed.left & 1 ? feed.values : feed.keys) += kTeams * Shape::kSlotBytes;
        --feed.left;
        ++feed.fill;
    };
    unsigned take = 0;                           // slots that this warp has used
    // A slot, once it has been filled; null if that did not happen.
    auto arrived = [&](unsigned number) -> const uint8_t* {
        const unsigned slot = number % kSlots;
        healthy = mbar_wait<false, true>(smem_u32(&bars[team][slot][0]), (number / kSlots) & 1, kKvGaveUp, p.cache.status) && healthy;
        healthy = __all_sync(0xffffffffu, healthy);
        return healthy ? ring + slot * Shape::kSlotBytes : nullptr;
    };
    auto release = [&]() {
        // (the slot was read through the generic proxy and is refilled through the async one: each lane orders its own reads)
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            if (MT > 1) mbar_arrive(smem_u32(&bars[team][take % kSlots][1]));
            if (member == 0) ask();
        }
        ++take;
    };
    bool first_segment = true;
    Segment seg;
    while (next_segment(p, end, at, seg)) {
        const int first_block = seg.begin + team;
        const size_t pair = static_cast<size_t>(seg.b) * p.cache.kv_heads + seg.head;
        const float* k_scales = p.cache.k_scales + pair * p.cache.blocks;
        const float* v_scales = p.cache.v_scales + pair * p.cache.blocks;
        const int coded = max(0, (seg.stop - first_block + kTeams - 1) / kTeams);
        float k_scale_set, v_scale_set;            // lane l: of this team's block number l since the last set
        auto load_scales = [&](int block) {
            const int mine = block + lane * kTeams;
            k_scale_set = mine < seg.stop ? k_scales[mine] : 0.0f;
            v_scale_set = mine < seg.stop ? v_scales[mine] : 0.0f;
        };
        load_scales(first_block);

        const int rows = seg.count * p.group, first_row = seg.tile * kTileRows;
        // The queries, requested in front of the codes: a thread takes sixteen dims of a row.
        constexpr int kPieces = (kTileRows * kSteps + kThreads - 1) / kThreads;       // of a thread
        uint32_t pieces[kPieces][8];
#pragma unroll
        for (int e = 0; e < kPieces; ++e) {
            const int at = tid + e * kThreads, row = first_row + at / kSteps, token = by_group(p, row);
            const bool there = at < kTileRows * kSteps && row < rows;
            const T* from = reinterpret_cast<const T*>(p.q) + seg.b * p.q_batch + token * p.q_token +
                            (seg.head * p.group + row - token * p.group) * p.q_head + at % kSteps * 16;
            uint32_t (&raw)[8] = pieces[e];
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i] = 0;
            if (there && p.q_wide) {
                const uint4 a = *reinterpret_cast<const uint4*>(from), b = *(reinterpret_cast<const uint4*>(from) + 1);
                raw[0] = a.x; raw[1] = a.y; raw[2] = a.z; raw[3] = a.w;
                raw[4] = b.x; raw[5] = b.y; raw[6] = b.z; raw[7] = b.w;
            } else if (there) {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(from);
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[i] = h[2 * i] | static_cast<uint32_t>(h[2 * i + 1]) << 16;
            }
        }
        if (first_segment && member == 0) {        // the ring's first slots: a lane for each, as far as this segment goes
            const int now = min(kSlots, 2 * coded);
            const uint8_t* keys = p.cache.k_codes + (pair * p.cache.blocks + first_block) * Shape::kSlotBytes;
            const uint8_t* values = p.cache.v_codes + (pair * p.cache.blocks + first_block) * Shape::kSlotBytes;
            if (lane < now) {
                const unsigned full_bar = smem_u32(&bars[team][lane][0]);
                mbar_arrive_expect_tx(full_bar, Shape::kSlotBytes);
                bulk_load(smem_u32(ring + lane * Shape::kSlotBytes), (lane & 1 ? values : keys) + lane / 2 * kTeams * Shape::kSlotBytes,
                          Shape::kSlotBytes, full_bar);
            }
            feed.at = at;
            feed.left = 2 * coded - now;
            feed.keys = keys + (now + 1) / 2 * kTeams * Shape::kSlotBytes;
            feed.values = values + now / 2 * kTeams * Shape::kSlotBytes;
            feed.fill = now;
            if (lane == 0) {
                for (int i = now; i < kSlots; ++i) ask();
            }
        }
        // They become the second operand: [8-row tile][two steps of sixteen dims][lane][...], dims in the order of the codes' bytes.
#pragma unroll
        for (int e = 0; e < kPieces; ++e) {
            const int at = tid + e * kThreads;
            if (at >= kTileRows * kSteps) break;       // (all of a warp)
            const int tile_row = at / kSteps, chunk = at % kSteps, row = first_row + tile_row;
            uint32_t (&raw)[8] = pieces[e];
            float back = 1.0f;
            if constexpr (kBf16) {
                // BF16 queries become FP16 by a power of two of their row's own: a number keeps all its bits unless it is 2^-23
                // of the row's largest or less.  FP16 ones are taken as they are.
                uint32_t largest = 0;                  // (FP32 bits: those of numbers without a sign are ordered like them)
#pragma unroll
                for (int i = 0; i < 8; ++i) largest = max(largest, max(raw[i] << 16 & 0x7fffffffu, raw[i] & 0x7fff0000u));
#pragma unroll
                for (int o = 1; o < kSteps; o <<= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
                const float by = power_for(__uint_as_float(min(largest, 0x7f7f0000u)), back);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 f = widen2<T>(raw[i]);
                    raw[i] = pack_half(f.x * by, f.y * by);
                }
            }
            // dims 4 w .. 4 w + 3 of the sixteen are step w of their run of 64: the first and third, the second and fourth
#pragma unroll
            for (int w = 0; w < 4; w += 2) {
                const int to = (tile_row / 8 * (kSteps / 2) + chunk / 4 * 2 + w / 2) * 32 + tile_row % 8 * 4 + chunk % 4;
                staged[to] = make_uint4(prmt(raw[2 * w], raw[2 * w + 1], 0x5410), prmt(raw[2 * w], raw[2 * w + 1], 0x7632),
                                        prmt(raw[2 * w + 2], raw[2 * w + 3], 0x5410), prmt(raw[2 * w + 2], raw[2 * w + 3], 0x7632));
            }
            if (chunk == 0) {
                row_scales[tile_row] = p.scale * back;
                row_places[tile_row] = row < rows ? seg.length - seg.count + by_group(p, row) : INT_MAX;      // (a row that is not there: anything goes)
            }
        }
        __syncthreads();
        uint32_t q[NT][kSteps][2];
        float q_scale[NT][2];                      // of rows 2c and 2c + 1
        int place[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int tile_row = (member * NT + n) * 8;
#pragma unroll
            for (int i = 0; i < kSteps; i += 2) {
                const uint4 four = staged[(tile_row / 8 * (kSteps / 2) + i / 2) * 32 + lane];
                q[n][i][0] = four.x;
                q[n][i][1] = four.y;
                q[n][i + 1][0] = four.z;
                q[n][i + 1][1] = four.w;
            }
            const float2 scales = *reinterpret_cast<const float2*>(row_scales + tile_row + 2 * c);
            const int2 places = *reinterpret_cast<const int2*>(row_places + tile_row + 2 * c);
            q_scale[n][0] = scales.x;
            q_scale[n][1] = scales.y;
            place[n][0] = places.x;
            place[n][1] = places.y;
        }
        const int lowest = row_places[member * NT * 8];        // (positions go up with the rows)

        float acc[NT][kSteps][4];                  // dims 16 j + g and + 8, rows 2c and 2c + 1
        // The largest score so far, the sum of the probabilities relative to it (of this lane's tokens), and the logarithm of what a
        // probability times its values' scale is multiplied with for the product: what brings the largest of those that the row has
        // seen to 2^10, wherever the largest probability is.
        float top[NT][2], sum[NT][2], level[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < kSteps; ++j) acc[n][j][0] = acc[n][j][1] = acc[n][j][2] = acc[n][j][3] = 0.0f;
            top[n][0] = top[n][1] = kNone;
            sum[n][0] = sum[n][1] = level[n][0] = level[n][1] = 0.0f;
        }

        // Scores of a block, [group of 16 tokens][token 2g: rows 2c, 2c + 1; token 2g + 1: the same], and the probabilities that come
        // of them, as operands of the second product: row g, tokens 4c, 4c + 2 and 4c + 1, 4c + 3 of each group.
        uint32_t prob[NT][2][2], rest[NT][2][2];       // (of FP16 caches)
        auto probabilities = [&](float (&score)[NT][2][4], int block, float k_scale, float v_scale) {
            const int token = block * kKvBlock + 2 * g;
            const float v_log = __log2f(v_scale);   // (minus infinity for a block of zeros, or NaN)
            bool lag = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    // (rounded here and the maximum taken off later: what is off by a rounding of 10^12 is then so for equal scores alike)
                    const float by = k_scale * q_scale[n][r], limit = top[n][r] == kNone ? -INFINITY : top[n][r] + kMaxLag;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        float& x = score[n][t >> 1][(t & 1) * 2 + r];
                        x *= by;
                        lag = lag || x > limit;
                    }
                    lag = lag || level[n][r] + v_log > kHeadroom + kMaxRise;
                }
            }
            if ((block + 1) * kKvBlock - 1 > lowest) {
                lag = true;                         // (what is masked now may have been what was large)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        if (token + (t >> 2) * 16 + (t >> 1 & 1) > place[n][t & 1]) score[n][t >> 2][t & 3] = -INFINITY;
                    }
                }
            }
            if (__any_sync(0xffffffffu, lag)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float shrink[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float here = fmaxf(fmaxf(score[n][0][r], score[n][0][2 + r]), fmaxf(score[n][1][r], score[n][1][2 + r]));
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, o));
                        const bool fresh = top[n][r] == kNone;
                        const float now = fmaxf(here, top[n][r]);         // (kNone while nothing has been seen)
                        // the largest weight, relative to the largest score: the one so far, and this block's
                        const float held = fresh ? -INFINITY : kHeadroom - level[n][r] + (top[n][r] - now);
                        const float largest = fmaxf(held, here - now + fmaxf(v_log, kLightest));
                        shrink[r] = fresh ? 1.0f : exp2_fast(held - largest);
                        sum[n][r] *= fresh ? 1.0f : exp2_fast(top[n][r] - now);
                        level[n][r] = now == kNone ? 0.0f : kHeadroom - largest;
                        top[n][r] = now;
                    }
#pragma unroll
                    for (int j = 0; j < kSteps; ++j) {
                        acc[n][j][0] *= shrink[0];
                        acc[n][j][1] *= shrink[1];
                        acc[n][j][2] *= shrink[0];
                        acc[n][j][3] *= shrink[1];
                    }
                }
            }
            const bool spoilt = v_scale != v_scale;  // the block's values are NaN, for the rows that see any of them
            if (spoilt) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (block * kKvBlock <= place[n][0]) sum[n][0] = __int_as_float(0x7fc00000);
                    if (block * kKvBlock <= place[n][1]) sum[n][1] = __int_as_float(0x7fc00000);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                // relative to the maximum so far, or to zero while the row has seen nothing
                float from[2], weight[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    from[r] = top[n][r] == kNone ? 0.0f : top[n][r];
                    weight[r] = spoilt ? 0.0f : exp2_fast(fminf(level[n][r] + v_log, 126.0f));
                }
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    float w[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float e = exp2_fast(score[n][t >> 1][(t & 1) * 2 + r] - from[r]);
                        sum[n][r] += e;
                        w[r] = e * weight[r];
                    }
                    const uint32_t rounded = pack_half(w[0], w[1]);
                    prob[n][t >> 1][t & 1] = transpose8x8(rounded);
                    if (!kBf16) {                   // what the rounding left, for a product of its own
                        const float2 held = widen2<__half>(rounded);
                        rest[n][t >> 1][t & 1] = transpose8x8(pack_half(w[0] - held.x, w[1] - held.y));
                    }
                }
            }
        };

        for (int i = 0; i < coded; ++i) {
            const int block = first_block + i * kTeams;
            if ((i & 31) == 0 && i > 0) load_scales(block);
            const uint8_t* keys = arrived(take);
            if (keys == nullptr) break;
            float score[NT][2][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int t = 0; t < 4; ++t) score[n][0][t] = score[n][1][t] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 even_token = *reinterpret_cast<const uint4*>(keys + ((half * 2) * (D / 64) + j) * 512 + lane * 16);
                    const uint4 odd_token = *reinterpret_cast<const uint4*>(keys + ((half * 2 + 1) * (D / 64) + j) * 512 + lane * 16);
                    const uint32_t even_words[4] = {even_token.x, even_token.y, even_token.z, even_token.w};
                    const uint32_t odd_words[4] = {odd_token.x, odd_token.y, odd_token.z, odd_token.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t a[4];
                        codes_to_half(even_words[w], a[0], a[2]);
                        codes_to_half(odd_words[w], a[1], a[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma16816(score[n][half], a, q[n][j * 4 + w][0], q[n][j * 4 + w][1]);
                    }
                }
            }
            release();
            probabilities(score, block, __shfl_sync(0xffffffffu, k_scale_set, i & 31), __shfl_sync(0xffffffffu, v_scale_set, i & 31));
            const uint8_t* values = arrived(take);
            if (values == nullptr) break;
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                const uint4 codes = *reinterpret_cast<const uint4*>(values + j * 512 + lane * 16);
                const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};     // [half of the sixteen dims][token group]
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t a[4];
                    codes_to_half(words[half], a[0], a[2]);
                    codes_to_half(words[2 + half], a[1], a[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma16816(acc[n][j], a, prob[n][half][0], prob[n][half][1]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (!kBf16) mma16816(acc[n][j], a, rest[n][half][0], rest[n][half][1]);
                    }
                }
            }
            release();
        }

        if (!healthy) break;

        // rows of this segment: a row's sums, then the teams' results
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) sum[n][r] += __shfl_xor_sync(0xffffffffu, sum[n][r], o);
            }
        }
        __syncthreads();                            // the segment before has been read
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float to_value = exp2_fast(-level[n][r]), shrink = kBf16 ? kShrink : 1.0f;
                float* to = merge + (team * kTileRows + member * 8 * NT + n * 8 + 2 * c + r) * (D + 2);
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    to[j * 16 + g] = acc[n][j][r] * shrink * to_value;
                    to[j * 16 + 8 + g] = acc[n][j][2 + r] * shrink * to_value;
                }
                if (g == 0) *reinterpret_cast<float2*>(to + D) = make_float2(top[n][r], sum[n][r]);
            }
        }
        __syncthreads();
        float* part = part_of(p, seg.b, seg.head, seg.tile, blockIdx.x, D);
        const int tile_rows = min(kTileRows, rows - seg.tile * kTileRows);
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
            float* to = part + row * (D + 2);
            *reinterpret_cast<float2*>(to + d) = make_float2(x, y);
            if (d == 0) *reinterpret_cast<float2*>(to + D) = make_float2(best, all);
        }
        first_segment = false;
    }
    if (!healthy && feeder) {                       // wait, within limits, for copies that are still on their way
        for (unsigned s = take; s < feed.fill; ++s) {
            mbar_wait<false, true>(smem_u32(&bars[team][s % kSlots][0]), (s / kSlots) & 1, kKvGaveUp, p.cache.status);
        }
    }
}

// Rows of the output: the parts that the runs have of each, in order, and the block that is being filled, whose 16-bit numbers are
// multiplied in FP32 as they are.  A CTA has `rows` rows of one sequence and key/value head, ROW_WARPS warps for each at a time.  What
// needs no part is done before the kernel in front has ended; that one lets this one start only when all before it has.
template <typename T, int D, int ROW_WARPS>
__global__ void __launch_bounds__(kThreads, ROW_WARPS > 1 ? 9 : 6)
kv_finish_kernel(const AttentionParams p, int rows_per_cta) {
    constexpr int kRows = kWarps / ROW_WARPS;            // at a time
    constexpr int kDims = D / 32;                        // of a lane
    constexpr int kStride = D + 8;                       // of a token's numbers in shared memory
    constexpr float kHeld = std::is_same<T, __nv_bfloat16>::value ? kShrink : 1.0f;      // what sums of values are held times
    __shared__ __align__(16) T keys[kKvBlock * kStride];
    __shared__ __align__(16) T values[kKvBlock * D];
    __shared__ __align__(16) float queries[kRows][D];
    __shared__ float sums[kWarps][D];
    __shared__ float2 states[kWarps];
    __shared__ int plan[2];                              // all work; work before this sequence
    if (p.grid == 0) pdl_wait_for_upstream();            // there is no kernel of ours in front
    pdl_release_downstream();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row_ctas = (p.tokens * p.group + rows_per_cta - 1) / rows_per_cta;
    const int pair = blockIdx.x / row_ctas, b = pair / p.cache.kv_heads, head = pair % p.cache.kv_heads;
    const int first_row = blockIdx.x % row_ctas * rows_per_cta;
    const int last_row = min(first_row + rows_per_cta, p.tokens * p.group);
    const Sequence s = sequence_of(p, b);
    const int held = s.length - s.blocks * kKvBlock;
    {
        const size_t from = (static_cast<size_t>(pair) * 2 + (s.blocks & 1)) * kKvBlock * D * sizeof(T);
        const uint4* k_tail = reinterpret_cast<const uint4*>(p.cache.k_tail + from);
        const uint4* v_tail = reinterpret_cast<const uint4*>(p.cache.v_tail + from);
#pragma unroll 4
        for (int i = tid; i < held * D / 8; i += kThreads) {
            *reinterpret_cast<uint4*>(keys + i / (D / 8) * kStride + i % (D / 8) * 8) = k_tail[i];
            reinterpret_cast<uint4*>(values)[i] = v_tail[i];
        }
    }
    if (warp == 0) {
        int total = 0, before = 0;
        for (int i = lane; i < p.cache.batch; i += 32) {
            const int work = work_of(p, i == b ? s : sequence_of(p, i));
            total += work;
            if (i < b) before += work;
        }
        total = __reduce_add_sync(0xffffffffu, total);
        before = __reduce_add_sync(0xffffffffu, before);
        if (lane == 0) {
            plan[0] = total;
            plan[1] = before;
            if (!s.sound) atomicOr(p.cache.status, kKvBadLength);
        }
    }
    for (int base = first_row; base < last_row; base += kRows) {
        const int row = base + warp / ROW_WARPS, i = by_group(p, row), q_head = head * p.group + row - i * p.group;
        const int share = warp % ROW_WARPS;
        const bool there = row < last_row && i < s.count;
        const int position = s.length - s.count + i;
        if (there && share == 0) {
            const T* from = reinterpret_cast<const T*>(p.q) + b * p.q_batch + i * p.q_token + q_head * p.q_head;
#pragma unroll
            for (int e = 0; e < kDims; ++e) queries[warp / ROW_WARPS][e * 32 + lane] = widen<T>(from[e * 32 + lane]);
        }
        __syncthreads();
        // the tail: lane t has token t's score, then each lane its dims
        float top = kNone, weight = 0.0f, acc[kDims];
#pragma unroll
        for (int e = 0; e < kDims; ++e) acc[e] = 0.0f;
        const int seen = there ? min(held, position - s.blocks * kKvBlock + 1) : 0;
        if (share == 0 && seen > 0) {
            float score = -INFINITY;
            if (lane < seen) {
                const float4* q = reinterpret_cast<const float4*>(queries[warp / ROW_WARPS]);
                const uint4* k = reinterpret_cast<const uint4*>(keys + lane * kStride);
                float dot[2] = {0.0f, 0.0f};
#pragma unroll
                for (int e = 0; e < D / 8; ++e) {
                    const uint4 eight = k[e];
                    const float4 q0 = q[2 * e], q1 = q[2 * e + 1];
                    const float2 k0 = widen2<T>(eight.x), k1 = widen2<T>(eight.y), k2 = widen2<T>(eight.z), k3 = widen2<T>(eight.w);
                    dot[0] = fmaf(q0.x, k0.x, fmaf(q0.y, k0.y, fmaf(q0.z, k1.x, fmaf(q0.w, k1.y, dot[0]))));
                    dot[1] = fmaf(q1.x, k2.x, fmaf(q1.y, k2.y, fmaf(q1.z, k3.x, fmaf(q1.w, k3.y, dot[1]))));
                }
                score = (dot[0] + dot[1]) * p.scale;
                top = fmaxf(top, score);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float mine = lane < seen ? exp2_fast(score - top) : 0.0f;
            weight = mine;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) weight += __shfl_xor_sync(0xffffffffu, weight, o);
#pragma unroll 4
            for (int t = 0; t < seen; ++t) {
                const float w = __shfl_sync(0xffffffffu, mine, t) * kHeld;
                const T* v = values + t * D + lane * kDims;
#pragma unroll
                for (int e = 0; e < kDims; e += 2) {
                    const float2 two = widen2<T>(*reinterpret_cast<const uint32_t*>(v + e));
                    acc[e] = fmaf(w, two.x, acc[e]);
                    acc[e + 1] = fmaf(w, two.y, acc[e + 1]);
                }
            }
        }
        const float* parts = nullptr;                     // of this row in the runs that have one, `stride` apart
        int count = 0;
        const size_t stride = static_cast<size_t>(p.tile_rows) * (D + 2);
        if (there && s.blocks > 0) {
            const Runs runs(p, plan[0]);
            const int tile = row / p.tile_rows;
            const int begin = plan[1] + (head * s.row_tiles + tile) * (s.blocks + kUnitCost) + kUnitCost;
            const int first = runs.of(begin);
            count = runs.of(begin + s.blocks - 1) - first + 1;
            parts = part_of(p, b, head, tile, first, D) + row % p.tile_rows * (D + 2);
        }
        // Before the first rows' parts are there the loop below goes over whatever lies in their place, and what comes of that is
        // dropped: it brings the code in, which otherwise takes as long as the work itself.
        const float tail_top = top, tail_weight = weight;
        float tail_acc[kDims];
#pragma unroll
        for (int d = 0; d < kDims; ++d) tail_acc[d] = acc[d];
        for (int pass = base == first_row ? 0 : 1; pass < 2; ++pass) {
            if (pass == 1 && base == first_row) pdl_wait_for_upstream();
            top = tail_top;
            weight = tail_weight;
#pragma unroll
            for (int d = 0; d < kDims; ++d) acc[d] = tail_acc[d];
            // a few parts at a time, all of their numbers requested together
            constexpr int kBatch = 16 / kDims;
            for (int r = share; r < count; r += kBatch * ROW_WARPS) {
                float2 state[kBatch], numbers[kBatch][kDims / 2];          // maximum and sum
                float best = top;
#pragma unroll
                for (int e = 0; e < kBatch; ++e) {
                    const float* from = parts + (r + e * ROW_WARPS) * stride;
                    const bool one = r + e * ROW_WARPS < count;
                    state[e] = one ? __ldcg(reinterpret_cast<const float2*>(from + D)) : make_float2(kNone, 0.0f);
#pragma unroll
                    for (int d = 0; d < kDims / 2; ++d) {
                        numbers[e][d] = one ? __ldcg(reinterpret_cast<const float2*>(from + lane * kDims) + d) : make_float2(0.0f, 0.0f);
                    }
                }
#pragma unroll
                for (int e = 0; e < kBatch; ++e) best = fmaxf(best, state[e].x);
                const float shrink = exp2_fast(top - best);
                top = best;
                weight *= shrink;
#pragma unroll
                for (int d = 0; d < kDims; ++d) acc[d] *= shrink;
#pragma unroll
                for (int e = 0; e < kBatch; ++e) {
                    const float w = exp2_fast(state[e].x - best);
                    weight = fmaf(w, state[e].y, weight);
#pragma unroll
                    for (int d = 0; d < kDims / 2; ++d) {
                        acc[2 * d] = fmaf(w, numbers[e][d].x, acc[2 * d]);
                        acc[2 * d + 1] = fmaf(w, numbers[e][d].y, acc[2 * d + 1]);
                    }
                }
            }
            if (ROW_WARPS > 1) {                          // (one row: the CTA's only one at a time)
                __syncthreads();
#pragma unroll
                for (int e = 0; e < kDims; ++e) sums[warp][lane * kDims + e] = acc[e];
                if (lane == 0) states[warp] = make_float2(top, weight);
                __syncthreads();
                top = kNone;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, states[w].x);
                weight = 0.0f;
#pragma unroll
                for (int e = 0; e < kDims; ++e) acc[e] = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float by = exp2_fast(states[w].x - top);
                    weight += by * states[w].y;
#pragma unroll
                    for (int e = 0; e < kDims; ++e) acc[e] += by * sums[w][lane * kDims + e];
                }
            }
        }
        if (row < last_row && share == 0) {
            const float by = weight > 0.0f ? 1.0f / kHeld / weight : weight;       // (no weight: nothing is seen)
            T* to = reinterpret_cast<T*>(p.out) + ((static_cast<size_t>(b) * p.tokens + i) * p.q_heads + q_head) * D + lane * kDims;
#pragma unroll
            for (int e = 0; e < kDims; e += 2) *reinterpret_cast<uint32_t*>(to + e) = narrow2<T>(acc[e] * by, acc[e + 1] * by);
        }
        __syncthreads();                                  // the next rows' queries take these rows' place
    }
}

struct DeviceState {
    int sms = 0;
};

template <typename Kernel>
int allow_shared(Kernel kernel, size_t bytes) {
    // (all that an SM has, so that the second kernel's CTAs find room beside the first's)
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) == cudaSuccess &&
                   cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) == cudaSuccess
               ? 0
               : W4A16_ERR_LAUNCH;
}

template <typename T, int D>
int allow_all() {
    return allow_shared(kv_attention_kernel<T, D, 1, 1>, AttentionShape<T, D, 1, 1>::kSharedBytes) |
           allow_shared(kv_attention_kernel<T, D, 2, 1>, AttentionShape<T, D, 2, 1>::kSharedBytes) |
           allow_shared(kv_attention_kernel<T, D, kWide<D>, 4 / kWide<D>>, AttentionShape<T, D, kWide<D>, 4 / kWide<D>>::kSharedBytes) |
           (D == 64 ? allow_shared(kv_attention_kernel<T, 64, kWide<64>, 8 / kWide<64>>, AttentionShape<T, 64, kWide<64>, 8 / kWide<64>>::kSharedBytes) : 0) |
           allow_shared(kv_finish_kernel<T, D, 1>, 0) | allow_shared(kv_finish_kernel<T, D, 4>, 0);
}

int device_state(const DeviceState** state) {
    static PerDevice<DeviceState> devices;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= kMaxDevices) return W4A16_ERR_LAUNCH;
    return devices.get(device, [&](DeviceState& fresh) -> int {
        if (cudaDeviceGetAttribute(&fresh.sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return W4A16_ERR_LAUNCH;
        const int allowed = allow_all<__half, 64>() | allow_all<__half, 128>() | allow_all<__nv_bfloat16, 64>() | allow_all<__nv_bfloat16, 128>();
        return allowed != 0 ? W4A16_ERR_LAUNCH : 0;
    }, state);
}

struct Shape {
    int tile_rows, row_tiles;      // rows of a CTA: 8, 16, 32, or 64 where D is 64
    int64_t units, grid;           // sequences x heads x tiles; CTAs of the first kernel, 0 where no block can be full
    size_t workspace;
};

Shape shape_of(const w4a16_kv8_cache& cache, int q_heads, int64_t tokens, int sms) {
    Shape s{};
    const int64_t rows = tokens * (q_heads / cache.kv_heads);
    s.tile_rows = rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    s.row_tiles = static_cast<int>((rows + s.tile_rows - 1) / s.tile_rows);
    s.units = static_cast<int64_t>(cache.batch) * cache.kv_heads * s.row_tiles;
    const int64_t blocks = cache.max_len / kKvBlock;
    const int resident = s.tile_rows == 8 ? 3 : 2;
    if (blocks > 0) s.grid = std::min<int64_t>(resident * sms, std::max<int64_t>(1, s.units * (blocks + kUnitCost) / kMinRun));
    s.workspace = static_cast<size_t>(s.units + s.grid) * s.tile_rows * (cache.head_dim + 2) * sizeof(float);
    return s;
}

template <typename T, int D>
int launch_shape(const AttentionParams& p, const Shape& s, bool programmatic, cudaStream_t stream) {
    auto run = [&](auto row_tiles, auto members) {
        constexpr int kNt = decltype(row_tiles)::value, kMt = decltype(members)::value;
        return kv_launch(kv_attention_kernel<T, D, kNt, kMt>, dim3(static_cast<unsigned>(s.grid)), dim3(kThreads),
                         AttentionShape<T, D, kNt, kMt>::kSharedBytes, programmatic, stream, p);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    using Wide = std::integral_constant<int, kWide<D>>;
    if (s.grid > 0) {
        int status;
        if (s.tile_rows == 8) {
            status = run(One{}, One{});
        } else if (s.tile_rows == 16) {
            status = run(Two{}, One{});
        } else if (s.tile_rows == 32) {
            status = run(Wide{}, std::integral_constant<int, 4 / kWide<D>>{});
        } else {
            if constexpr (D == 64) status = run(Wide{}, std::integral_constant<int, 8 / kWide<D>>{});
            else return W4A16_ERR_BAD_SHAPE;        // (the other kernel's)
        }
        if (status != W4A16_OK) return status;
    }
    // Behind the first kernel always programmatic: it waits for that one itself.  Four warps a row while rows are few.
    const int64_t pairs = static_cast<int64_t>(p.cache.batch) * p.cache.kv_heads, rows = p.tokens * static_cast<int64_t>(p.group);
    const bool few = pairs * rows <= 1024;
    const int rows_per_cta = few ? 1 : 4;
    const int64_t ctas = pairs * ((rows + rows_per_cta - 1) / rows_per_cta);
    return kv_launch(few ? kv_finish_kernel<T, D, 4> : kv_finish_kernel<T, D, 1>, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), 0,
                     s.grid > 0 || programmatic, stream, p, rows_per_cta);
}

}  // namespace

size_t kv_attention_workspace_bytes(const w4a16_kv8_cache& cache, int q_heads, int64_t tokens) {
    const DeviceState* state = nullptr;
    const int sms = device_state(&state) == 0 ? state->sms : 148;
    const Shape s = shape_of(cache, q_heads, tokens, sms);
    return s.grid > 0 ? s.workspace : 0;
}

int launch_kv_attention(const w4a16_kv8_cache& cache, const w4a16_rows& q, void* out, int q_heads, int64_t tokens,
                        const long long* lengths, const long long* counts, float softmax_scale, void* workspace, size_t workspace_bytes,
                        bool programmatic, cudaStream_t stream) {
    const DeviceState* state = nullptr;
    if (const int status = device_state(&state); status != 0) return status;
    const Shape s = shape_of(cache, q_heads, tokens, state->sms);
    const int64_t rows = static_cast<int64_t>(cache.batch) * q_heads * tokens;
    if (rows > INT32_MAX || rows / cache.batch / cache.kv_heads >= 1 << 24 || s.units > INT32_MAX / (cache.max_len / kKvBlock + kUnitCost)) return W4A16_ERR_TOO_LARGE;
    if (s.grid > 0 && (workspace == nullptr || workspace_bytes < s.workspace)) return W4A16_ERR_WORKSPACE;
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
    p.per_group = 1.0f / static_cast<float>(p.group);
    p.tile_rows = s.tile_rows;
    p.row_tiles = s.row_tiles;
    p.lengths = lengths;
    p.counts = counts;
    p.scale = softmax_scale * kLog2e;
    p.parts = static_cast<float*>(workspace);
    p.grid = static_cast<int>(s.grid);
    const bool bf16 = cache.type == W4A16_TYPE_BF16;
    if (cache.head_dim == 64) {
        return bf16 ? launch_shape<__nv_bfloat16, 64>(p, s, programmatic, stream) : launch_shape<__half, 64>(p, s, programmatic, stream);
    }
    return bf16 ? launch_shape<__nv_bfloat16, 128>(p, s, programmatic, stream) : launch_shape<__half, 128>(p, s, programmatic, stream);
}

}  // namespace w4a16
