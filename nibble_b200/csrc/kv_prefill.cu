// Attention of many new tokens (a prompt, or a chunk of one) over the 8-bit cache, on the 5th-generation tensor cores.
//
// The same definition as kv_attention.cu, and the same arithmetic: codes are exact FP16 integers in both products, the keys' scales
// multiply FP32 scores, the values' scales enter the probabilities before those are rounded to FP16 (relative to the largest such weight
// that the row has seen, times 2^9; here once, without what the rounding leaves), maxima, sums and outputs are FP32.
//
// A unit of work is 256 rows (row = query * group + head in group) of one sequence and key/value head, as two tiles A and B of 128,
// against its visible tokens in steps of 128 (four blocks).  Roles of a CTA's sixteen warps, one CTA per SM:
//   warps 0-3, 4-7   softmax of tile A and of tile B: a thread per row.  Stages its row of queries, then in every step takes the
//                    row's 128 scores out of TMEM, leaves the probabilities there, and in the end takes the output.
//   warps 8-11       make FP16 operands in shared memory of a block's codes each (which they have copied in a step ahead), swizzled by
//                    128 bytes: keys [token][d], values [d][token]; of the block that is being filled, of its 16-bit numbers; zeros
//                    behind the last.
//   warp 12          (13-15: nothing) allocates TMEM and issues the MMAs: S = Q K^T with both operands in shared memory, O += P V
//                    with P in TMEM.
// TMEM: 128 columns of scores, 64 of probabilities for each tile, 128 of outputs for each.
//
// The tiles share the columns of the scores: a softmax thread takes its row's into registers in one go, and the MMAs of the other
// tile's scores, which that will want half a round later, follow in their place.  So neither softmax waits for its scores.
// 2048 queries of 64 heads on 8 at the end of 8192 tokens, D = 128, take 484 us: 0.99 PFLOP/s, of a measured 1.63 for a plain product.
// What it was before: 592 with columns for each tile and the probabilities in the scores' place, where a tile's next scores had to
// wait for its last output, and its softmax for both; 670 with 64 tokens at a time, twice buffered, since MMAs of 64 columns read
// twice as much shared memory a column; 505 with the maximum of every block sought before its probabilities.  Bounds: on paper MMAs
// and exponentials take 2048 clocks of a step each, and shared memory (operands written once and read by two MMAs each) 2800;
// measured, a step is 4530 with what starting and ending a piece costs (600 a step there), of which MMAs are under way in 3060 and a
// softmax in 3400.
//
// Work split.  As many whole units as make full rounds of the CTAs; what is left for the last round is cut along the tokens, where that
// are half as many units as CTAs or fewer, and a small kernel adds the pieces up.  (2048 tokens of 64 heads on 8: 512 units, 148 CTAs.)
//
// Every wait is bounded; one that gives up sets the cache's status word, later ones return at once, and the CTA still runs to its
// TMEM deallocation.
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

constexpr int kRows = 128;                      // of a tile
constexpr int kUnitRows = 2 * kRows;
constexpr int kStepBlocks = 4;
constexpr int kStepTokens = kStepBlocks * kKvBlock;
constexpr int kSoftmaxWarps = 8, kDequantWarps = 4;
constexpr int kMmaWarp = kSoftmaxWarps + kDequantWarps;
constexpr int kPrefillThreads = (kMmaWarp + 4) * 32;      // (registers are handed over by four warps at a time)
// Registers of a thread: of 128 at launch the makers of operands and the issuer give up what the softmax, which holds a row's 128
// scores, is short of.  FP16 at D = 128 leaves the makers more (2048 queries at 8192: 488 us, with the others' split 503); the others do not
// (D = 64 FP16 229 and 222, BF16 94 and 92; D = 128 BF16 255 and 248).
template <typename T, int D>
struct PrefillRegisters {
    static constexpr bool kMakersMore = std::is_same<T, __half>::value && D == 128;
    static constexpr int kSoftmax = kMakersMore ? 200 : 208, kDequant = kMakersMore ? 80 : 64, kIssuer = 32;
    static_assert(2 * kSoftmax + kDequant + kIssuer <= 4 * 128);
};
constexpr float kHeadroom = 9.0f;               // weights are held in FP16 times 2^9 (times 2^10 they outgrow it sooner: 3 % at D = 64)
constexpr float kLightestHalf = -40.0f;         // the same for FP16 (kLightest): all scales are above it but zero
constexpr float kFar = 0x1p16f;                 // a score that is so large is rounded before the maximum is taken off
// What is noted of the block that is being filled: values that are infinite or NaN; BF16 keys or values that lie so far apart that the
// small ones would not keep their bits beside the largest.
constexpr unsigned kOddValues = 1, kApart = 2;
constexpr float kLargestSum = 65000.0f;         // of a block's weights: none is beyond FP16 then

struct PrefillParams {
    KvCache cache;
    const char* q;
    long long q_batch, q_token, q_head;
    bool q_wide;
    char* out;                                   // [batch][tokens][q heads][D]
    int tokens, q_heads, group;
    float per_group;                             // 1 / group
    int row_tiles;                               // units of a sequence and head: as many as `tokens` queries make
    const long long* lengths;
    const long long* counts;
    float scale;                                 // |softmax scale| * log2 e
    bool negate;                                 // the softmax scale is negative: the queries are taken with the other sign
    float* parts;                                // [piece][256][D + 4]: sums, what they are relative to (as two logarithms), sum of probabilities
    int units, whole, pieces;                    // units in all; those of full rounds; pieces of each of the others
};

// A unit or a piece of one: steps [begin, stop) of its visible tokens.
struct Work {
    int b, head, first_row, rows, length, count;      // rows: of the sequence, from row 0 of the unit's tile 0 on
    int begin, stop;
    int full, held;                                   // full blocks, tokens of the block that is being filled
    int piece;                                        // -1: a whole unit
};

__device__ __forceinline__ Work unit_of(const PrefillParams& p, int unit, int piece) {
    Work w;
    const int pairs = p.cache.batch * p.cache.kv_heads;
    const int tile = p.row_tiles - 1 - unit / pairs;      // the longest first
    const int pair = unit % pairs;
    w.b = pair / p.cache.kv_heads;
    w.head = pair - w.b * p.cache.kv_heads;
    w.first_row = tile * kUnitRows;
    w.piece = piece;
    const long long length = p.lengths[w.b], count = p.counts == nullptr ? p.tokens : p.counts[w.b];
    const bool sound = length >= 0 && length <= p.cache.max_len && count >= 0 && count <= p.tokens;
    if (!sound && threadIdx.x == 0) atomicOr(p.cache.status, kKvBadLength);
    w.length = sound ? static_cast<int>(length) : 0;
    w.count = sound ? static_cast<int>(count) : 0;
    w.rows = w.count * p.group;
    w.full = w.length / kKvBlock;
    w.held = w.length - w.full * kKvBlock;
    const int last_row = min(w.rows, w.first_row + kUnitRows) - 1;
    const int last = last_row >= w.first_row ? w.length - w.count + by_group(p, last_row) : -1;      // position of its query
    const int steps = last < 0 ? 0 : last / kStepTokens + 1;
    w.begin = piece < 0 ? 0 : static_cast<int>(static_cast<long long>(steps) * piece / p.pieces);
    w.stop = piece < 0 ? steps : static_cast<int>(static_cast<long long>(steps) * (piece + 1) / p.pieces);
    return w;
}

// This CTA's n-th work; false behind the last.
__device__ __forceinline__ bool work_of(const PrefillParams& p, int n, Work& w) {
    const int unit = static_cast<int>(blockIdx.x) + n * static_cast<int>(gridDim.x);
    if (unit < p.whole) {
        w = unit_of(p, unit, -1);
        return true;
    }
    if (n * static_cast<int>(gridDim.x) != p.whole || static_cast<int>(blockIdx.x) >= (p.units - p.whole) * p.pieces) return false;
    w = unit_of(p, p.whole + blockIdx.x / p.pieces, blockIdx.x % p.pieces);
    return true;
}

template <int D>
struct PrefillShape {
    static constexpr int kHalves = D / 64;                              // 128-byte halves of a row of keys or queries
    static constexpr int kQueryBytes = kRows * D * 2;                   // of a tile
    static constexpr int kKeyBytes = kStepTokens * D * 2, kValueBytes = D * kStepTokens * 2;      // of a step
    static constexpr int kKeysAt = 2 * kQueryBytes, kValuesAt = kKeysAt + 2 * kKeyBytes;
    static constexpr int kCodesAt = kValuesAt + 2 * kValueBytes;
    static constexpr size_t kSharedBytes = kCodesAt + kDequantWarps * 2 * kKvBlock * D + 1024;    // and to align it
};

// Each is waited for phase by phase by whoever waits for it, so that a parity names a phase.
struct PrefillBarriers {
    unsigned long long q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2];
    unsigned long long s_full[2], s_taken[2], p_full[2], o_done[2];      // of a tile
    unsigned long long codes[kDequantWarps][2];
};

// Two FP32 operations an instruction.
__device__ __forceinline__ uint64_t pair_of(uint32_t a, uint32_t b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint64_t pair_of(float a, float b) { return pair_of(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ float2 both_of(uint64_t pair) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(pair));
    return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// D (TMEM) += A (shared memory) x B (shared memory).
__device__ __forceinline__ void umma_f16_shared(unsigned tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t instr_desc,
                                                uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(instr_desc), "r"(accumulate)
        : "memory");
}

// Columns of this thread's TMEM lane, there once this returns.  Load and wait are one statement: between two, registers that have not
// arrived yet could be moved or spilled.
__device__ __forceinline__ void tmem_load32(unsigned address, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(address)
        : "memory");
}
__device__ __forceinline__ void tmem_load128(unsigned address, uint32_t (&v)[128]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%128];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%129];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
        "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95}, [%130];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,"
        "%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%131];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]),
          "=r"(v[32]), "=r"(v[33]), "=r"(v[34]), "=r"(v[35]), "=r"(v[36]), "=r"(v[37]), "=r"(v[38]), "=r"(v[39]),
          "=r"(v[40]), "=r"(v[41]), "=r"(v[42]), "=r"(v[43]), "=r"(v[44]), "=r"(v[45]), "=r"(v[46]), "=r"(v[47]),
          "=r"(v[48]), "=r"(v[49]), "=r"(v[50]), "=r"(v[51]), "=r"(v[52]), "=r"(v[53]), "=r"(v[54]), "=r"(v[55]),
          "=r"(v[56]), "=r"(v[57]), "=r"(v[58]), "=r"(v[59]), "=r"(v[60]), "=r"(v[61]), "=r"(v[62]), "=r"(v[63]),
          "=r"(v[64]), "=r"(v[65]), "=r"(v[66]), "=r"(v[67]), "=r"(v[68]), "=r"(v[69]), "=r"(v[70]), "=r"(v[71]),
          "=r"(v[72]), "=r"(v[73]), "=r"(v[74]), "=r"(v[75]), "=r"(v[76]), "=r"(v[77]), "=r"(v[78]), "=r"(v[79]),
          "=r"(v[80]), "=r"(v[81]), "=r"(v[82]), "=r"(v[83]), "=r"(v[84]), "=r"(v[85]), "=r"(v[86]), "=r"(v[87]),
          "=r"(v[88]), "=r"(v[89]), "=r"(v[90]), "=r"(v[91]), "=r"(v[92]), "=r"(v[93]), "=r"(v[94]), "=r"(v[95]),
          "=r"(v[96]), "=r"(v[97]), "=r"(v[98]), "=r"(v[99]), "=r"(v[100]), "=r"(v[101]), "=r"(v[102]), "=r"(v[103]),
          "=r"(v[104]), "=r"(v[105]), "=r"(v[106]), "=r"(v[107]), "=r"(v[108]), "=r"(v[109]), "=r"(v[110]), "=r"(v[111]),
          "=r"(v[112]), "=r"(v[113]), "=r"(v[114]), "=r"(v[115]), "=r"(v[116]), "=r"(v[117]), "=r"(v[118]), "=r"(v[119]),
          "=r"(v[120]), "=r"(v[121]), "=r"(v[122]), "=r"(v[123]), "=r"(v[124]), "=r"(v[125]), "=r"(v[126]), "=r"(v[127])
        : "r"(address), "r"(address + 32), "r"(address + 64), "r"(address + 96)
        : "memory");
}
__device__ __forceinline__ void tmem_store16(unsigned address, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(address),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
        "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

// Token of a step's column.  Of a block's 32: four tokens of the first sixteen, then the four of the second sixteen that a lane's values
// codes hold beside them, each four in the order 0, 2, 1, 3 in which bytes become pairs of FP16.
__device__ __forceinline__ constexpr int token_of(int column) {
    const int four = column / 4 % 8;
    return column / 32 * 32 + four % 2 * 16 + four / 2 * 4 + (column & 1) * 2 + (column & 2) / 2;
}

// 128-byte swizzle: where 16-byte chunk c of row r of a [rows][128 bytes] tile lies.
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// Of `count` numbers (a multiple of eight, 16-byte aligned), by a warp: the largest finite magnitude, and the smallest of the eights' largest
// that is not zero (infinite, if there is none).  Sets `odd` if one of them is an infinity or NaN.
template <typename T>
__device__ __forceinline__ float2 range_of(const T* numbers, int count, int lane, bool& odd) {
    float top = 0.0f, least = INFINITY;
    bool strange = false;
#pragma unroll 2
    for (int i = lane; i < count / 8; i += 32) {
        const uint4 eight = reinterpret_cast<const uint4*>(numbers)[i];
        const uint32_t words[4] = {eight.x, eight.y, eight.z, eight.w};
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = widen2<T>(words[e]);
            const float a = fabsf(f.x), b = fabsf(f.y);
            if (a <= 3.4028235e38f) most = fmaxf(most, a);
            else strange = true;
            if (b <= 3.4028235e38f) most = fmaxf(most, b);
            else strange = true;
        }
        top = fmaxf(top, most);
        if (most > 0.0f) least = fminf(least, most);
    }
    odd = __any_sync(0xffffffffu, strange);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
    }
    return make_float2(top, least);
}

// The inverse of a power of two.
__device__ __forceinline__ float inverse_power(float power) { return __uint_as_float(0x7f000000u - __float_as_uint(power)); }

// Adds the block that is being filled, of BF16 numbers that lie far apart, to a row's results: all in FP32 from the numbers as they came, a
// thread for its row, as the kernel for few rows does.  `top`, `level` and `sum` are the row's, its numbers lie in TMEM; by a whole warp.
template <int D>
__device__ __forceinline__ void add_tail(const __nv_bfloat16* q, const __nv_bfloat16* keys, const __nv_bfloat16* values, int seen, float scale,
                                         unsigned out_at, float& top, float& level, float& sum) {
    float scores[kKvBlock];
    for (int t = 0; t < kKvBlock; ++t) scores[t] = 0.0f;
    for (int d = 0; d < D; d += 8) {
        float row[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) row[e] = seen > 0 ? __bfloat162float(q[d + e]) : 0.0f;
        for (int t = 0; t < seen; ++t) {
            const uint4 eight = *reinterpret_cast<const uint4*>(keys + t * D + d);
            const uint32_t words[4] = {eight.x, eight.y, eight.z, eight.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 k = widen2<__nv_bfloat16>(words[e]);
                scores[t] = fmaf(row[2 * e], k.x, fmaf(row[2 * e + 1], k.y, scores[t]));
            }
        }
    }
    float now = top;
    for (int t = 0; t < seen; ++t) {
        scores[t] = __fmul_rn(scores[t], scale);
        now = fmaxf(now, scores[t]);
    }
    const float shrink = top > kNone ? exp2_fast(top - now) : 1.0f, factor = exp2_fast(level - kHeadroom) * kShrink * shrink;
    sum *= shrink;
    for (int t = 0; t < seen; ++t) {
        scores[t] = exp2_fast(scores[t] - now);
        sum += scores[t];
    }
#pragma unroll 1
    for (int d = 0; d < D; d += 32) {
        uint32_t o[32];
        tmem_load32(out_at + d, o);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
        for (int t = 0; t < seen; ++t) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                const float v = __bfloat162float(values[t * D + d + e]);
                // (infinities and NaN are added in the end)
                if (fabsf(v) <= 3.4028235e38f) o[e] = __float_as_uint(fmaf(scores[t] * kShrink, v, __uint_as_float(o[e])));
            }
        }
        tmem_store16(out_at + d, o);
        tmem_store16(out_at + d + 16, o + 16);
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    static_assert(kShrink == 0x1p-32f);
    top = now;
    level = kHeadroom + 32.0f;                           // TMEM holds sums times kShrink
}

template <typename T, int D>
__global__ void __launch_bounds__(kPrefillThreads, 1)
kv_prefill_kernel(const PrefillParams p) {
    using Shape = PrefillShape<D>;
    constexpr int kHalves = Shape::kHalves;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    // TMEM columns: scores, probabilities of A, of B, outputs of A, of B
    constexpr unsigned kProbabilities = 128, kOutputs = 256;
    extern __shared__ uint8_t unaligned[];
    __shared__ __align__(8) PrefillBarriers bars;
    __shared__ unsigned tmem_word;
    // Of a step's blocks, keys' and values', four steps: operands are made two steps ahead of the scores, and those of step n + 2 are
    // formed only when both tiles' probabilities of step n + 1 are there.
    // (Keys' scales; logarithms of the values' scales; and, for FP16, the inverses of what those are the logarithms of.)
    __shared__ __align__(16) float4 scales[4][kStepBlocks];
    // What there is to note of a step's block that is being filled: by steps like the factors, written and read at the same places.  (By
    // works it would be overwritten: works without a step are passed over at once, and one tile may be at the end of a work while the
    // other is in the next but three.)
    __shared__ uint8_t tail_notes[4][kStepBlocks];
    uint8_t* const shared = unaligned + (1024 - (smem_u32(unaligned) & 1023)) % 1024;
    pdl_wait_for_upstream();
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (tid == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(smem_u32(&bars.q_full[t]), 4);
            mbar_init(smem_u32(&bars.k_full[t]), kDequantWarps);
            mbar_init(smem_u32(&bars.v_full[t]), kDequantWarps);
            mbar_init(smem_u32(&bars.k_empty[t]), 1);
            mbar_init(smem_u32(&bars.v_empty[t]), 1);
            mbar_init(smem_u32(&bars.s_full[t]), 1);
            mbar_init(smem_u32(&bars.s_taken[t]), 4);
            mbar_init(smem_u32(&bars.p_full[t]), 4);
            mbar_init(smem_u32(&bars.o_done[t]), 1);
        }
        for (int i = 0; i < kDequantWarps; ++i) {
            mbar_init(smem_u32(&bars.codes[i][0]), 1);
            mbar_init(smem_u32(&bars.codes[i][1]), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_word)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_word;
    pdl_release_downstream();                  // (behind the allocation: a kernel that starts beside this one may want TMEM too)
    bool healthy = true;
    // Waits for phase number `n` of a barrier; by a converged warp, all of whose lanes then know whether it came.
    auto wait = [&](unsigned long long& bar, int n) {
        if (healthy) healthy = mbar_wait<false, true>(smem_u32(&bar), n & 1, kKvGaveUp, p.cache.status);
        healthy = __all_sync(0xffffffffu, healthy);
    };
    // This warp's arrival, behind its writes to shared memory for the tensor core.
    auto arrive = [&](unsigned long long& bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar));
    };

    if (warp < kSoftmaxWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PrefillRegisters<T, D>::kSoftmax));
        // ---------------------------------------------------------------- softmax: one row a thread
        const int t = warp / 4, row_in_tile = tid & (kRows - 1);
        const unsigned lanes = static_cast<unsigned>(warp % 4 * 32) << 16;
        const unsigned score_at = tmem + lanes, prob_at = tmem + kProbabilities + t * 64 + lanes, out_at = tmem + kOutputs + t * 128 + lanes;
        int steps_done = 0, steps_of_all = 0;            // of this tile; of both, up to this work
        Work w;
        for (int n = 0; work_of(p, n, w); steps_of_all += w.stop - w.begin, ++n) {
            const int row = w.first_row + t * kRows + row_in_tile, token = by_group(p, row);
            const int place = row < w.rows ? w.length - w.count + token : -1;
            const int q_head = w.head * p.group + row - token * p.group;
            const size_t pair = static_cast<size_t>(w.b) * p.cache.kv_heads + w.head;
            const bool active = w.stop > w.begin && w.rows > w.first_row + t * kRows;      // this tile has rows, and they see something
            const bool has_tail = active && w.held > 0 && w.stop * kStepBlocks > w.full;
            const T* v_tail = reinterpret_cast<const T*>(p.cache.v_tail) + (pair * 2 + (w.full & 1)) * kKvBlock * D;
            const T* q_row = reinterpret_cast<const T*>(p.q) + w.b * p.q_batch + token * p.q_token + q_head * p.q_head;
            // What this row's weights, exp2(score) times the scale of the values, are relative to: the largest that it has seen (or a
            // little less).  FP16: `top` is that one's score and `level` the logarithm of its scale, and the sum is relative to it
            // too.  BF16, whose scales lie so far apart that weights which count for nothing can be those of the largest
            // probabilities: `top` is the largest score, which the sum is relative to, and `level` the weight relative to it.
            float top = kNone, level = 0.0f, sum = 0.0f, q_scale = p.scale;
            bool far = false;                            // a row of the warp has a maximum beyond kFar
            bool odd = false;                            // the tail's values have an infinity or NaN
            bool apart = false;                          // its numbers lie far apart: it is added behind the steps
            if (active) {
                // the row of queries: [half][row][128 bytes], dims in the order of the codes' bytes
                uint8_t* const to = shared + t * Shape::kQueryBytes;
                const uint32_t sign = p.negate ? 0x80008000u : 0u;
                uint32_t raw[D / 2];
#pragma unroll
                for (int i = 0; i < D / 2; i += 4) {                     // (all of it requested together)
                    raw[i] = raw[i + 1] = raw[i + 2] = raw[i + 3] = 0;
                    if (row < w.rows && p.q_wide) {
                        const uint4 four = *reinterpret_cast<const uint4*>(q_row + 2 * i);
                        raw[i] = four.x; raw[i + 1] = four.y; raw[i + 2] = four.z; raw[i + 3] = four.w;
                    } else if (row < w.rows) {
                        const uint16_t* h = reinterpret_cast<const uint16_t*>(q_row + 2 * i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) raw[i + e] = h[2 * e] | static_cast<uint32_t>(h[2 * e + 1]) << 16;
                    }
                }
                if constexpr (kBf16) {
                    // BF16 becomes FP16 by a power of two of the row's own: a number keeps all its bits unless it is 2^-26 of the
                    // row's largest or less
                    uint32_t largest = 0;
#pragma unroll
                    for (int i = 0; i < D / 2; ++i) largest = max(largest, max(raw[i] << 16 & 0x7fffffffu, raw[i] & 0x7fff0000u));
                    float back;
                    const float by = power_for(__uint_as_float(min(largest, 0x7f7f0000u)), back);
                    q_scale *= back;
#pragma unroll
                    for (int i = 0; i < D / 2; ++i) {
                        const float2 f = widen2<T>(raw[i]);
                        raw[i] = pack_half(f.x * by, f.y * by);
                    }
                }
#pragma unroll
                for (int i = 0; i < D / 2; i += 4) {
                    *reinterpret_cast<uint4*>(to + i / 32 * (kRows * 128) + swizzled(row_in_tile, i / 4 % 8)) =
                        make_uint4(prmt(raw[i], raw[i + 1], 0x5410) ^ sign, prmt(raw[i], raw[i + 1], 0x7632) ^ sign,
                                   prmt(raw[i + 2], raw[i + 3], 0x5410) ^ sign, prmt(raw[i + 2], raw[i + 3], 0x7632) ^ sign);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                arrive(bars.q_full[t]);
            }
            const int lowest = __reduce_min_sync(0xffffffffu, row < w.rows ? place : INT_MAX);
            for (int step = w.begin; active && step < w.stop; ++step, ++steps_done) {
                wait(bars.s_full[t], steps_done);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t score[kStepTokens];
                tmem_load128(score_at, score);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                arrive(bars.s_taken[t]);                 // the other tile's scores may come in their place
                // Of each block: a score's factor, not negative, and the logarithm of its values' scale, which goes into the exponent (and out
                // of the sum again; BF16: beside it).  Either may be NaN; a row that sees nothing of the block is kept out of that.
                const float4* const of_blocks = scales[(steps_of_all + step - w.begin) & 3];
                const unsigned notes = has_tail && step + 1 == w.stop ? tail_notes[(steps_of_all + step - w.begin) & 3][w.full % kStepBlocks] : 0u;
                odd = (notes & kOddValues) != 0;
                apart = kBf16 && (notes & kApart) != 0;
                const bool masked = (step + 1) * kStepTokens - 1 > lowest;
                // Tokens of the step up to this one are seen.  (The step with the block that is being filled goes on behind the last token,
                // so it is masked.)
                const int last = (apart ? min(place, w.full * kKvBlock - 1) : place) - step * kStepTokens;
                auto factors_of = [&](int block, float& by, float& value, float& inverse) {
                    const float4 of = of_blocks[block];
                    by = of.x * q_scale;
                    value = of.y;
                    inverse = of.z;
                    if (by == 0.0f) by = 0x1p-100f;
                    if (masked && block * kKvBlock > last) {
                        by = 1.0f;
                        value = 0.0f;
                    }
                    if (far) by = 1.0f;
                };
                if (masked) {
#pragma unroll
                    for (int i = 0; i < kStepTokens; ++i) {
                        if (token_of(i) > last) score[i] = 0xff800000u;
                    }
                }
                if (steps_done > 0) wait(bars.o_done[t], steps_done - 1);      // the probabilities before these have been used
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                // The largest weight is looked for in the first step, and where the weights relative to the last one have become too large
                // for FP16: then once more, relative to the new one.
                float step_sum = 0.0f;
                bool anew = step == w.begin || far;
#pragma unroll 1
                for (int attempt = 0; attempt < 2; ++attempt) {
                    if (anew) {
                        float largest[kStepBlocks], value[kStepBlocks];
                        far = false;
#pragma unroll
                        for (int block = 0; block < kStepBlocks; ++block) {
                            float by, inverse;
                            factors_of(block, by, value[block], inverse);
                            const float* x = reinterpret_cast<const float*>(score + block * 32);
                            float two[2] = {max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5])};
#pragma unroll
                            for (int i = 6; i < 30; i += 4) {
                                two[0] = max3(two[0], x[i], x[i + 1]);
                                two[1] = max3(two[1], x[i + 2], x[i + 3]);
                            }
                            largest[block] = max3(max3(two[0], x[30], x[31]), two[1], two[1]) * by;
                        }
                        float now = top, shrink = 1.0f;
                        if constexpr (kBf16) {
                            float most = kNone;
#pragma unroll
                            for (int block = 0; block < kStepBlocks; ++block) now = fmaxf(now, largest[block]);
                            const float before = top > kNone ? level + (top - now) : -INFINITY;
#pragma unroll
                            for (int block = 0; block < kStepBlocks; ++block) most = fmaxf(most, largest[block] - now + fmaxf(value[block], kLightest));
                            most = fmaxf(most, before);
                            if (top > kNone) {
                                shrink = exp2_fast(before - most);
                                sum *= exp2_fast(top - now);
                            }
                            level = now > kNone ? most : 0.0f;
                        } else {
                            float of_now = level;
#pragma unroll
                            for (int block = 0; block < kStepBlocks; ++block) {
                                if (largest[block] - now + (value[block] - of_now) > 0.0f) {
                                    now = largest[block];
                                    of_now = value[block];
                                }
                            }
                            if (top > kNone) shrink = exp2_fast(top - now + (level - of_now));
                            sum *= shrink;
                            level = of_now;
                        }
                        top = now;
                        if (step > w.begin) {
#pragma unroll 1
                            for (int d = 0; d < D; d += 32) {
                                uint32_t o[32];
                                tmem_load32(out_at + d, o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * shrink);
                                tmem_store16(out_at + d, o);
                                tmem_store16(out_at + d + 16, o + 16);
                            }
                        }
                        anew = false;
                        far = __any_sync(0xffffffffu, top > kNone && fabsf(top) > kFar);
                        if (far) {
                            // Product and difference in one rounding would leave the product's own, which for 10^12 is some 10^4: equal
                            // scores would be beyond or below their maximum.  (The maximum is that of this step, so that there is no
                            // second attempt.)
                            const float from = top > kNone ? top : 0.0f;
#pragma unroll
                            for (int block = 0; block < kStepBlocks; ++block) {
                                float by, value, inverse;
                                far = false;
                                factors_of(block, by, value, inverse);
                                far = true;
#pragma unroll
                                for (int i = 0; i < kKvBlock; ++i) {
                                    score[block * kKvBlock + i] = __float_as_uint(__fadd_rn(__fmul_rn(__uint_as_float(score[block * kKvBlock + i]), by), -from));
                                }
                            }
                        }
                    }
                    const float from = !far && top > kNone ? top : 0.0f;      // (a row that has seen nothing yet: all it meets is masked)
                    step_sum = 0.0f;
                    float largest_sum = 0.0f;
#pragma unroll
                    for (int block = 0; block < kStepBlocks; ++block) {
                        uint32_t packed[16];
                        float by, value, inverse;
                        factors_of(block, by, value, inverse);
                        const float rise = value - level + kHeadroom;
                        const float with = kBf16 ? -from : rise - from;
                        const float factor = kBf16 ? exp2_fast(rise > 126.0f ? 126.0f : rise) : inverse;      // (NaN stays)
                        // Where results are FP16 the sum is of the weights as they were rounded, so that what a row's large ones were
                        // off by goes out of its result: root mean square 1.4 times the result's own rounding at most, where it was up to
                        // 1.6 (2048 queries at 8192 take 12 us longer for it).  Not of a block whose values are so small that its weights
                        // run out of bits.
                        const bool as_rounded = !kBf16 && rise >= kHeadroom - 4.0f;
                        const uint64_t by2 = pair_of(by, by), with2 = pair_of(with, with), factor2 = pair_of(factor, factor);
                        uint64_t sums[2] = {0, 0};
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 x = both_of(fma2(pair_of(score[block * 32 + i], score[block * 32 + i + 1]), by2, with2));
                            float a = exp2_fast(x.x), b = exp2_fast(x.y);
                            if constexpr (kBf16) {
                                const float2 weights = both_of(mul2(pair_of(a, b), factor2));
                                packed[i / 2] = pack_half(weights.x, weights.y);
                            } else {
                                packed[i / 2] = pack_half(a, b);
                                if (as_rounded) {
                                    const float2 held = widen2<__half>(packed[i / 2]);
                                    a = held.x;
                                    b = held.y;
                                }
                            }
                            sums[i / 2 % 2] = add2(sums[i / 2 % 2], pair_of(a, b));
                        }
                        const float2 all = both_of(add2(sums[0], sums[1]));
                        const float block_sum = all.x + all.y;
                        largest_sum = fmaxf(largest_sum, kBf16 ? fmaxf(block_sum, block_sum * factor) : block_sum);
                        step_sum = kBf16 ? step_sum + block_sum : fmaf(block_sum, factor, step_sum);
                        tmem_store16(prob_at + block * 16, packed);
                    }
                    anew = __any_sync(0xffffffffu, largest_sum > kLargestSum);
                    if (!anew) break;
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");      // (these weights are written over)
                }
                sum += step_sum;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                arrive(bars.p_full[t]);
            }
            // the rows' results
            const bool to_part = w.piece >= 0;
            float* part = p.parts + (static_cast<size_t>(blockIdx.x) * kUnitRows + t * kRows + row_in_tile) * (D + 4);
            const bool write = to_part ? active : row < p.tokens * p.group;
            T* out = reinterpret_cast<T*>(p.out) + ((static_cast<size_t>(w.b) * p.tokens + token) * p.q_heads + q_head) * D;
            if (active) {
                wait(bars.o_done[t], steps_done - 1);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if constexpr (kBf16) {
                    if (apart) {
                        add_tail<D>(q_row, reinterpret_cast<const T*>(p.cache.k_tail) + (pair * 2 + (w.full & 1)) * kKvBlock * D, v_tail,
                                    row < w.rows ? min(w.held, place - w.full * kKvBlock + 1) : 0, p.negate ? -p.scale : p.scale, out_at, top, level, sum);
                    }
                }
            }
            const float unit = exp2_fast(level - kHeadroom), by = to_part ? unit : sum > 0.0f ? (kBf16 ? unit / sum : 1.0f / sum) : sum;
            const float shrink = kBf16 && to_part ? kShrink : 1.0f;
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
                uint32_t o[32];
                if (active) tmem_load32(out_at + d, o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = active && row < w.rows ? __float_as_uint(__uint_as_float(o[i]) * shrink * by) : 0u;
                if (odd) {                               // infinities and NaN of the tail, which were kept out of the products
                    for (int i = 0; i < w.held; ++i) {
                        if (w.full * kKvBlock + i > place) break;
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float v = widen<T>(v_tail[i * D + d + e]);
                            if (!(fabsf(v) <= 3.4028235e38f)) o[e] = __float_as_uint(__uint_as_float(o[e]) + v);
                        }
                    }
                }
                if (!write) continue;
                if (to_part) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(part + d + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        auto two = [&](int j) { return narrow2<T>(__uint_as_float(o[i + j]), __uint_as_float(o[i + j + 1])); };
                        *reinterpret_cast<uint4*>(out + d + i) = make_uint4(two(0), two(2), two(4), two(6));
                    }
                }
            }
            if (write && to_part) *reinterpret_cast<float2*>(part + D) = make_float2(top, kBf16 ? sum : sum * unit);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");      // (the next work's first arrival lets O be overwritten)
        }
    } else if (warp < kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PrefillRegisters<T, D>::kDequant));
        // ---------------------------------------------------------------- operands: one block of a step a warp
        const int mine = warp - kSoftmaxWarps, g = lane >> 2, c = lane & 3;
        constexpr int kVectors = D / 16;                 // 16-byte pieces of a block's keys, and values, for a lane
        constexpr int kBlockBytes = kKvBlock * D;
        uint8_t* const codes = shared + Shape::kCodesAt + mine * 2 * kBlockBytes;      // of a block's keys, and of its values
        // Asks for a block's codes (which: 0 keys, 1 values), behind all lanes' reads of those before.
        auto ask = [&](int which, int pair, int block) {
            const unsigned bar = smem_u32(&bars.codes[mine][which]);
            mbar_arrive_expect_tx(bar, kBlockBytes);
            bulk_load(smem_u32(codes + which * kBlockBytes), (which == 0 ? p.cache.k_codes : p.cache.v_codes) + (static_cast<size_t>(pair) * p.cache.blocks + block) * kBlockBytes,
                      kBlockBytes, bar);
        };
        int steps = 0, read = 0;                         // steps of all, this CTA's works one after the other; blocks of codes
        Work w;
        bool asked = false;                              // whether the next step's codes were asked for
        // of the block that is being filled, where it is this warp's
        unsigned notes = 0;
        float k_by = 1.0f, v_by = 1.0f;                  // what its numbers are multiplied with
        bool v_none = false;                             // all zeros: it counts for no more than a full block of zeros
        for (int n = 0; work_of(p, n, w); ++n) {
            if (w.stop <= w.begin) continue;
            const int pair = w.b * p.cache.kv_heads + w.head;
            // the step behind this work's last
            Work after;
            int follower = n + 1;
            bool follows = work_of(p, follower, after);
            while (follows && after.stop <= after.begin) follows = work_of(p, ++follower, after);
            const int after_pair = after.b * p.cache.kv_heads + after.head;
            const int after_block = after.begin * kStepBlocks + mine;
            const bool after_coded = follows && after_block < after.full;
            if (!asked && w.begin * kStepBlocks + mine < w.full && lane == 0) {
                ask(0, pair, w.begin * kStepBlocks + mine);
                ask(1, pair, w.begin * kStepBlocks + mine);
            }
            if (w.held > 0 && w.full % kStepBlocks == mine && w.full / kStepBlocks >= w.begin && w.full / kStepBlocks < w.stop) {
                // What the numbers of the block that is being filled are multiplied with to become FP16, and what is to be noted.  FP16
                // keys stay as they are; other numbers are brought to the size of codes, so that weights keep as many bits beside small
                // ones.  They keep their bits down to 2^-23 of the block's largest (BF16 2^-26), and are off by 2^-34 of it below that.
                // (As codes they count as zero below 2^-8 of it; with more room for them weights would have less.)  BF16 reaches further: where that is more than a 2^-22nd of eight keys' largest, or a 2^-17th
                // of eight values', which takes one far out that a query may not even see, the block is left to add_tail().
                const size_t tail = (static_cast<size_t>(pair) * 2 + (w.full & 1)) * kKvBlock * D;
                bool odd, unused;
                float inverse;
                const float2 values = range_of(reinterpret_cast<const T*>(p.cache.v_tail) + tail, w.held * D, lane, odd);
                notes = odd ? kOddValues : 0u;
                v_by = power_for(values.x, inverse);
                v_none = values.x == 0.0f;
                if constexpr (kBf16) {
                    const float2 keys = range_of(reinterpret_cast<const T*>(p.cache.k_tail) + tail, w.held * D, lane, unused);
                    k_by = power_for(keys.x, inverse);
                    if (values.y < values.x * 0x1p-17f || keys.y < keys.x * 0x1p-12f) notes |= kApart;
                }
            }
#pragma unroll 1
            for (int step = w.begin; step < w.stop; ++step, ++steps) {
                const int block = step * kStepBlocks + mine, stage = steps & 1;
                const bool coded = block < w.full, tail = block == w.full && w.held > 0;
                const bool last = step + 1 == w.stop;
                asked = last ? after_coded : block + kStepBlocks < w.full;
                const int next_pair = last ? after_pair : pair;
                const int next_block = last ? after_block : block + kStepBlocks;
                const T* k_tail = reinterpret_cast<const T*>(p.cache.k_tail) + (static_cast<size_t>(pair) * 2 + (block & 1)) * kKvBlock * D;
                const T* v_tail = reinterpret_cast<const T*>(p.cache.v_tail) + (static_cast<size_t>(pair) * 2 + (block & 1)) * kKvBlock * D;
                float k_scale = 0.0f, v_scale = 0.0f;
                if (coded) {
                    k_scale = p.cache.k_scales[static_cast<size_t>(pair) * p.cache.blocks + block];
                    v_scale = p.cache.v_scales[static_cast<size_t>(pair) * p.cache.blocks + block];
                } else if (tail) {
                    k_scale = inverse_power(k_by);
                    v_scale = v_none ? 0.0f : inverse_power(v_by);
                    if (lane == 0) tail_notes[steps & 3][mine] = static_cast<uint8_t>(notes);
                }
                auto to_half = [&](uint32_t word, float by) {
                    const float2 f = widen2<T>(word);
                    return pack_half(f.x * by, f.y * by);
                };
                auto key_to_half = [&](uint32_t word) { return kBf16 ? to_half(word, k_by) : word; };
                // keys: row of a token, in the order of the columns (token_of)
                if (coded) wait(bars.codes[mine][0], read);
                if (steps >= 2) wait(bars.k_empty[stage], steps / 2 - 1);
                {
                    uint8_t* const to = shared + Shape::kKeysAt + stage * Shape::kKeyBytes;
                    auto store = [&](int i, const uint32_t (&words)[8]) {      // piece i: [group of 16 tokens][parity][half of the dims]
                        const int half = i % kHalves, parity = i / kHalves % 2, group = i / kHalves / 2;
                        const int row = mine * 32 + g / 2 * 8 + group * 4 + g % 2 + parity * 2;
                        uint8_t* const at = to + half * (kStepTokens * 128);
                        *reinterpret_cast<uint4*>(at + swizzled(row, 2 * c)) = make_uint4(words[0], words[1], words[2], words[3]);
                        *reinterpret_cast<uint4*>(at + swizzled(row, 2 * c + 1)) = make_uint4(words[4], words[5], words[6], words[7]);
                    };
                    if (coded) {
#pragma unroll 4                 // (all eight: 7 us more)
                        for (int i = 0; i < kVectors; ++i) {
                            const uint4 four = *reinterpret_cast<const uint4*>(codes + i * 512 + lane * 16);
                            uint32_t words[8];
                            codes_to_half(four.x, words[0], words[1]);
                            codes_to_half(four.y, words[2], words[3]);
                            codes_to_half(four.z, words[4], words[5]);
                            codes_to_half(four.w, words[6], words[7]);
                            store(i, words);
                        }
                    } else {
#pragma unroll 1
                        for (int i = 0; i < kVectors; ++i) {
                            uint32_t words[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                            const int token = i / kHalves / 2 * 16 + g * 2 + i / kHalves % 2;
                            if (tail && token < w.held) {
                                const uint32_t* raw = reinterpret_cast<const uint32_t*>(k_tail + token * D + i % kHalves * 64 + c * 16);
#pragma unroll
                                for (int e = 0; e < 8; e += 2) {
                                    const uint32_t lo = key_to_half(raw[e]), hi = key_to_half(raw[e + 1]);
                                    words[e] = prmt(lo, hi, 0x5410);
                                    words[e + 1] = prmt(lo, hi, 0x7632);
                                }
                            }
                            store(i, words);
                        }
                    }
                }
                if (lane == 0) {
                    const float v_log = !kBf16 && v_scale < 0x1p-40f ? kLightestHalf : __log2f(v_scale);
                    scales[steps & 3][mine] = make_float4(k_scale, v_log, v_scale != v_scale ? 0.0f : exp2_fast(-v_log), 0.0f);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                arrive(bars.k_full[stage]);
                if (asked && healthy && lane == 0) ask(0, next_pair, next_block);
                // values: row of a dim, tokens in the columns' order
                if (coded) wait(bars.codes[mine][1], read++);
                if (steps >= 2) wait(bars.v_empty[stage], steps / 2 - 1);
                uint8_t* const to = shared + Shape::kValuesAt + stage * Shape::kValueBytes + mine / 2 * (D * 128);
                if (coded || !tail) {
#pragma unroll 4
                    for (int i = 0; i < kVectors; ++i) {         // sixteen dims: [half of them][group of 16 tokens]
                        uint4 four = make_uint4(0u, 0u, 0u, 0u);
                        if (coded) four = *reinterpret_cast<const uint4*>(codes + kBlockBytes + i * 512 + lane * 16);
                        const uint32_t words[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            uint4 eight;
                            codes_to_half(words[2 * half], eight.x, eight.y);
                            codes_to_half(words[2 * half + 1], eight.z, eight.w);
                            *reinterpret_cast<uint4*>(to + swizzled(i * 16 + half * 8 + g, mine % 2 * 4 + c)) = eight;
                        }
                    }
                } else {
                    for (int i = lane; i < 8 * (D / 8); i += 32) {      // eight dims of four tokens
                        const int quad = i / (D / 8), d0 = i % (D / 8) * 8;
                        uint32_t raw[4][4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            uint4 four = make_uint4(0u, 0u, 0u, 0u);
                            if (quad * 4 + e < w.held) four = *reinterpret_cast<const uint4*>(v_tail + (quad * 4 + e) * D + d0);
                            raw[e][0] = four.x; raw[e][1] = four.y; raw[e][2] = four.z; raw[e][3] = four.w;
#pragma unroll
                            for (int f = 0; f < 4; ++f) {
                                const float2 v = widen2<T>(raw[e][f]);
                                if (!(fabsf(v.x) <= 3.4028235e38f)) raw[e][f] &= 0xffff0000u;
                                if (!(fabsf(v.y) <= 3.4028235e38f)) raw[e][f] &= 0x0000ffffu;
                                raw[e][f] = to_half(raw[e][f], v_by);
                            }
                        }
#pragma unroll
                        for (int f = 0; f < 4; ++f) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const unsigned pick = h == 0 ? 0x5410u : 0x7632u;
                                const int chunk = mine % 2 * 4 + quad % 4;
                                *reinterpret_cast<uint2*>(to + swizzled(d0 + 2 * f + h, chunk) + quad / 4 * 8) =
                                    make_uint2(prmt(raw[0][f], raw[2][f], pick), prmt(raw[1][f], raw[3][f], pick));
                            }
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                arrive(bars.v_full[stage]);
                if (asked && healthy && lane == 0) ask(1, next_pair, next_block);
            }
        }
        if (!healthy && lane == 0) {                     // wait, within limits, for copies that may still be on their way
            for (int which = 0; which < 2; ++which) mbar_wait<false, true>(smem_u32(&bars.codes[mine][which]), read & 1, kKvGaveUp, p.cache.status);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PrefillRegisters<T, D>::kIssuer));
        // ---------------------------------------------------------------- MMAs
        constexpr uint32_t kCommon = (1u << 4) | (static_cast<uint32_t>(kRows >> 4) << 24);      // FP32 sums of FP16, 128 rows, K-major
        constexpr uint32_t kScoreDesc = kCommon | (static_cast<uint32_t>(kStepTokens >> 3) << 17);
        constexpr uint32_t kOutputDesc = kCommon | (static_cast<uint32_t>(D >> 3) << 17);
        const bool chosen = elect_one();
        int steps = 0, works[2] = {0, 0};                // steps of all, up to this work; works of each tile
        int issued[2] = {0, 0}, used[2] = {0, 0};        // of each tile: scores, outputs
        int holder = -1;                                 // whose scores lie in TMEM
        Work w;
        for (int n = 0; warp == kMmaWarp && work_of(p, n, w); ++n) {
            if (w.stop <= w.begin || w.rows <= w.first_row) continue;
            const int tiles = w.rows > w.first_row + kRows ? 2 : 1, count = w.stop - w.begin;
            auto scores = [&](int t, int step) {
                if (step >= count) return;
                const int stage = (steps + step) & 1;
                if (t == 0) wait(bars.k_full[stage], (steps + step) / 2);
                if (holder >= 0) wait(bars.s_taken[holder], issued[holder] - 1);
                holder = t;
                ++issued[t];
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (chosen && healthy) {
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const uint64_t a = operand_desc(smem_u32(shared) + t * Shape::kQueryBytes + i / 4 * (kRows * 128) + i % 4 * 32);
                        const uint64_t b = operand_desc(smem_u32(shared) + Shape::kKeysAt + stage * Shape::kKeyBytes + i / 4 * (kStepTokens * 128) + i % 4 * 32);
                        umma_f16_shared(tmem, a, b, kScoreDesc, i > 0 ? 1u : 0u);
                    }
                    umma_commit(smem_u32(&bars.s_full[t]));
                    if (t == tiles - 1) umma_commit(smem_u32(&bars.k_empty[stage]));
                }
                __syncwarp();
            };
            auto outputs = [&](int t, int step) {
                const int stage = (steps + step) & 1;
                if (t == 0) wait(bars.v_full[stage], (steps + step) / 2);
                wait(bars.p_full[t], used[t]++);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (chosen && healthy) {
#pragma unroll
                    for (int i = 0; i < kStepTokens / 16; ++i) {
                        const uint64_t b = operand_desc(smem_u32(shared) + Shape::kValuesAt + stage * Shape::kValueBytes + i / 4 * (D * 128) + i % 4 * 32);
                        umma_f16_tmem_a(tmem + kOutputs + t * 128, tmem + kProbabilities + t * 64 + i * 8, b, kOutputDesc, step > 0 || i > 0 ? 1u : 0u);
                    }
                    umma_commit(smem_u32(&bars.o_done[t]));
                    if (t == tiles - 1) umma_commit(smem_u32(&bars.v_empty[stage]));
                }
                __syncwarp();
            };
            // A tile takes its scores as soon as it is done with the last; then the other's, which it will want half a round later, are
            // formed in their place.
            for (int t = 0; t < tiles; ++t) {
                wait(bars.q_full[t], works[t]++);
                scores(t, 0);
            }
            scores(0, 1);
            for (int step = 0; step < count; ++step) {
                outputs(0, step);
                if (tiles == 2) {
                    scores(1, step + 1);
                    outputs(1, step);
                }
                scores(0, step + 2);
            }
            steps += count;
        }
        // nothing may be in flight when TMEM goes
        for (int t = 0; t < 2; ++t) {
            if (used[t] > 0) mbar_wait<false, true>(smem_u32(&bars.o_done[t]), (used[t] - 1) & 1, kKvGaveUp, p.cache.status);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == kMmaWarp) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Adds up the pieces of the units that were cut; a warp for a row, BATCH pieces requested together: two where there are no more (with eight
// 2048 queries at 8192 take 12 us more), else eight (40 rows of one sequence of 8000 22 us, one by one 25).
template <typename T, int D, int BATCH>
__global__ void __launch_bounds__(128)
kv_pieces_kernel(const PrefillParams p) {
    pdl_wait_for_upstream();
    pdl_release_downstream();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int unit = blockIdx.x / (kUnitRows / 4), in_unit = blockIdx.x % (kUnitRows / 4) * 4 + warp;
    const Work first = unit_of(p, p.whole + unit, -1);
    const int row = first.first_row + in_unit;
    if (row >= p.tokens * p.group) return;
    constexpr int kDims = D / 32;
    float top = kNone, weight = 0.0f, acc[kDims];
#pragma unroll
    for (int d = 0; d < kDims; ++d) acc[d] = 0.0f;
    if (row < first.rows) {
        for (int begin = 0; begin < p.pieces; begin += BATCH) {
            float2 state[BATCH], numbers[BATCH][kDims / 2];
            float best = top;
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const int piece = begin + e;
                const bool some = piece < p.pieces && static_cast<long long>(first.stop) * piece / p.pieces <
                                                          static_cast<long long>(first.stop) * (piece + 1) / p.pieces;
                const float* part = p.parts + (static_cast<size_t>(unit * p.pieces + piece) * kUnitRows + in_unit) * (D + 4);
                state[e] = some ? *reinterpret_cast<const float2*>(part + D) : make_float2(kNone, 0.0f);
#pragma unroll
                for (int d = 0; d < kDims / 2; ++d) {
                    numbers[e][d] = some ? reinterpret_cast<const float2*>(part + lane * kDims)[d] : make_float2(0.0f, 0.0f);
                }
            }
#pragma unroll
            for (int e = 0; e < BATCH; ++e) best = fmaxf(best, state[e].x);
            const float mine = exp2_fast(top - best);
            top = best;
            weight *= mine;
#pragma unroll
            for (int d = 0; d < kDims; ++d) acc[d] *= mine;
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const float theirs = exp2_fast(state[e].x - best);
                weight = fmaf(state[e].y, theirs, weight);
#pragma unroll
                for (int d = 0; d < kDims / 2; ++d) {
                    acc[2 * d] = fmaf(numbers[e][d].x, theirs, acc[2 * d]);
                    acc[2 * d + 1] = fmaf(numbers[e][d].y, theirs, acc[2 * d + 1]);
                }
            }
        }
    }
    constexpr float kHeld = std::is_same<T, __nv_bfloat16>::value ? kShrink : 1.0f;      // what the sums are held times
    const float by = weight > 0.0f ? 1.0f / kHeld / weight : weight;
    const int token = by_group(p, row), q_head = first.head * p.group + row - token * p.group;
    T* to = reinterpret_cast<T*>(p.out) + ((static_cast<size_t>(first.b) * p.tokens + token) * p.q_heads + q_head) * D + lane * kDims;
#pragma unroll
    for (int d = 0; d < kDims; d += 2) *reinterpret_cast<uint32_t*>(to + d) = narrow2<T>(acc[d] * by, acc[d + 1] * by);
}

struct DeviceState {
    int sms = 0;
};

template <typename T, int D>
int allow_shared() {
    return cudaFuncSetAttribute(kv_prefill_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(PrefillShape<D>::kSharedBytes)) == cudaSuccess
               ? 0
               : W4A16_ERR_LAUNCH;
}

int device_state(const DeviceState** state) {
    static PerDevice<DeviceState> devices;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= kMaxDevices) return W4A16_ERR_LAUNCH;
    return devices.get(device, [&](DeviceState& fresh) -> int {
        if (cudaDeviceGetAttribute(&fresh.sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return W4A16_ERR_LAUNCH;
        const int allowed = allow_shared<__half, 64>() | allow_shared<__half, 128>() | allow_shared<__nv_bfloat16, 64>() |
                            allow_shared<__nv_bfloat16, 128>();
        return allowed != 0 ? W4A16_ERR_LAUNCH : 0;
    }, state);
}

struct Split {
    int64_t row_tiles, units, whole, pieces, grid;
};

Split split_of(const w4a16_kv8_cache& cache, int q_heads, int64_t tokens, int sms) {
    Split s;
    const int64_t rows = tokens * (q_heads / cache.kv_heads);
    s.row_tiles = (rows + kUnitRows - 1) / kUnitRows;
    s.units = s.row_tiles * cache.batch * cache.kv_heads;
    s.whole = s.units / sms * sms;
    const int64_t rest = s.units - s.whole;
    // (a piece is worth two steps or more)
    const int64_t steps = (cache.max_len + kStepTokens - 1) / kStepTokens;
    s.pieces = rest > 0 ? std::max<int64_t>(1, std::min<int64_t>(sms / rest, steps / 2)) : 1;
    if (s.pieces == 1) s.whole = s.units;            // (nothing to be added up: 128 units of D = 128 take 14 us less)
    s.grid = s.whole > 0 ? std::min<int64_t>(s.units, sms) : rest * s.pieces;
    return s;
}

}  // namespace

size_t kv_prefill_workspace_bytes(const w4a16_kv8_cache& cache, int q_heads, int64_t tokens) {
    const DeviceState* state = nullptr;
    const Split s = split_of(cache, q_heads, tokens, device_state(&state) == 0 ? state->sms : 148);
    return static_cast<size_t>((s.units - s.whole) * s.pieces) * kUnitRows * (cache.head_dim + 4) * sizeof(float);
}

int launch_kv_prefill(const w4a16_kv8_cache& cache, const w4a16_rows& q, void* out, int q_heads, int64_t tokens, const long long* lengths,
                      const long long* counts, float softmax_scale, void* workspace, size_t workspace_bytes, bool programmatic,
                      cudaStream_t stream) {
    const DeviceState* state = nullptr;
    if (const int status = device_state(&state); status != 0) return status;
    const Split s = split_of(cache, q_heads, tokens, state->sms);
    const int64_t group = q_heads / cache.kv_heads;
    if (s.units > INT32_MAX / 2 || tokens * group >= 1 << 24) return W4A16_ERR_TOO_LARGE;
    const int64_t rest = s.units - s.whole;
    if (rest > 0 && (workspace == nullptr || workspace_bytes < kv_prefill_workspace_bytes(cache, q_heads, tokens))) return W4A16_ERR_WORKSPACE;
    PrefillParams p{};
    p.cache = kv_view(cache);
    p.q = static_cast<const char*>(q.data);
    p.q_batch = q.batch_stride;
    p.q_token = q.token_stride;
    p.q_head = q.head_stride;
    p.q_wide = reinterpret_cast<uintptr_t>(q.data) % 16 == 0 && q.batch_stride % 8 == 0 && q.token_stride % 8 == 0 && q.head_stride % 8 == 0;
    p.out = static_cast<char*>(out);
    p.tokens = static_cast<int>(tokens);
    p.q_heads = q_heads;
    p.group = static_cast<int>(group);
    p.per_group = 1.0f / static_cast<float>(group);
    p.row_tiles = static_cast<int>(s.row_tiles);
    p.lengths = lengths;
    p.counts = counts;
    p.scale = (softmax_scale < 0.0f ? -softmax_scale : softmax_scale) * kLog2e;
    p.negate = softmax_scale < 0.0f;
    p.parts = static_cast<float*>(workspace);
    p.units = static_cast<int>(s.units);
    p.whole = static_cast<int>(s.whole);
    p.pieces = static_cast<int>(s.pieces);
    const bool bf16 = cache.type == W4A16_TYPE_BF16;
    auto run = [&](auto type, auto dims) {
        using T = decltype(type);
        constexpr int kD = decltype(dims)::value;
        const int status = kv_launch(kv_prefill_kernel<T, kD>, dim3(static_cast<unsigned>(s.grid)), dim3(kPrefillThreads),
                                     PrefillShape<kD>::kSharedBytes, programmatic, stream, p);
        if (status != W4A16_OK || rest == 0) return status;
        return kv_launch(s.pieces <= 2 ? kv_pieces_kernel<T, kD, 2> : kv_pieces_kernel<T, kD, 8>, dim3(static_cast<unsigned>(rest * (kUnitRows / 4))), dim3(128), 0, true, stream, p);
    };
    using Small = std::integral_constant<int, 64>;
    using Large = std::integral_constant<int, 128>;
    if (cache.head_dim == 64) return bf16 ? run(__nv_bfloat16(), Small{}) : run(__half(), Small{});
    return bf16 ? run(__nv_bfloat16(), Large{}) : run(__half(), Large{});
}

}  // namespace w4a16
