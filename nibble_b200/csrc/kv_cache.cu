// Rotary positions, and the 8-bit key/value cache written and read back (its format: kv_cache.cuh).
//
// Rotary positions.  Pair j of a head, at position p, is turned by the angle p * inv_freq[j]:
//     (a, b) -> (a cos - b sin, b cos + a sin),      cos and sin times `scale`
// with pairs (2j, 2j + 1) or (j, j + rotary_dim / 2), numbers from rotary_dim on left as they are.  Ways of stretching a context
// (interpolated, by parts, with a temperature) change inv_freq and scale and nothing here.  At a position of 10^6 an FP32 angle
// is off by up to 0.03, so the angle is formed and reduced to a turn in FP64; from there on FP32, rounded once.
//
// Bounds: all three are made of one pass over their data, HBM for prompts and launch latency for a token.  Measured, of 6.5 TB/s
// that a copy reaches: 4096 tokens of 72 heads of 128 turned 28.7 us (5.3 TB/s); 2 x 8191 tokens of 8 heads of 128 written 23 us (4.3);
// 32768 tokens read back 36 us (5.6); one token turned or read back 2.3 us, written 2.2, turned and written 3.0 with its queries.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "kv_cache.cuh"
#include "unpack.cuh"

namespace w4a16 {
namespace {

// ------------------------------------------------------------------ rotary positions

struct RowView {
    const char* data;                            // 16-bit numbers; strides in numbers
    long long batch, token, head;
};

template <typename T>
__device__ __forceinline__ const T* row_of(const RowView& v, long long b, long long i, int h) {
    return reinterpret_cast<const T*>(v.data) + b * v.batch + i * v.token + h * v.head;
}

__device__ __forceinline__ double turns_of(float inv_freq) { return static_cast<double>(inv_freq) * 0.15915494309189533577; }      // 1 / (2 pi)
__device__ __forceinline__ float2 rotary_factors(long long position, double turns_each, float scale) {
    double turns = static_cast<double>(position) * turns_each;
    turns -= rint(turns);
    float s, c;
    sincospif(static_cast<float>(2.0 * turns), &s, &c);
    return make_float2(c * scale, s * scale);
}

// The two numbers of a pair; the same instructions wherever a pair is turned, so that all ways give the same bits.
__device__ __forceinline__ float rotary_first(float a, float b, float2 f) { return __fmaf_rn(a, f.x, -__fmul_rn(b, f.y)); }
__device__ __forceinline__ float rotary_second(float a, float b, float2 f) { return __fmaf_rn(b, f.x, __fmul_rn(a, f.y)); }

template <typename T>
__device__ __forceinline__ void turn8_halves(uint4& lo, uint4& hi, const float2* f) {      // lo[i], hi[i] are pair i
    uint32_t* a = reinterpret_cast<uint32_t*>(&lo);
    uint32_t* b = reinterpret_cast<uint32_t*>(&hi);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = widen2<T>(a[i]), y = widen2<T>(b[i]);
        const float2 f0 = f[2 * i], f1 = f[2 * i + 1];
        a[i] = narrow2<T>(rotary_first(x.x, y.x, f0), rotary_first(x.y, y.y, f1));
        b[i] = narrow2<T>(rotary_second(x.x, y.x, f0), rotary_second(x.y, y.y, f1));
    }
}
template <typename T>
__device__ __forceinline__ void turn8_pairs(uint4& v, const float2* f) {
    uint32_t* a = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = widen2<T>(a[i]);
        a[i] = narrow2<T>(rotary_first(x.x, x.y, f[i]), rotary_second(x.x, x.y, f[i]));
    }
}

struct RotaryRows {
    RowView in, out;
    int head_dim, rotary_dim;
    bool interleaved;
    bool aligned;                                // rows can be read and written 16 bytes at a time,
    bool wide;                                   // and so can either half of what is turned
    bool in_place;                               // what is not turned is there already
    int pieces, piece_bits;                      // of a head, eight numbers or eight pairs (wide) each, and bits that number them
};

// Turns `heads` heads from `first_head` on of `tokens` tokens; table[token * rotary_dim / 2 + pair] holds the factors.
//
// Wide rows: a thread keeps to one piece of a head and takes heads (and tokens, while heads are few) in turn, so that nothing is
// divided out on the way and a token's factors are read once.  (With the pieces of a tile numbered through, 4096 tokens of 72
// heads of 128 took 77 us, most of it divisions.)
template <typename T, bool INTERLEAVED>
__device__ __forceinline__ void rotate_rows_wide(const RotaryRows& r, const float2* table, long long b, long long first_token, int tokens,
                                                 int first_head, int heads) {
    constexpr int kFactors = INTERLEAVED ? 4 : 8;
    constexpr int kBatch = INTERLEAVED ? 4 : 2;  // heads requested together
    const int half = r.rotary_dim / 2, turned = half / kFactors;
    const int piece = threadIdx.x & ((1 << r.piece_bits) - 1), row = threadIdx.x >> r.piece_bits, rows = blockDim.x >> r.piece_bits;
    if (piece >= r.pieces) return;
    const bool plain = piece >= turned;          // left as it is
    const int d = plain ? r.rotary_dim + (piece - turned) * 8 : piece * 8;
    int abreast = 1;                             // heads that a pass takes side by side
    while (abreast < heads && abreast < rows) abreast *= 2;
    const int token_step = rows / abreast, first = row & (abreast - 1);
    const long long in_step = abreast * r.in.head, out_step = abreast * r.out.head;
    for (int token = row / abreast; token < tokens; token += token_step) {
        const float2* factors = table + token * half + piece * kFactors;
        const T* in = row_of<T>(r.in, b, first_token + token, first_head + first) + d;
        T* out = const_cast<T*>(row_of<T>(r.out, b, first_token + token, first_head + first)) + d;
        float2 f[kFactors];
#pragma unroll
        for (int i = 0; i < kFactors; i += 2) {
            if (plain) break;
            const float4 two = *reinterpret_cast<const float4*>(factors + i);      // (a piece's factors begin at an even one)
            f[i] = make_float2(two.x, two.y);
            f[i + 1] = make_float2(two.z, two.w);
        }
        for (int head = first; head < heads; head += kBatch * abreast, in += kBatch * in_step, out += kBatch * out_step) {
            uint4 lo[kBatch], hi[kBatch];
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                if (head + e * abreast >= heads) break;
                lo[e] = *reinterpret_cast<const uint4*>(in + e * in_step);
                if (!INTERLEAVED && !plain) hi[e] = *reinterpret_cast<const uint4*>(in + e * in_step + half);
            }
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                if (head + e * abreast >= heads) break;
                if (!plain) {
                    if constexpr (INTERLEAVED) {
                        turn8_pairs<T>(lo[e], f);
                    } else {
                        turn8_halves<T>(lo[e], hi[e], f);
                        *reinterpret_cast<uint4*>(out + e * out_step + half) = hi[e];
                    }
                }
                *reinterpret_cast<uint4*>(out + e * out_step) = lo[e];
            }
        }
    }
}

enum class Pairs { kInterleaved, kHalvesOfWords, kHalves };      // neighbours; half a head apart, an even or an odd number of places

// The same where halves begin anywhere: a thread turns eight numbers that lie together, and reads each one's partner for itself.  The
// pieces of a head are lanes of one warp, which has read all of them before it writes one (rows may be turned in place).  (4096 tokens
// of 72 heads of 128: 90 numbers turned 49 us, 92 37, 90 in neighbouring pairs 35; number by number 171.)
template <typename T, Pairs PAIRS>
__device__ __forceinline__ void rotate_rows_aligned(const RotaryRows& r, const float2* table, long long b, long long first_token, int tokens,
                                                    int first_head, int heads) {
    constexpr int kBatch = 2;                    // heads requested together
    const int half = r.rotary_dim / 2;
    const int piece = threadIdx.x & ((1 << r.piece_bits) - 1), row = threadIdx.x >> r.piece_bits, rows = blockDim.x >> r.piece_bits;
    const int d = piece * 8;
    int abreast = 1;                             // heads that a pass takes side by side
    while (abreast < heads && abreast < rows) abreast *= 2;
    const int first = row & (abreast - 1);
    for (int token_base = 0; token_base < tokens; token_base += rows / abreast) {
        const int token = token_base + row / abreast;
        const bool there = piece < r.pieces && token < tokens;
        float2 f[8];                             // of each number: what it is multiplied with, and its partner
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int pair = PAIRS == Pairs::kInterleaved ? (d + i) / 2 : d + i < half ? d + i : d + i - half;
            f[i] = there && d + i < r.rotary_dim ? table[token * half + pair] : make_float2(1.0f, 0.0f);
            if (PAIRS == Pairs::kInterleaved ? i % 2 == 0 : d + i < half) f[i].y = -f[i].y;
        }
        const T* const in = row_of<T>(r.in, b, first_token + token, first_head);
        unsigned place[8];                       // of its partner; numbers that are not turned are read themselves
#pragma unroll
        for (int i = 0; i < 8; ++i) place[i] = d + i < half ? d + i + half : d + i < r.rotary_dim ? d + i - half : d + i;
        T* const out = const_cast<T*>(row_of<T>(r.out, b, first_token + token, first_head)) + d;
        for (int head_base = 0; head_base < heads; head_base += kBatch * abreast) {
            uint4 own[kBatch];
            uint32_t partner[kBatch][4];
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                const int head = head_base + e * abreast + first;
                if (!there || head >= heads) break;
                const T* from = in + head * r.in.head;
                own[e] = *reinterpret_cast<const uint4*>(from + d);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    if (PAIRS == Pairs::kInterleaved) {
                        partner[e][i / 2] = __byte_perm((&own[e].x)[i / 2], 0, 0x1032);
                        continue;
                    }
                    if (PAIRS == Pairs::kHalvesOfWords) {
                        partner[e][i / 2] = *reinterpret_cast<const uint32_t*>(from + place[i]);
                    } else {
                        const uint16_t* numbers = reinterpret_cast<const uint16_t*>(from);
                        partner[e][i / 2] = numbers[place[i]] | static_cast<uint32_t>(numbers[place[i + 1]]) << 16;
                    }
                }
            }
            if (r.in_place) __syncwarp();
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                const int head = head_base + e * abreast + first;
                if (!there || head >= heads) break;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    uint32_t& word = (&own[e].x)[i / 2];
                    const float2 x = widen2<T>(word), y = widen2<T>(partner[e][i / 2]);
                    // (rotary_first and rotary_second, the sign being in the factor)
                    const uint32_t turned = narrow2<T>(__fmaf_rn(x.x, f[i].x, __fmul_rn(y.x, f[i].y)),
                                                       __fmaf_rn(x.y, f[i + 1].x, __fmul_rn(y.y, f[i + 1].y)));
                    if (d + i < r.rotary_dim) word = turned;      // (an even number of them)
                }
                *reinterpret_cast<uint4*>(out + head * r.out.head) = own[e];
            }
        }
    }
}

template <typename T>
__device__ void rotate_rows(const RotaryRows& r, const float2* table, long long b, long long first_token, int tokens, int first_head,
                            int heads) {
    if (r.wide) {
        if (r.interleaved) rotate_rows_wide<T, true>(r, table, b, first_token, tokens, first_head, heads);
        else rotate_rows_wide<T, false>(r, table, b, first_token, tokens, first_head, heads);
        return;
    }
    if (r.aligned) {
        if (r.interleaved) rotate_rows_aligned<T, Pairs::kInterleaved>(r, table, b, first_token, tokens, first_head, heads);
        else if (r.rotary_dim % 4 == 0) rotate_rows_aligned<T, Pairs::kHalvesOfWords>(r, table, b, first_token, tokens, first_head, heads);
        else rotate_rows_aligned<T, Pairs::kHalves>(r, table, b, first_token, tokens, first_head, heads);
        return;
    }
    const int half = r.rotary_dim / 2, pieces = half + (r.in_place ? 0 : r.head_dim - r.rotary_dim);      // pairs, and the rest
    const int total = tokens * heads * pieces;
    for (int at = threadIdx.x; at < total; at += blockDim.x) {
        const int row = at / pieces, piece = at - row * pieces, token = row / heads, head = row - token * heads;
        const T* from = row_of<T>(r.in, b, first_token + token, first_head + head);
        T* to = const_cast<T*>(row_of<T>(r.out, b, first_token + token, first_head + head));
        if (piece >= half) {
            to[half + piece] = from[half + piece];
            continue;
        }
        const int da = r.interleaved ? 2 * piece : piece, db = r.interleaved ? da + 1 : da + half;
        const float x = widen<T>(from[da]), y = widen<T>(from[db]);
        const float2 f = table[token * half + piece];
        to[da] = narrow<T>(rotary_first(x, y, f));
        to[db] = narrow<T>(rotary_second(x, y, f));
    }
}

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTokens = 4;                 // of a CTA, which forms their cosines and sines once for all its heads
constexpr int kMaxRotaryDim = 256;

struct RotaryParams {
    RotaryRows rows;
    const long long* positions;                  // [batch * tokens]; null: those from start[batch] on
    const long long* start;
    const float* inv_freq;
    float scale;
    long long tokens;
    int heads, heads_per_cta, token_tiles, head_parts;
};

template <typename T>
__global__ void __launch_bounds__(kRotaryThreads, 4)
rotary_kernel(const RotaryParams p) {
    __shared__ __align__(16) float2 table[kRotaryTokens * kMaxRotaryDim / 2];
    pdl_release_downstream();
    pdl_wait_for_upstream();
    const int part = blockIdx.x % p.head_parts;
    const unsigned rest = blockIdx.x / p.head_parts;
    const long long b = rest / p.token_tiles;
    const long long first = static_cast<long long>(rest % p.token_tiles) * kRotaryTokens;
    const int tokens = static_cast<int>(min(static_cast<long long>(kRotaryTokens), p.tokens - first));
    const int half = p.rows.rotary_dim / 2;
    for (int i = threadIdx.x; i < tokens * half; i += blockDim.x) {
        const long long token = first + i / half;
        table[i] = rotary_factors(p.positions != nullptr ? p.positions[b * p.tokens + token] : p.start[b] + token, turns_of(p.inv_freq[i % half]), p.scale);
    }
    __syncthreads();
    const int first_head = part * p.heads_per_cta;
    rotate_rows<T>(p.rows, table, b, first, tokens, first_head, min(p.heads_per_cta, p.heads - first_head));
}

// ------------------------------------------------------------------ tokens into the cache

constexpr int kAppendThreads = 768;               // of an SM: what 80 registers each allow

struct AppendParams {
    KvCache cache;
    RowView k, v;
    long long tokens;
    const long long* start;
    const long long* counts;                     // null: all `tokens` of every sequence
    bool wide;                                   // k and v can be read 16 bytes at a time
    int chunks;                                  // CTAs of a sequence and head, which take the blocks that its tokens touch in turn
    // with rotary positions
    const float* inv_freq;
    float rope_scale;
    int rotary_dim;
    bool interleaved;
    RotaryRows q;
    int q_heads, q_heads_per_cta, q_parts;       // q_parts == 0: no queries
};

// Sixteen numbers of a row, as eight words.
template <typename T>
__device__ __forceinline__ void load16(const T* src, bool wide, uint32_t (&w)[8]) {
    if (wide) {
        const uint4 a = *reinterpret_cast<const uint4*>(src), b = *(reinterpret_cast<const uint4*>(src) + 1);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = h[2 * i] | static_cast<uint32_t>(h[2 * i + 1]) << 16;
    }
}

// Largest magnitude of sixteen numbers, NaN if one is NaN.
__device__ __forceinline__ uint32_t max2_or_nan(uint32_t a, uint32_t b, __half) {
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    return a;
}
__device__ __forceinline__ uint32_t max2_or_nan(uint32_t a, uint32_t b, __nv_bfloat16) {
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    return a;
}
// (Bits of 16-bit numbers without a sign are ordered as the numbers are, NaN last: from here on the maximum is an integer's.)
template <typename T>
__device__ __forceinline__ unsigned magnitude16(const uint32_t (&w)[8]) {
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max2_or_nan(m, w[i] & 0x7fff7fffu, T());
    return max(m & 0xffffu, m >> 16);
}

// Four codes of a word each: round_half_even(127 x / top).
//
// Exactly: x and top have eleven bits at most, so 127 x / top is either on a tie k + 1/2 or further from one than 2^-20 of itself.
// 127 / top is taken a little too large and a little too small (by 2^-22 to 2^-21); the products with x, rounded to an integer by adding
// 1.5 * 2^23, whose low byte then is the code, are the same unless 127 x / top is a tie.  A lane that sees one does its sixteen
// over with the division: 127 x has 18 bits, and the quotient, correctly rounded, is the tie.  (With the division throughout 2 x 8191
// tokens written and read back took 62 us.)
template <typename T>
__device__ __forceinline__ void codes16(const uint32_t (&w)[8], float top, uint32_t (&codes)[4]) {
    constexpr float kMagic = 12582912.0f;
    if (!(top > 0.0f && top <= 3.4028235e38f)) {                         // a block of zeros, or with a NaN or infinity in it
        codes[0] = codes[1] = codes[2] = codes[3] = 0;
        return;
    }
    const float by = __fdividef(127.0f, top);
    const float above = by * 1.0000004f, below = by * 0.9999996f;
    uint32_t differ = top > 1.0e-30f && top < 1.0e30f ? 0u : 1u;         // (beyond these 127 / top may not be a normal number)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = widen2<T>(w[2 * i]), b = widen2<T>(w[2 * i + 1]);
        const float x[4] = {a.x, a.y, b.x, b.y};
        uint32_t bits[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            bits[e] = __float_as_uint(fmaf(x[e], above, kMagic));
            differ |= bits[e] ^ __float_as_uint(fmaf(x[e], below, kMagic));
        }
        codes[i] = __byte_perm(__byte_perm(bits[0], bits[1], 0x0040), __byte_perm(bits[2], bits[3], 0x0040), 0x5410);
    }
    if (differ != 0) {
        // (a top near the end of BF16's range: both brought down, so that 127 x stays finite)
        const float shrink = top > 1.0e36f ? 1.0f / 256.0f : 1.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t word = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float2 x = widen2<T>(w[2 * i + e]);
                const int lo = __float2int_rn(__fdiv_rn(x.x * shrink * 127.0f, top * shrink));
                const int hi = __float2int_rn(__fdiv_rn(x.y * shrink * 127.0f, top * shrink));
                word |= (static_cast<uint32_t>(lo) & 0xffu | (static_cast<uint32_t>(hi) & 0xffu) << 8) << (16 * e);
            }
            codes[i] = word;
        }
    }
}

// Four words of four bytes each, rows and columns exchanged.
__device__ __forceinline__ void transpose_bytes(uint32_t (&w)[4]) {
    const uint32_t lo01 = __byte_perm(w[0], w[1], 0x5140), hi01 = __byte_perm(w[0], w[1], 0x7362);      // 0a 1a 0b 1b; 0c 1c 0d 1d
    const uint32_t lo23 = __byte_perm(w[2], w[3], 0x5140), hi23 = __byte_perm(w[2], w[3], 0x7362);
    w[0] = __byte_perm(lo01, lo23, 0x5410);
    w[1] = __byte_perm(lo01, lo23, 0x7632);
    w[2] = __byte_perm(hi01, hi23, 0x5410);
    w[3] = __byte_perm(hi01, hi23, 0x7632);
}

// Where a 16-byte piece of a block's value codes is kept in shared memory: in its line of 32, moved so that threads that work on
// other lines meet other banks.
__device__ __forceinline__ int value_piece(int line, int piece) { return line * 32 + (piece ^ (line & 7)); }

__device__ __forceinline__ float scale_of(float top) {
    return top <= 3.4028235e38f ? __fdiv_rn(top, 127.0f) : __int_as_float(0x7fc00000);
}

// A CTA takes blocks of one sequence and key/value head that the new tokens touch: a thread owns sixteen numbers of a key and of a
// value.  A block that becomes full is read (older tokens from the tail), its codes and scales are written; of the last token's block and
// the one before it the numbers themselves go to the tail, into the slot of the block's parity.  The CTA of the first block reads a tail
// slot that one of those two may write, so it writes that slot itself, after it has read.
template <typename T, int D, bool ROTARY>
__global__ void __launch_bounds__(2 * D, kAppendThreads / (2 * D))
kv_append_kernel(const AppendParams p) {
    constexpr int kThreads = 2 * D, kWarps = kThreads / 32;
    extern __shared__ __align__(16) float2 factors[];                              // [32][rotary_dim / 2]
    __shared__ __align__(16) uint4 turned_codes[2 * D];               // a block's value codes in the cache's order
    __shared__ unsigned tops[2][kWarps];
    pdl_release_downstream();
    pdl_wait_for_upstream();
    const int tid = threadIdx.x;
    // The factors of tokens [from, to) of 32 whose first is at position `first`: a thread keeps to one pair, several tokens under way.
    // (2048 tokens of 8 heads of 128 turned and written: 14.5 us; pairs and tokens numbered through, and partners read one by one, 24.7.)
    auto form_factors = [&](long long first, int from, int to) {
        const int half = p.rotary_dim / 2, pair = tid % (D / 2);
        if (pair >= half) return;
        const double turns = turns_of(p.inv_freq[pair]);
#pragma unroll 4
        for (int token = from + tid / (D / 2); token < to; token += kThreads / (D / 2)) {
            factors[token * half + pair] = rotary_factors(first + token, turns, p.rope_scale);
        }
    };
    const unsigned cache_ctas = static_cast<unsigned>(p.cache.batch) * p.cache.kv_heads * p.chunks;
    if (ROTARY && blockIdx.x >= cache_ctas) {                         // queries
        const unsigned at = blockIdx.x - cache_ctas;
        const int part = at % p.q_parts;
        const long long b = at / p.q_parts;
        const int tokens = static_cast<int>(p.tokens);                // (a block's worth at most)
        form_factors(p.start[b], 0, tokens);
        __syncthreads();
        const int head = part * p.q_heads_per_cta;
        rotate_rows<T>(p.q, factors, b, 0, tokens, head, min(p.q_heads_per_cta, p.q_heads - head));
        return;
    }
    const int chunk = blockIdx.x % p.chunks;
    const unsigned pair = blockIdx.x / p.chunks;                       // sequence and head
    const int b = pair / p.cache.kv_heads, head = pair % p.cache.kv_heads;
    const long long start = p.start[b];
    const long long count = p.counts == nullptr ? p.tokens : p.counts[b];
    if (start < 0 || count < 0 || count > p.tokens || start > p.cache.max_len - count) {
        if (tid == 0) atomicOr(p.cache.status, kKvBadLength);
        return;
    }
    const int begin = static_cast<int>(start), end = begin + static_cast<int>(count);
    if (count == 0) return;
    const int first_block = begin / kKvBlock, newest = end / kKvBlock;   // `newest`: the one that the next token goes to
    const int last_block = (end - 1) / kKvBlock;                         // the last token's
    // this thread's token and sixteen dims of the keys: byte tid * 16 of the block's key codes
    constexpr int kRuns = D / 64, kChunks = D / 16;
    const int line = tid / 32, lane = tid % 32;
    const int slot = line / kRuns / 2 * 16 + lane / 4 * 2 + line / kRuns % 2;
    const int d0 = line % kRuns * 64 + lane % 4 * 16;
    // and of the values: four lanes kChunks apart have four tokens in a row
    const int v_slot = tid / kChunks, v_d0 = tid % kChunks * 16;

    T* const k_tail = reinterpret_cast<T*>(p.cache.k_tail) + static_cast<size_t>(pair) * 2 * kKvBlock * D;
    T* const v_tail = reinterpret_cast<T*>(p.cache.v_tail) + static_cast<size_t>(pair) * 2 * kKvBlock * D;

    // The numbers of a block's token as the cache gets them (the key turned), as they lie in the tail where the block is going to be
    // full, or zeros.
    auto fetch = [&](int of_block, uint32_t (&k)[8], uint32_t (&v)[8]) {
        const int t = of_block * kKvBlock + slot, v_t = of_block * kKvBlock + v_slot;
        const bool whole = of_block < newest;
        if (whole && v_t < begin) {
            load16<T>(v_tail + ((of_block & 1) * kKvBlock + v_slot) * D + v_d0, true, v);
        } else if (v_t >= begin && v_t < end) {
            load16<T>(row_of<T>(p.v, b, v_t - begin, head) + v_d0, p.wide, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0;
        }
        if (ROTARY) {
            __syncthreads();
            form_factors(static_cast<long long>(of_block) * kKvBlock, max(0, begin - of_block * kKvBlock), min(kKvBlock, end - of_block * kKvBlock));
            __syncthreads();
        }
        if (whole && t < begin) {
            load16<T>(k_tail + ((of_block & 1) * kKvBlock + slot) * D + d0, true, k);
        } else if (t >= begin && t < end) {
            const T* from = row_of<T>(p.k, b, t - begin, head);
            load16<T>(from + d0, p.wide, k);
            if (ROTARY) {
                const int half = p.rotary_dim / 2;
                const float2* f = factors + slot * half;
                if (!p.interleaved && half % 16 == 0) {               // the partners lie together too
                    if (d0 >= p.rotary_dim) return;
                    const bool upper = d0 >= half;
                    uint32_t partner[8];
                    load16<T>(from + (upper ? d0 - half : d0 + half), p.wide, partner);
                    f += upper ? d0 - half : d0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 x = widen2<T>(k[i]), y = widen2<T>(partner[i]);
                        const float4 two = *reinterpret_cast<const float4*>(f + 2 * i);
                        const float2 f0 = make_float2(two.x, two.y), f1 = make_float2(two.z, two.w);
                        k[i] = upper ? narrow2<T>(rotary_second(y.x, x.x, f0), rotary_second(y.y, x.y, f1))
                                     : narrow2<T>(rotary_first(x.x, y.x, f0), rotary_first(x.y, y.y, f1));
                    }
                    return;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int d = d0 + 2 * i;
                    const float2 own = widen2<T>(k[i]);
                    float x[2] = {own.x, own.y};
                    if (p.interleaved) {
                        if (d < p.rotary_dim) {
                            x[0] = rotary_first(own.x, own.y, f[d / 2]);
                            x[1] = rotary_second(own.x, own.y, f[d / 2]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if (d + e < half) x[e] = rotary_first(x[e], widen<T>(from[d + e + half]), f[d + e]);
                            else if (d + e < p.rotary_dim) x[e] = rotary_second(widen<T>(from[d + e - half]), x[e], f[d + e - half]);
                        }
                    }
                    k[i] = narrow2<T>(x[0], x[1]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) k[i] = 0;
        }
    };
    auto keep = [&](int of_block, const uint32_t (&k)[8], const uint32_t (&v)[8]) {
        const int t = of_block * kKvBlock + slot, v_t = of_block * kKvBlock + v_slot;
        if (t >= begin && t < end) {
            uint4* to = reinterpret_cast<uint4*>(k_tail + static_cast<size_t>((of_block & 1) * kKvBlock + slot) * D + d0);
            to[0] = make_uint4(k[0], k[1], k[2], k[3]);
            to[1] = make_uint4(k[4], k[5], k[6], k[7]);
        }
        if (v_t >= begin && v_t < end) {
            uint4* to = reinterpret_cast<uint4*>(v_tail + static_cast<size_t>((of_block & 1) * kKvBlock + v_slot) * D + v_d0);
            to[0] = make_uint4(v[0], v[1], v[2], v[3]);
            to[1] = make_uint4(v[4], v[5], v[6], v[7]);
        }
    };

    // The one of the last two blocks that has the first one's parity shares its tail slot: the first one's CTA writes it, if it read
    // that slot.
    const int shared = ((last_block - first_block) & 1) == 0 ? last_block : last_block - 1;
    const bool first_reads = begin % kKvBlock != 0 && first_block < newest && shared > first_block;
    uint32_t k[8], v[8], next_k[8], next_v[8];
    // A block ahead (2 x 8191 tokens of 8 heads of 128 written and read back: 42 us, each block fetched in its turn 50; where keys are
    // turned the cosines take the registers).
    auto ask = [&](int block) {
        if (!ROTARY && block * kKvBlock < end) fetch(block, next_k, next_v);
    };
    ask(first_block + chunk);
    for (int block = first_block + chunk; block * kKvBlock < end; block += p.chunks) {
        if (ROTARY) {
            fetch(block, k, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                k[i] = next_k[i];
                v[i] = next_v[i];
            }
            ask(block + p.chunks);
        }
        if (block < newest) {                                             // all of its 32 tokens are there
            unsigned k_bits = __reduce_max_sync(0xffffffffu, magnitude16<T>(k)), v_bits = __reduce_max_sync(0xffffffffu, magnitude16<T>(v));
            if (lane == 0) {
                tops[0][tid / 32] = k_bits;
                tops[1][tid / 32] = v_bits;
            }
            __syncthreads();
            k_bits = __reduce_max_sync(0xffffffffu, tops[0][lane % kWarps]);
            v_bits = __reduce_max_sync(0xffffffffu, tops[1][lane % kWarps]);
            const float k_top = widen2<T>(k_bits).x, v_top = widen2<T>(v_bits).x;
            const size_t at = static_cast<size_t>(pair) * p.cache.blocks + block;
            uint32_t codes[4];
            codes16<T>(k, k_top, codes);
            *reinterpret_cast<uint4*>(p.cache.k_codes + at * (kKvBlock * D) + tid * 16) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
            codes16<T>(v, v_top, codes);
            // Four tokens of four dims each to a lane, in two exchanges (word i of a lane is dims 4 i to 4 i + 3 of its token; then word u
            // of lane i is those of token u), and then bytes, so that a word is four tokens of a dim.
            const int quarter = lane / kChunks % 4;
#pragma unroll
            for (int bit = 1; bit < 4; bit *= 2) {
                const bool upper = (quarter & bit) != 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (i & bit) continue;
                    const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? codes[i] : codes[i + bit], bit * kChunks);
                    if (upper) codes[i] = got;
                    else codes[i + bit] = got;
                }
            }
            transpose_bytes(codes);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at_byte = kv_value_offset<D>(v_slot & ~3, v_d0 + quarter * 4 + i);
                reinterpret_cast<uint32_t*>(turned_codes + value_piece(at_byte / 512, at_byte / 16 % 32))[at_byte / 4 % 4] = codes[i];
            }
            if (tid == 0) {
                p.cache.k_scales[at] = scale_of(k_top);
                p.cache.v_scales[at] = scale_of(v_top);
            }
            __syncthreads();
            *reinterpret_cast<uint4*>(p.cache.v_codes + at * (kKvBlock * D) + tid * 16) = turned_codes[value_piece(line, lane)];
        }
        if (block >= last_block - 1 && !(first_reads && block == shared)) keep(block, k, v);
        if (first_reads && block == first_block) {
            __syncthreads();                                              // all of the old slot has been read
            fetch(shared, k, v);
            keep(shared, k, v);
        }
    }
}

// ------------------------------------------------------------------ the cache read back

struct ReadParams {
    KvCache cache;
    const long long* lengths;
    const long long* first;                      // null: from the first token on
    long long tokens;
    char* k_out;                                 // [batch][tokens][kv heads][D]
    char* v_out;
    int chunks;
};

// A word of four codes times a scale, rounded: (c0, c1) and (c2, c3).
template <typename T>
__device__ __forceinline__ uint2 values4(uint32_t word, float scale) {
    const uint32_t even = hsub2_u32(and_xor(word, 0x00ff00ffu, 0x64806480u), 0x64806480u);              // c0, c2 in FP16
    const uint32_t odd = hsub2_u32(and_xor(word >> 8, 0x00ff00ffu, 0x64806480u), 0x64806480u);
    const float2 a = widen2<__half>(even), b = widen2<__half>(odd);
    return make_uint2(narrow2<T>(a.x * scale, b.x * scale), narrow2<T>(a.y * scale, b.y * scale));
}

// A CTA for a block of one sequence and head; a thread for sixteen numbers of a key, and of the values for four dims of four tokens.
template <typename T, int D>
__global__ void __launch_bounds__(2 * D)
kv_read_kernel(const ReadParams p) {
    constexpr int kRuns = D / 64;
    __shared__ __align__(16) uint4 turned_codes[2 * D];
    pdl_release_downstream();
    pdl_wait_for_upstream();
    const int tid = threadIdx.x, line = tid / 32, lane = tid % 32;
    const int chunk = blockIdx.x % p.chunks;
    const unsigned pair = blockIdx.x / p.chunks;
    const int b = pair / p.cache.kv_heads, head = pair % p.cache.kv_heads;
    long long length = p.lengths[b];
    long long first = p.first == nullptr ? 0 : p.first[b];
    if (length < 0 || length > p.cache.max_len || first < 0 || first > p.cache.max_len) {
        if (tid == 0) atomicOr(p.cache.status, kKvBadLength);
        length = first = 0;
    }
    const long long block = first / kKvBlock + chunk;
    const int slot = line / kRuns / 2 * 16 + lane / 4 * 2 + line / kRuns % 2;
    const int d0 = line % kRuns * 64 + lane % 4 * 16;
    const int quad = tid / (D / 4), v_d0 = tid % (D / 4) * 4;          // tokens 4 quad to 4 quad + 3, dims v_d0 to v_d0 + 3
    uint2 k[4], v[4];
    if (block < length / kKvBlock) {
        const size_t at = static_cast<size_t>(pair) * p.cache.blocks + block;
        const uint4 k_codes = __ldcs(reinterpret_cast<const uint4*>(p.cache.k_codes + at * (kKvBlock * D) + tid * 16));
        turned_codes[value_piece(line, lane)] = __ldcs(reinterpret_cast<const uint4*>(p.cache.v_codes + at * (kKvBlock * D) + tid * 16));
        const float k_scale = p.cache.k_scales[at], v_scale = p.cache.v_scales[at];
        k[0] = values4<T>(k_codes.x, k_scale);
        k[1] = values4<T>(k_codes.y, k_scale);
        k[2] = values4<T>(k_codes.z, k_scale);
        k[3] = values4<T>(k_codes.w, k_scale);
        __syncthreads();
        uint32_t words[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at_byte = kv_value_offset<D>(quad * 4, v_d0 + i);
            words[i] = reinterpret_cast<const uint32_t*>(turned_codes + value_piece(at_byte / 512, at_byte / 16 % 32))[at_byte / 4 % 4];
        }
        transpose_bytes(words);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = values4<T>(words[i], v_scale);
    } else {
        const size_t tail = (static_cast<size_t>(pair) * 2 + (block & 1)) * kKvBlock * D;
        const T* k_tail = reinterpret_cast<const T*>(p.cache.k_tail) + tail + slot * D + d0;
        const T* v_tail = reinterpret_cast<const T*>(p.cache.v_tail) + tail + quad * 4 * D + v_d0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            k[i] = block * kKvBlock + slot < length ? reinterpret_cast<const uint2*>(k_tail)[i] : make_uint2(0u, 0u);
            v[i] = block * kKvBlock + quad * 4 + i < length ? *reinterpret_cast<const uint2*>(v_tail + i * D) : make_uint2(0u, 0u);
        }
    }
    const long long before = block * kKvBlock - first;                  // rows of the output in front of this block's
    const size_t row_numbers = static_cast<size_t>(p.cache.kv_heads) * D;
    const size_t out = (static_cast<size_t>(b) * p.tokens * p.cache.kv_heads + head) * D;
    if (before + slot >= 0 && before + slot < p.tokens) {
        uint4* to = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.k_out) + out + (before + slot) * row_numbers + d0);
        __stcs(to, make_uint4(k[0].x, k[0].y, k[1].x, k[1].y));
        __stcs(to + 1, make_uint4(k[2].x, k[2].y, k[3].x, k[3].y));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long row = before + quad * 4 + i;
        if (row < 0 || row >= p.tokens) continue;
        __stcs(reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.v_out) + out + row * row_numbers + v_d0), v[i]);
    }
}

bool wide_rows(const w4a16_rows& r) {
    return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.batch_stride % 8 == 0 && r.token_stride % 8 == 0 && r.head_stride % 8 == 0;
}

RowView view_of(const w4a16_rows& r) {
    return RowView{static_cast<const char*>(r.data), r.batch_stride, r.token_stride, r.head_stride};
}

RotaryRows rotary_rows(const w4a16_rotary_spec& spec, const w4a16_rows& in, const w4a16_rows& out, int head_dim) {
    RotaryRows rows{view_of(in), view_of(out), head_dim, spec.rotary_dim, spec.interleaved != 0, false, false, in.data == out.data, 0, 0};
    rows.aligned = wide_rows(in) && wide_rows(out) && head_dim % 8 == 0;
    rows.wide = rows.aligned && (spec.interleaved ? spec.rotary_dim : spec.rotary_dim / 2) % 8 == 0;
    rows.pieces = rows.wide ? spec.rotary_dim / (spec.interleaved ? 8 : 16) + (rows.in_place ? 0 : (head_dim - spec.rotary_dim) / 8)
                            : (rows.in_place ? spec.rotary_dim + 7 : head_dim) / 8;
    while (1 << rows.piece_bits < rows.pieces) ++rows.piece_bits;
    return rows;
}

// Heads of a CTA where `ctas` CTAs take all heads of some tokens: all of them for prompts, which then form each cosine once; fewer
// where that would leave SMs idle, but eight.
int heads_per_cta(int heads, long long ctas) {
    int parts = 1;
    while (parts * ctas < 296 && heads / (2 * parts) >= 8) parts *= 2;
    return (heads + parts - 1) / parts;
}

}  // namespace

static int turn_rows(const w4a16_rotary_spec& spec, const w4a16_rows& x, const w4a16_rows& out, int64_t batch, int64_t tokens, int heads,
                     int head_dim, const long long* positions, const long long* start, bool bf16, bool programmatic, cudaStream_t stream) {
    RotaryParams p{};
    p.rows = rotary_rows(spec, x, out, head_dim);
    p.positions = positions;
    p.start = start;
    p.inv_freq = spec.inv_freq;
    p.scale = spec.scale;
    p.tokens = tokens;
    p.heads = heads;
    const int64_t tiles = (tokens + kRotaryTokens - 1) / kRotaryTokens;
    if (tiles > INT32_MAX / batch) return W4A16_ERR_TOO_LARGE;
    p.token_tiles = static_cast<int>(tiles);
    p.heads_per_cta = heads_per_cta(heads, tiles * batch);
    p.head_parts = (heads + p.heads_per_cta - 1) / p.heads_per_cta;
    if (tiles * batch > INT32_MAX / p.head_parts) return W4A16_ERR_TOO_LARGE;
    const dim3 grid(static_cast<unsigned>(tiles * batch * p.head_parts));
    auto kernel = bf16 ? rotary_kernel<__nv_bfloat16> : rotary_kernel<__half>;
    return kv_launch(kernel, grid, dim3(kRotaryThreads), 0, programmatic, stream, p);
}

int launch_rotary(const w4a16_rotary_spec& spec, const w4a16_rows& x, const w4a16_rows& out, int64_t batch, int64_t tokens, int heads,
                  int head_dim, const long long* positions, bool bf16, bool programmatic, cudaStream_t stream) {
    return turn_rows(spec, x, out, batch, tokens, heads, head_dim, positions, nullptr, bf16, programmatic, stream);
}

int launch_kv_append(const w4a16_kv8_cache& cache, const w4a16_rows& k, const w4a16_rows& v, int64_t tokens, const long long* start,
                     const long long* counts, const w4a16_rotary_spec* rotary, const w4a16_rows* q, const w4a16_rows* q_out, int q_heads,
                     bool programmatic, cudaStream_t stream) {
    AppendParams p{};
    p.cache = kv_view(cache);
    p.k = view_of(k);
    p.v = view_of(v);
    p.tokens = tokens;
    p.start = start;
    p.counts = counts;
    p.wide = wide_rows(k) && wide_rows(v);
    // (tokens beyond the cache are refused on the device; here they would only make CTAs without work)
    const int64_t at_most = tokens < cache.max_len ? tokens : cache.max_len;
    const int64_t pairs = static_cast<int64_t>(cache.batch) * cache.kv_heads, touched = (at_most + 2 * kKvBlock - 2) / kKvBlock;
    const int64_t resident = 148 * (kAppendThreads / (2 * cache.head_dim));
    p.chunks = static_cast<int>(std::min(touched, std::max<int64_t>(1, resident / pairs)));
    int64_t ctas = pairs * p.chunks;
    const bool bf16 = cache.type == W4A16_TYPE_BF16;
    size_t smem = 0;
    if (rotary != nullptr) {
        p.inv_freq = rotary->inv_freq;
        p.rope_scale = rotary->scale;
        p.rotary_dim = rotary->rotary_dim;
        p.interleaved = rotary->interleaved != 0;
        smem = static_cast<size_t>(kKvBlock) * (rotary->rotary_dim / 2) * sizeof(float2);
        if (q != nullptr && tokens > kKvBlock) {
            // Many queries are turned by a launch of their own (8191 tokens, 64 heads beside 8 of keys: 115 us with that, 127 by CTAs of
            // the same launch).
            if (const int status = turn_rows(*rotary, *q, *q_out, cache.batch, tokens, q_heads, cache.head_dim, nullptr, start, bf16, programmatic, stream);
                status != W4A16_OK) {
                return status;
            }
        } else if (q != nullptr) {
            p.q = rotary_rows(*rotary, *q, *q_out, cache.head_dim);
            p.q_heads = q_heads;
            p.q_heads_per_cta = heads_per_cta(q_heads, cache.batch);
            p.q_parts = (q_heads + p.q_heads_per_cta - 1) / p.q_heads_per_cta;
            ctas += static_cast<int64_t>(cache.batch) * p.q_parts;
        }
    }
    if (ctas > INT32_MAX) return W4A16_ERR_TOO_LARGE;
    auto pick = [&](auto turned) {
        constexpr bool kTurned = decltype(turned)::value;
        return cache.head_dim == 64 ? (bf16 ? kv_append_kernel<__nv_bfloat16, 64, kTurned> : kv_append_kernel<__half, 64, kTurned>)
                                    : (bf16 ? kv_append_kernel<__nv_bfloat16, 128, kTurned> : kv_append_kernel<__half, 128, kTurned>);
    };
    auto kernel = rotary != nullptr ? pick(std::true_type{}) : pick(std::false_type{});
    return kv_launch(kernel, dim3(static_cast<unsigned>(ctas)), dim3(2 * cache.head_dim), smem, programmatic, stream, p);
}

int launch_kv_read(const w4a16_kv8_cache& cache, const long long* lengths, const long long* first, int64_t tokens, void* k_out,
                   void* v_out, bool programmatic, cudaStream_t stream) {
    ReadParams p{};
    p.cache = kv_view(cache);
    p.lengths = lengths;
    p.first = first;
    p.tokens = tokens;
    p.k_out = static_cast<char*>(k_out);
    p.v_out = static_cast<char*>(v_out);
    const int64_t chunks = (tokens + (first == nullptr ? kKvBlock - 1 : 2 * kKvBlock - 2)) / kKvBlock;
    const int64_t ctas = static_cast<int64_t>(cache.batch) * cache.kv_heads;
    if (chunks > INT32_MAX / ctas) return W4A16_ERR_TOO_LARGE;
    p.chunks = static_cast<int>(chunks);
    const bool bf16 = cache.type == W4A16_TYPE_BF16;
    auto kernel = cache.head_dim == 64 ? (bf16 ? kv_read_kernel<__nv_bfloat16, 64> : kv_read_kernel<__half, 64>)
                                       : (bf16 ? kv_read_kernel<__nv_bfloat16, 128> : kv_read_kernel<__half, 128>);
    return kv_launch(kernel, dim3(static_cast<unsigned>(ctas * chunks)), dim3(2 * cache.head_dim), 0, programmatic, stream, p);
}

}  // namespace w4a16
