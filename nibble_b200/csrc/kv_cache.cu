// Rotary positions, and the 8-bit key/value cache written and read back (its format: kv_cache.cuh).
//
// Rotary positions.  Pair j of a head, at position p, is turned by the angle p * inv_freq[j]:
//     (a, b) -> (a cos - b sin, b cos + a sin),      cos and sin times `scale`
// with pairs (2j, 2j + 1) or (j, j + rotary_dim / 2), numbers from rotary_dim on left as they are.  Ways of stretching a context
// (interpolated, by parts, with a temperature) change inv_freq and scale and nothing here.  At a position of 10^6 an FP32 angle
// is off by up to 0.03, so the angle is formed and reduced to a turn in FP64; from there on FP32, rounded once.
//
// Bounds: all three are made of one pass over their data, HBM for prompts and launch latency for a token.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

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

__device__ __forceinline__ float2 rotary_factors(long long position, float inv_freq, float scale) {
    constexpr double kTurnsPerRadian = 0.15915494309189533577;
    double turns = static_cast<double>(position) * (static_cast<double>(inv_freq) * kTurnsPerRadian);
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
    bool wide;                                   // rows can be read and written 16 bytes at a time
    bool in_place;                               // what is not turned is there already
};

// Turns `heads` heads from `first_head` on of `tokens` tokens; table[token * rotary_dim / 2 + pair] holds the factors.
template <typename T>
__device__ void rotate_rows(const RotaryRows& r, const float2* table, long long b, long long first_token, int tokens, int first_head,
                            int heads) {
    const int half = r.rotary_dim / 2;
    const int unit = r.wide ? 8 : 1;             // pairs of a piece (halves); numbers of a piece (pairs, rest)
    const int turned = r.interleaved ? (r.wide ? r.rotary_dim / 8 : half) : half / unit;
    const int pieces = turned + (r.in_place ? 0 : (r.head_dim - r.rotary_dim) / unit);
    const int total = tokens * heads * pieces;
    const int per_token = heads * pieces;
    constexpr int kBatch = 4;                    // pieces requested together
    for (int base = threadIdx.x; base < total; base += kBatch * blockDim.x) {
        const T* from[kBatch];
        T* to[kBatch];
        int piece[kBatch];
        const float2* f[kBatch];
        uint4 lo[kBatch], hi[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int at = base + e * static_cast<int>(blockDim.x);
            if (at >= total) break;
            const int token = at / per_token, rest = at - token * per_token;
            const int head = rest / pieces;
            piece[e] = rest - head * pieces;
            from[e] = row_of<T>(r.in, b, first_token + token, first_head + head);
            to[e] = const_cast<T*>(row_of<T>(r.out, b, first_token + token, first_head + head));
            f[e] = table + token * half;
            if (!r.wide) continue;
            if (piece[e] >= turned) {
                const int d = r.rotary_dim + (piece[e] - turned) * 8;
                lo[e] = *reinterpret_cast<const uint4*>(from[e] + d);
            } else {
                lo[e] = *reinterpret_cast<const uint4*>(from[e] + piece[e] * 8);
                if (!r.interleaved) hi[e] = *reinterpret_cast<const uint4*>(from[e] + half + piece[e] * 8);
            }
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            if (base + e * static_cast<int>(blockDim.x) >= total) break;
            if (r.wide) {
                if (piece[e] >= turned) {
                    const int d = r.rotary_dim + (piece[e] - turned) * 8;
                    *reinterpret_cast<uint4*>(to[e] + d) = lo[e];
                } else if (r.interleaved) {
                    turn8_pairs<T>(lo[e], f[e] + piece[e] * 4);
                    *reinterpret_cast<uint4*>(to[e] + piece[e] * 8) = lo[e];
                } else {
                    turn8_halves<T>(lo[e], hi[e], f[e] + piece[e] * 8);
                    *reinterpret_cast<uint4*>(to[e] + piece[e] * 8) = lo[e];
                    *reinterpret_cast<uint4*>(to[e] + half + piece[e] * 8) = hi[e];
                }
            } else if (piece[e] >= turned) {
                const int d = r.rotary_dim + piece[e] - turned;
                to[e][d] = from[e][d];
            } else {
                const int da = r.interleaved ? 2 * piece[e] : piece[e], db = r.interleaved ? da + 1 : da + half;
                const float x = widen<T>(from[e][da]), y = widen<T>(from[e][db]);
                to[e][da] = narrow<T>(rotary_first(x, y, f[e][piece[e]]));
                to[e][db] = narrow<T>(rotary_second(x, y, f[e][piece[e]]));
            }
        }
    }
}

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTokens = 8;                 // of a CTA, which forms their cosines and sines once for all its heads
constexpr int kMaxRotaryDim = 256;

struct RotaryParams {
    RotaryRows rows;
    const long long* positions;                  // [batch * tokens]
    const float* inv_freq;
    float scale;
    long long tokens;
    int heads, heads_per_cta, token_tiles, head_parts;
};

template <typename T>
__global__ void __launch_bounds__(kRotaryThreads)
rotary_kernel(const RotaryParams p) {
    __shared__ float2 table[kRotaryTokens * kMaxRotaryDim / 2];
    pdl_release_downstream();
    pdl_wait_for_upstream();
    const int part = blockIdx.x % p.head_parts;
    const unsigned rest = blockIdx.x / p.head_parts;
    const long long b = rest / p.token_tiles;
    const long long first = static_cast<long long>(rest % p.token_tiles) * kRotaryTokens;
    const int tokens = static_cast<int>(min(static_cast<long long>(kRotaryTokens), p.tokens - first));
    const int half = p.rows.rotary_dim / 2;
    for (int i = threadIdx.x; i < tokens * half; i += blockDim.x) {
        table[i] = rotary_factors(p.positions[b * p.tokens + first + i / half], p.inv_freq[i % half], p.scale);
    }
    __syncthreads();
    const int first_head = part * p.heads_per_cta;
    rotate_rows<T>(p.rows, table, b, first, tokens, first_head, min(p.heads_per_cta, p.heads - first_head));
}

// ------------------------------------------------------------------ tokens into the cache

// The larger of two numbers; NaN if either is.
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

struct AppendParams {
    KvCache cache;
    RowView k, v;
    long long tokens;
    const long long* start;
    const long long* counts;                     // null: all `tokens` of every sequence
    bool wide;                                   // k and v can be read 16 bytes at a time
    int chunks;                                  // CTAs of a sequence and head: blocks that its tokens can touch
    // with rotary positions
    const float* inv_freq;
    float rope_scale;
    int rotary_dim;
    bool interleaved;
    RotaryRows q;
    int q_heads, q_heads_per_cta, q_parts, q_tiles;        // q_parts == 0: no queries
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
template <typename T>
__device__ __forceinline__ float magnitude16(const uint32_t (&w)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 f = widen2<T>(w[i]);
        m = max_or_nan(m, max_or_nan(fabsf(f.x), fabsf(f.y)));
    }
    return m;
}

// Four codes of a word each.  round_half_even(127 x / top): 127 x is exact in FP32 (11 + 7 bits) and the quotient is rounded
// correctly; unless 127 x / top lies on a tie it is further from one than the quotient's rounding, and a tie is exact.  So the
// codes are those of exact arithmetic.
template <typename T>
__device__ __forceinline__ void codes16(const uint32_t (&w)[8], float top, uint32_t (&codes)[4]) {
    // (a top near the end of BF16's range: both brought down, so that 127 x stays finite)
    const float shrink = top > 1.0e36f ? 1.0f / 256.0f : 1.0f;
    const float by = top * shrink;
    const bool plain = top > 0.0f && top <= 3.4028235e38f;               // not for blocks of zeros, nor with a NaN or infinity
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = widen2<T>(w[2 * i]), b = widen2<T>(w[2 * i + 1]);
        const float x[4] = {a.x, a.y, b.x, b.y};
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int code = plain ? __float2int_rn(__fdiv_rn(x[e] * shrink * 127.0f, by)) : 0;
            word |= (static_cast<uint32_t>(code) & 0xffu) << (8 * e);
        }
        codes[i] = word;
    }
}

__device__ __forceinline__ float scale_of(float top) {
    return top <= 3.4028235e38f ? __fdiv_rn(top, 127.0f) : __int_as_float(0x7fc00000);
}

// One CTA for a block of one sequence and key/value head that the new tokens touch: a thread owns sixteen numbers of a key and of a
// value.  A block that becomes full is read (older tokens from the tail), its codes and scales are written; of the newest two blocks
// the numbers themselves go to the tail, into the slot of the block's parity.  The CTA of the first block reads a tail slot that the
// newest blocks may write, so it writes that slot itself, after it has read.
template <typename T, int D, bool ROTARY>
__global__ void __launch_bounds__(2 * D)
kv_append_kernel(const AppendParams p) {
    constexpr int kThreads = 2 * D, kWarps = kThreads / 32;
    extern __shared__ float2 factors[];                              // [32][rotary_dim / 2]
    __shared__ __align__(16) uint8_t turned_codes[kKvBlock * D];      // a block's value codes in the cache's order
    __shared__ float tops[2][kWarps];
    pdl_release_downstream();
    pdl_wait_for_upstream();
    const int tid = threadIdx.x;
    const unsigned cache_ctas = static_cast<unsigned>(p.cache.batch) * p.cache.kv_heads * p.chunks;
    if (ROTARY && blockIdx.x >= cache_ctas) {                         // queries
        const unsigned at = blockIdx.x - cache_ctas;
        const int part = at % p.q_parts;
        const unsigned rest = at / p.q_parts;
        const long long b = rest / p.q_tiles, first = static_cast<long long>(rest % p.q_tiles) * kKvBlock;
        const int tokens = static_cast<int>(min(static_cast<long long>(kKvBlock), p.tokens - first)), half = p.rotary_dim / 2;
        const long long start = p.start[b];
        for (int i = tid; i < tokens * half; i += kThreads) {
            factors[i] = rotary_factors(start + first + i / half, p.inv_freq[i % half], p.rope_scale);
        }
        __syncthreads();
        const int head = part * p.q_heads_per_cta;
        rotate_rows<T>(p.q, factors, b, first, tokens, head, min(p.q_heads_per_cta, p.q_heads - head));
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
    const int first_block = begin / kKvBlock, newest = end / kKvBlock;   // `newest`: the one that the next token goes to
    const int block = first_block + chunk;
    if (count == 0 || block * kKvBlock >= end) return;
    // this thread's token and sixteen dims: byte tid * 16 of the block's key codes
    constexpr int kRuns = D / 64;
    const int line = tid / 32, lane = tid % 32;
    const int slot = line / kRuns / 2 * 16 + lane / 4 * 2 + line / kRuns % 2;
    const int d0 = line % kRuns * 64 + lane % 4 * 16;

    T* const k_tail = reinterpret_cast<T*>(p.cache.k_tail) + static_cast<size_t>(pair) * 2 * kKvBlock * D;
    T* const v_tail = reinterpret_cast<T*>(p.cache.v_tail) + static_cast<size_t>(pair) * 2 * kKvBlock * D;

    // The numbers of a block's token as the cache gets them (the key turned), as they lie in the tail, or zeros.
    auto fetch = [&](int of_block, uint32_t (&k)[8], uint32_t (&v)[8]) {
        const int t = of_block * kKvBlock + slot;
        if (ROTARY) {
            __syncthreads();
            const int half = p.rotary_dim / 2;
            for (int i = tid; i < kKvBlock * half; i += kThreads) {
                factors[i] = rotary_factors(static_cast<long long>(of_block) * kKvBlock + i / half, p.inv_freq[i % half], p.rope_scale);
            }
            __syncthreads();
        }
        if (t < begin) {
            load16<T>(k_tail + ((of_block & 1) * kKvBlock + slot) * D + d0, true, k);
            load16<T>(v_tail + ((of_block & 1) * kKvBlock + slot) * D + d0, true, v);
        } else if (t < end) {
            const T* from = row_of<T>(p.k, b, t - begin, head);
            load16<T>(from + d0, p.wide, k);
            load16<T>(row_of<T>(p.v, b, t - begin, head) + d0, p.wide, v);
            if (ROTARY) {
                const int half = p.rotary_dim / 2;
                const float2* f = factors + slot * half;
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
            for (int i = 0; i < 8; ++i) k[i] = v[i] = 0;
        }
    };
    auto keep = [&](int of_block, const uint32_t (&k)[8], const uint32_t (&v)[8]) {
        const int t = of_block * kKvBlock + slot;
        if (t < begin || t >= end) return;
        const size_t at = static_cast<size_t>((of_block & 1) * kKvBlock + slot) * D + d0;
        uint4* to_k = reinterpret_cast<uint4*>(k_tail + at);
        uint4* to_v = reinterpret_cast<uint4*>(v_tail + at);
        to_k[0] = make_uint4(k[0], k[1], k[2], k[3]);
        to_k[1] = make_uint4(k[4], k[5], k[6], k[7]);
        to_v[0] = make_uint4(v[0], v[1], v[2], v[3]);
        to_v[1] = make_uint4(v[4], v[5], v[6], v[7]);
    };

    uint32_t k[8], v[8];
    fetch(block, k, v);
    if (block < newest) {                                             // all of its 32 tokens are there
        float k_top = magnitude16<T>(k), v_top = magnitude16<T>(v);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            k_top = max_or_nan(k_top, __shfl_xor_sync(0xffffffffu, k_top, o));
            v_top = max_or_nan(v_top, __shfl_xor_sync(0xffffffffu, v_top, o));
        }
        if (lane == 0) {
            tops[0][tid / 32] = k_top;
            tops[1][tid / 32] = v_top;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            k_top = max_or_nan(k_top, tops[0][w]);
            v_top = max_or_nan(v_top, tops[1][w]);
        }
        const size_t at = static_cast<size_t>(pair) * p.cache.blocks + block;
        uint32_t codes[4];
        codes16<T>(k, k_top, codes);
        *reinterpret_cast<uint4*>(p.cache.k_codes + at * (kKvBlock * D) + tid * 16) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
        codes16<T>(v, v_top, codes);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            turned_codes[kv_value_offset<D>(slot, d0 + e)] = static_cast<uint8_t>(codes[e / 4] >> (8 * (e % 4)));
        }
        if (tid == 0) {
            p.cache.k_scales[at] = scale_of(k_top);
            p.cache.v_scales[at] = scale_of(v_top);
        }
        __syncthreads();
        *reinterpret_cast<uint4*>(p.cache.v_codes + at * (kKvBlock * D) + tid * 16) = *reinterpret_cast<const uint4*>(turned_codes + tid * 16);
    }
    // A newest block of the first one's parity shares its tail slot: the first one's CTA writes it, if it read that slot.
    const int shared = ((newest - first_block) & 1) == 0 ? newest : newest - 1;
    const bool first_reads = begin % kKvBlock != 0 && first_block < newest && shared > first_block;
    if (block >= newest - 1 && !(first_reads && block == shared)) keep(block, k, v);
    if (first_reads && block == first_block && shared * kKvBlock < end) {
        __syncthreads();                                              // all of the old slot has been read
        fetch(shared, k, v);
        keep(shared, k, v);
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

// A CTA for a block of one sequence and head; a thread for sixteen numbers of a key and of a value.
template <typename T, int D>
__global__ void __launch_bounds__(2 * D)
kv_read_kernel(const ReadParams p) {
    constexpr int kRuns = D / 64;
    __shared__ __align__(16) uint8_t turned_codes[kKvBlock * D];
    pdl_release_downstream();
    pdl_wait_for_upstream();
    const int tid = threadIdx.x, line = tid / 32, lane = tid % 32;
    const int chunk = blockIdx.x % p.chunks;
    const unsigned pair = blockIdx.x / p.chunks;
    const int b = pair / p.cache.kv_heads, head = pair % p.cache.kv_heads;
    long long length = p.lengths[b];
    const long long first = p.first == nullptr ? 0 : p.first[b];
    if (length < 0 || length > p.cache.max_len || first < 0) {
        if (tid == 0) atomicOr(p.cache.status, kKvBadLength);
        length = 0;
    }
    const long long block = (first < 0 ? 0 : first / kKvBlock) + chunk;
    const int slot = line / kRuns / 2 * 16 + lane / 4 * 2 + line / kRuns % 2;
    const int d0 = line % kRuns * 64 + lane % 4 * 16;
    const long long t = block * kKvBlock + slot;
    const long long row = t - (first < 0 ? 0 : first);                 // of the output
    uint32_t k[8], v[8];
    if (block < length / kKvBlock) {
        const size_t at = static_cast<size_t>(pair) * p.cache.blocks + block;
        const uint4 k_codes = __ldcs(reinterpret_cast<const uint4*>(p.cache.k_codes + at * (kKvBlock * D) + tid * 16));
        *reinterpret_cast<uint4*>(turned_codes + tid * 16) =
            __ldcs(reinterpret_cast<const uint4*>(p.cache.v_codes + at * (kKvBlock * D) + tid * 16));
        const float k_scale = p.cache.k_scales[at], v_scale = p.cache.v_scales[at];
        const int8_t* codes = reinterpret_cast<const int8_t*>(&k_codes);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            k[i] = narrow2<T>(codes[2 * i] * k_scale, codes[2 * i + 1] * k_scale);
            const int8_t a = static_cast<int8_t>(turned_codes[kv_value_offset<D>(slot, d0 + 2 * i)]);
            const int8_t c = static_cast<int8_t>(turned_codes[kv_value_offset<D>(slot, d0 + 2 * i + 1)]);
            v[i] = narrow2<T>(a * v_scale, c * v_scale);
        }
    } else if (t < length) {
        const size_t at = ((static_cast<size_t>(pair) * 2 + (block & 1)) * kKvBlock + slot) * D + d0;
        load16<T>(reinterpret_cast<const T*>(p.cache.k_tail) + at, true, k);
        load16<T>(reinterpret_cast<const T*>(p.cache.v_tail) + at, true, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = v[i] = 0;
    }
    if (row < 0 || row >= p.tokens) return;
    const size_t at = ((static_cast<size_t>(b) * p.tokens + row) * p.cache.kv_heads + head) * D + d0;
    uint4* to_k = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.k_out) + at);
    uint4* to_v = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.v_out) + at);
    __stcs(to_k, make_uint4(k[0], k[1], k[2], k[3]));
    __stcs(to_k + 1, make_uint4(k[4], k[5], k[6], k[7]));
    __stcs(to_v, make_uint4(v[0], v[1], v[2], v[3]));
    __stcs(to_v + 1, make_uint4(v[4], v[5], v[6], v[7]));
}

bool wide_rows(const w4a16_rows& r) {
    return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.batch_stride % 8 == 0 && r.token_stride % 8 == 0 && r.head_stride % 8 == 0;
}

RowView view_of(const w4a16_rows& r) {
    return RowView{static_cast<const char*>(r.data), r.batch_stride, r.token_stride, r.head_stride};
}

RotaryRows rotary_rows(const w4a16_rotary_spec& spec, const w4a16_rows& in, const w4a16_rows& out, int head_dim) {
    RotaryRows rows{view_of(in), view_of(out), head_dim, spec.rotary_dim, spec.interleaved != 0, false, in.data == out.data};
    rows.wide = wide_rows(in) && wide_rows(out) && head_dim % 8 == 0 &&
                (spec.interleaved ? spec.rotary_dim : spec.rotary_dim / 2) % 8 == 0 && (head_dim - spec.rotary_dim) % 8 == 0;
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

int launch_rotary(const w4a16_rotary_spec& spec, const w4a16_rows& x, const w4a16_rows& out, int64_t batch, int64_t tokens, int heads,
                  int head_dim, const long long* positions, bool bf16, bool programmatic, cudaStream_t stream) {
    RotaryParams p{};
    p.rows = rotary_rows(spec, x, out, head_dim);
    p.positions = positions;
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
    p.chunks = static_cast<int>((at_most + 2 * kKvBlock - 2) / kKvBlock);
    int64_t ctas = static_cast<int64_t>(cache.batch) * cache.kv_heads * p.chunks;
    size_t smem = 0;
    if (rotary != nullptr) {
        p.inv_freq = rotary->inv_freq;
        p.rope_scale = rotary->scale;
        p.rotary_dim = rotary->rotary_dim;
        p.interleaved = rotary->interleaved != 0;
        smem = static_cast<size_t>(kKvBlock) * (rotary->rotary_dim / 2) * sizeof(float2);
        if (q != nullptr) {
            p.q = rotary_rows(*rotary, *q, *q_out, cache.head_dim);
            p.q_heads = q_heads;
            const int64_t tiles = (tokens + kKvBlock - 1) / kKvBlock;
            p.q_heads_per_cta = heads_per_cta(q_heads, tiles * cache.batch);
            p.q_parts = (q_heads + p.q_heads_per_cta - 1) / p.q_heads_per_cta;
            p.q_tiles = static_cast<int>(tiles);
            ctas += tiles * cache.batch * p.q_parts;
        }
    }
    if (ctas > INT32_MAX) return W4A16_ERR_TOO_LARGE;
    const bool bf16 = cache.type == W4A16_TYPE_BF16;
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
