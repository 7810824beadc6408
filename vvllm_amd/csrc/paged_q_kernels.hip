// A paged key-value cache held in 8 and 4 bits: the append that rotates and quantises, rows read back as values, and
// attention of one query per sequence over the codes.  A group of G dims of a row is a minimum m, a scale s (fp16 each) and
// codes c that stand for m + s c.  Row r of page p, kv head h is row (p * KVH + h) * P + r of the page arrays: a kv head's
// keys lie together (16 keys of 128 dims in 4 bits are 1 KB), so that attention reads whole lines of them.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

#include "common.h"
#include "device.h"
#include "paged_split.h"

namespace vvh {

namespace {

// Row of the pages that holds position p of sequence s for kv head 0 (head h: h * P further), -1 for none.
__device__ __forceinline__ int64_t paged_q_row(const PagedQArgs& c, int32_t s, int32_t p)
{
    if (s < 0 || s >= c.B || p < 0 || p / c.P >= c.max_pages) return -1;
    const int32_t page = c.table[(int64_t)s * c.max_pages + p / c.P];
    return page < 0 || page >= c.pages ? -1 : (int64_t)page * c.KVH * c.P + p % c.P;
}

// Place of unit u (8 dims) in a key's row of D dims: units of a 32-dim step apart, the steps of one place together.
__device__ __forceinline__ int32_t key_unit(int32_t u, int32_t D) { return (u & 3) * (D / 32) + (u >> 2); }

template <typename T>
struct __attribute__((aligned(16))) Eight {
    T v[8];
};

__device__ __forceinline__ uint32_t scale_pair(float s, float m)
{
    return (uint32_t)__builtin_bit_cast(uint16_t, (f16)s) | (uint32_t)__builtin_bit_cast(uint16_t, (f16)m) << 16;
}
__device__ __forceinline__ float pair_scale(uint32_t x) { return (float)__builtin_bit_cast(h2, x)[0]; }
__device__ __forceinline__ float pair_min(uint32_t x) { return (float)__builtin_bit_cast(h2, x)[1]; }

// Codes of a lane's 8 values, whose group is the `lanes` lanes around it, to `to`; the group's first lane writes {s, m}.
// A code is a choice between two neighbours, and the formula's in 64 bits.  In 32 bits the level (x - m) / s is off by at most
// 2^-22 of itself (a difference, a reciprocal of one step, a product): where it is further than that from the middle of
// two levels its nearest is the exact one's, else (4 bits: one value in 65536, and real ties) the lane takes 64 bits.
__device__ __forceinline__ void quantise8(const float (&x)[8], int bits, int lanes, uint8_t* to, uint32_t* sm, bool first)
{
    float lo = x[0], hi = x[0], z = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        z = __builtin_fmaf(x[i], 0.0f, z);  // NaN for a value that is not finite
    }
    lo = -group_max(-lo, lanes);
    hi = group_max(hi, lanes);
    const bool fine = group_max(z == 0.0f ? 0.0f : 1.0f, lanes) == 0.0f;
    const float top = bits == 8 ? 255.0f : 15.0f;
    const f16 m = (f16)__builtin_amdgcn_fmed3f(lo, -65504.0f, 65504.0f);
    // (hi - m) / top in 64 bits: by the reciprocal and its remainder, which is the quotient rounded once
    const double r = bits == 8 ? 1.0 / 255.0 : 1.0 / 15.0, range = (double)hi - (double)m, q0 = range * r;
    const double quot = __builtin_fma(__builtin_fma(-(double)top, q0, range), r, q0);
    const f16 s = (f16)__builtin_amdgcn_fmed3f((float)quot, -65504.0f, 65504.0f);
    if (first) *sm = fine ? scale_pair((float)s, (float)m) : 0x7e007e00u;
    uint32_t w[2] = {0, 0};
    if (fine && s != (f16)0.0f) {
        const float rs = __builtin_amdgcn_rcpf((float)s);
        float c[8], far = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float level = (x[i] - (float)m) * rs;
            c[i] = __builtin_rintf(level);
            far = fmaxf(far, __builtin_fabsf(level - c[i]));
        }
        if (far > 0.5f - (bits == 8 ? 0x1p-13f : 0x1p-17f)) {
#pragma unroll
            for (int i = 0; i < 8; i++) c[i] = (float)__builtin_rint(((double)x[i] - (double)m) / (double)s);
        }
        // bytes, within 0 .. 255 by the conversion; 4 bits: those of even and of odd codes, then as halves of bytes
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int word = bits == 8 ? i / 4 : i % 2, byte = bits == 8 ? i % 4 : i / 2;
            w[word] = __builtin_amdgcn_cvt_pk_u8_f32(fminf(c[i], top), byte, w[word]);
        }
    }
    if (bits == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(to) = w[0] | w[1] << 4;
}

// A block a token.  Items: 8 dims of a key (its own 8 values and the 8 that the rotation pairs them with), 8 of a value,
// or 8 pairs of a query head.  A group is 4, 8 or 16 lanes in a row of one wave.  4001 tokens of 32 query and 8 kv heads of
// 128 in fp16 to 4 bits, 88 MB: 21.5 us, 4.1 TB/s, 0.86 of a large copy's rate (with 64-bit divisions for every code 25); 8 tokens of
// 14 and 2 heads of 64: 3.1 us, a launch and its round trips.
template <typename T, int D>
__global__ __launch_bounds__(512) void k_rope_append_paged_q(PagedQArgs c, T* q_out, const T* q, const T* __restrict__ k,
                                                             const T* __restrict__ v, const int32_t* __restrict__ seqs,
                                                             const int32_t* __restrict__ positions, int32_t H,
                                                             const float* __restrict__ rope, int32_t rope_positions)
{
    constexpr int half = D / 2, per = D / 8;
    // queries in waves of their own
    const int32_t kvu = c.KVH * per, qi = (2 * kvu + 63) / 64 * 64, items = qi + H * (half / 8);
    const int64_t t = blockIdx.x;
    const int32_t s = seqs ? seqs[t] : (int32_t)t, p = positions[t];
    if (rope && p >= rope_positions) return;
    const int64_t row = paged_q_row(c, s, p);
    if (row < 0) return;
    const int lanes = c.group / 8;
    for (int32_t i = threadIdx.x; i < items; i += blockDim.x) {
        if (i >= 2 * kvu && i < qi) continue;
        if (i < 2 * kvu) {
            const bool key = i < kvu;
            const int32_t j = key ? i : i - kvu, h = j / per, u = j - h * per;
            const T* src = (key ? k : v) + (t * c.KVH + h) * D;
            const Eight<T> a = *reinterpret_cast<const Eight<T>*>(src + 8 * u);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = (float)a.v[j];
            if (key && rope) {
                const bool low = 8 * u < half;
                const int32_t d = low ? 8 * u : 8 * u - half;
                const Eight<T> b = *reinterpret_cast<const Eight<T>*>(src + (low ? 8 * u + half : 8 * u - half));
                const f4* cs = reinterpret_cast<const f4*>(rope + ((int64_t)p * half + d) * 2);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const f4 w = cs[j / 2];
                    const double co = w[j % 2 * 2], si = w[j % 2 * 2 + 1];
                    const double o = (double)(float)b.v[j] * (low ? -si : si);  // exact, like the product that it is added to
                    x[j] = (float)__builtin_fma((double)x[j], co, o);
                }
            }
            const int bits = key ? c.kb : c.vb;
            const int64_t r = row + (int64_t)h * c.P;
            uint8_t* to = (key ? c.kp : c.vp) + r * (D * bits / 8) + (key ? key_unit(u, D) : u) * bits;
            uint32_t* sm = (key ? c.ks : c.vs) + r * (D / c.group) + u / lanes;
            quantise8(x, bits, lanes, to, sm, u % lanes == 0);
            continue;
        }
        const int32_t j = i - qi, h = j / (half / 8), d = (j - h * (half / 8)) * 8;
        const int64_t at = (t * H + h) * D + d;
        Eight<T> a = *reinterpret_cast<const Eight<T>*>(q + at), b = *reinterpret_cast<const Eight<T>*>(q + at + half);
        const f4* cs = reinterpret_cast<const f4*>(rope + ((int64_t)p * half + d) * 2);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const f4 w = cs[e / 2];
            float r0, r1;
            rope_apply((float)a.v[e], (float)b.v[e], w[e % 2 * 2], w[e % 2 * 2 + 1], r0, r1);
            a.v[e] = (T)r0;
            b.v[e] = (T)r1;
        }
        *reinterpret_cast<Eight<T>*>(q_out + at) = a;
        *reinterpret_cast<Eight<T>*>(q_out + at + half) = b;
    }
}

// A block takes up to 32 tokens: their rows are looked up first, then a wave takes the keys or the values of one kv head at a
// time (gridDim.y blocks share them), 64 pieces of its tokens' rows together, which lie in a row where the tokens do.  A piece
// is 16 bytes of output; UN of them a lane are on their way at a time (a token left out loads row 0).  40 contexts of up to 2000
// tokens, 8 heads of 128 in 4 bits to fp16, 97 MB: 23.7 us, 4.1 TB/s (a lane a unit after another 48); 3 of 20001 in 8 bits to fp32,
// 148 MB: 35.7 us (with 32 bytes a lane, in two stores of half lines, 45).  Bound by HBM, four fifths of it writes.
constexpr int kReadTokens = 32;
template <typename T, int D, int UN>
__global__ __launch_bounds__(256) void k_read_paged_q(PagedQArgs c, T* __restrict__ k_out, T* __restrict__ v_out,
                                                      const int32_t* __restrict__ seqs, const int32_t* __restrict__ positions,
                                                      int64_t tokens, int32_t before, int32_t each)
{
    constexpr int V = 16 / sizeof(T), per = D / V;
    struct __attribute__((aligned(16))) Out {
        T v[V];
    };
    __shared__ int64_t rows[kReadTokens];
    const int64_t t0 = (int64_t)blockIdx.x * each;
    const int32_t n = tokens - t0 < each ? (int32_t)(tokens - t0) : each, lane = threadIdx.x & 63;
    if ((int32_t)threadIdx.x < n) {
        const int64_t t = t0 + threadIdx.x;
        rows[threadIdx.x] = paged_q_row(c, seqs ? seqs[t] : before + (int32_t)t, positions[t]);  // before: tokens of other launches
    }
    __syncthreads();
    const int32_t NG = D / c.group, glog = __builtin_ctz(c.group / V);
    for (int32_t part = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); part < 2 * c.KVH; part += gridDim.y * 4) {
        const bool key = part < c.KVH;
        T* out = key ? k_out : v_out;
        if (!out) continue;
        const int32_t h = key ? part : part - c.KVH;
        const uint8_t* held = key ? c.kp : c.vp;
        const uint32_t* scales = key ? c.ks : c.vs;
        auto some = [&](auto b) {
            constexpr int B = decltype(b)::value;
            typedef typename std::conditional<V * B == 16, uint16_t, typename std::conditional<V * B == 32, uint32_t, uint2>::type>::type Codes;
            for (int32_t i0 = lane; i0 < n * per; i0 += 64 * UN) {
                Codes w[UN];
                uint32_t sm[UN];
                int64_t to[UN];
#pragma unroll
                for (int j = 0; j < UN; j++) {
                    const int32_t i = i0 + 64 * j < n * per ? i0 + 64 * j : 0, tt = i / per, u = i - tt * per;
                    const int64_t row = rows[tt], r = (row < 0 ? 0 : row) + (int64_t)h * c.P;
                    to[j] = row < 0 || i0 + 64 * j >= n * per ? -1 : ((t0 + tt) * c.KVH + h) * D + V * u;
                    const int32_t place = key ? key_unit(V * u / 8, D) * 8 + V * u % 8 : V * u;  // of the piece's codes
                    w[j] = *reinterpret_cast<const Codes*>(held + r * (D * B / 8) + place * B / 8);
                    sm[j] = scales[r * NG + (u >> glog)];
                }
#pragma unroll
                for (int j = 0; j < UN; j++) {
                    const float s = pair_scale(sm[j]), m = pair_min(sm[j]);
                    uint32_t x[2];  // bytes: the codes in order, or of 4 bits the even and the odd ones
                    if constexpr (V * B == 64) {
                        x[0] = w[j].x;
                        x[1] = w[j].y;
                    } else {
                        x[0] = B == 8 ? (uint32_t)w[j] : (uint32_t)w[j] & 0x0f0f0f0fu;
                        x[1] = B == 8 ? 0 : (uint32_t)w[j] >> 4 & 0x0f0f0f0fu;
                    }
                    Out y;
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        const int word = B == 8 ? e / 4 : e % 2, byte = B == 8 ? e % 4 : e / 2;
                        y.v[e] = (T)__builtin_fmaf(s, (float)(x[word] >> (8 * byte) & 255), m);
                    }
                    if (to[j] >= 0) *reinterpret_cast<Out*>(out + to[j]) = y;
                }
            }
        };
        (key ? c.kb : c.vb) == 8 ? some(std::integral_constant<int, 8>{}) : some(std::integral_constant<int, 4>{});
    }
}

// ---------------------------------------------------------------------------
// Attention on the matrix cores, a tile of up to 16 query heads of one kv head (paged_split.h says how tiles and chunks of keys
// are shared out).  A wave takes CH keys at a time, in tiles of 16 that lie together in a page:
//   S^T = K . q^T   A = K's codes less their middle b (8 or 128) as fp16 values, exact.  A group's sum is scaled in fp32:
//                     score = sum_g s_g part_g + (m_g + b s_g) Q_g, Q_g the sum of the group's q.
//                   4-bit codes of fp16 rows are taken as 16 + c instead, and their sums begin at -16 Q_g.
//                   q is scaled by a power of two to a largest of 2^10 .. 2^11 in its row (fp32: high and low part, 22 bits).
//   softmax         online; weights are powers of two of (score - R) kl, R the row's largest score when it last rose by a factor
//                   of more than 2: subtracted before scores are taken to log2 units, so that a row of one key is exact, and scores
//                   of any size, past fp32's range too, give the weights they stand for.
//   O^T += V^T P^T  V's codes go through the wave's LDS region and its transposing reads of 4 and 8 bits, which give a lane the
//                   codes of 16 (8) keys of one dim, less their middle b.  B = p s_g, the weights times their keys'
//                   scales, as fp16 pairs high + low.  What the groups' middles give, sum_k p (m_g + b s_g), is added up in
//                   fp32 beside.
//                   Weights are times 2^14 over 2^es, a power of two above every scale so far, so that p s_g has fp16's range.
// Column r of the products is head r / NGS and, of its groups, every NGS-th from r % NGS on: few heads leave columns free,
// and scaling scores and weights is most of what a chunk costs (96 ragged contexts of 4 heads a kv head and 4 groups 116 us with a
// column a head, which scales everything 4 times).  A column's q is 0 outside of the group, so that an instruction sums
// each column's own; the scores of a head's columns are then added.  Of the output's columns those of a dim's group count.
// Loads of the next chunk are in flight while a chunk is worked on: V and the scales are free once they are in LDS, K once
// the scores are there.  A tile past the end or on no page loads the first rows of page 0 instead; its scores
// become -infinity and its scales 0, whatever they hold.
// Measured in graphs: 32 contexts of 8192 keys, 32 heads on 8 of 128, 4 bits in groups of 32, 336 MB: 72-75 us, 4.6 TB/s; 32 of
// 4096, 8 heads on 8, 8 bits: 285 MB in 58-59 us; 96 from 1 to 8192 keys, 206 MB: 54.8 us.  Large ones are bound by HBM: 32
// contexts of 2048, 4096, 8192 and 16384 keys take 28.2, 43.9, 74.5 and 133 us, 5.6 TB/s for the differences and 14 us beside,
// 4.8 of them the merge, 4 what comes before the first rows (lengths, the search, pages).  The same at head_dim 64, where a chunk
// has half the bytes for as many scores: 128 contexts of 8192 keys, 14 heads on 2, 168 MB: 48-49 us, and 256 of them 83-86, 4.5
// to 4.8 TB/s for the difference.  32 of 8192 keys, 64 heads on 4, whose scales are applied per group: 58 us for 169 MB.
// ---------------------------------------------------------------------------
template <int N>
struct __attribute__((packed, aligned(4))) Words {
    uint32_t w[N];
};

// Codes are less their middle in the products, and minima moved by as much: m + b s is the middle of the group's values, so that
// what sums are made of is not much larger than the values.  (A bias left in, 64 + c or 1024 + c, is fewer instructions, but sums of
// n keys then hold n times the bias: fp16 outputs of 32 contexts of 32768 keys had a fourth of their elements rounded to a neighbour,
// now 0.5 %, for 1 to 6 % of the time.  The code's bits alone, an fp16 subnormal, would cost less yet, but the matrix instruction
// keeps only about 17 bits of products of subnormals.)
template <int BITS>
constexpr float CodeMiddle = BITS == 8 ? 128.0f : 8.0f;

// Masks that the compiler knows nothing of: one in a vector and one in a scalar register are what v_and_or_b32 takes.
struct CodeMasks {
    uint32_t mid, low, high, mid_one, low_one, high_one;
};
__device__ __forceinline__ CodeMasks code_masks()
{
    CodeMasks k{0x00f000f0u, 0x000f000fu, 0x03c003c0u, 0x54005400u, 0x64006400u, 0x4c004c00u};
    asm("" : "+v"(k.mid), "+s"(k.mid_one));
    asm("" : "+v"(k.low), "+s"(k.low_one));
    asm("" : "+v"(k.high), "+s"(k.high_one));
    return k;
}

// 8 codes less their middle as an operand.  4 bits: code pairs (0, 4), (1, 5), (2, 6), (3, 7) of a word, the code in the
// mantissa's bits 4 to 7 (64 + c) or 0 to 3 (1024 + c), then less 72 or 1032; 8 bits: in order, in the mantissa's low bits (1024
// + c), then less 1152.
__device__ __forceinline__ h8 codes4(uint32_t w, const CodeMasks& k)
{
    const uint32_t v = w >> 8;
    const h2 c72 = {(f16)72.0f, (f16)72.0f}, c1032 = {(f16)1032.0f, (f16)1032.0f};
    const h2 a = __builtin_bit_cast(h2, (w & k.low) | k.low_one) - c1032, b = __builtin_bit_cast(h2, (w & k.mid) | k.mid_one) - c72;
    const h2 c = __builtin_bit_cast(h2, (v & k.low) | k.low_one) - c1032, d = __builtin_bit_cast(h2, (v & k.mid) | k.mid_one) - c72;
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ h8 codes8(uint32_t w0, uint32_t w1)
{
    const u4 x = {__builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u),
                  __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)};
    return __builtin_bit_cast(h8, x) - (f16)1152.0f;
}
// 4 bits, in the same order, as 16 + c (the mantissa's bits 6 to 9): for the sums of a key's dims, where 16 is next to the
// largest code (128 contexts of 8192 keys, 14 heads on 2 of 64, 48.3 us, with the codes above 50.0).
__device__ __forceinline__ h8 codes4_plus_16(uint32_t w, const CodeMasks& k)
{
    return __builtin_bit_cast(h8, u4{(w << 6 & k.high) | k.high_one, (w << 2 & k.high) | k.high_one,
                                     (w >> 2 & k.high) | k.high_one, (w >> 6 & k.high) | k.high_one});
}
// High and low fp16 part of a pair of weights; minus: -1, in a register that the compiler knows nothing of, so that a
// difference is one instruction that takes the fp16 as it is.
__device__ __forceinline__ void weight_parts(float a, float b, float minus, uint32_t& hi, uint32_t& lo)
{
    const h2 h = {(f16)a, (f16)b};
    const h2 o = {(f16)__builtin_fmaf((float)h[0], minus, a), (f16)__builtin_fmaf((float)h[1], minus, b)};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, o);
}
// v of the lane that the quad permutation names, as an operand of the instruction that takes it
template <int CTRL>
__device__ __forceinline__ float quad(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

template <typename T_, int D_, int NG, int NGS, int KB, int VBITS>
struct PagedQTiles {
    typedef PagedQArgs Args;
    typedef T_ T;
    static constexpr bool COLUMNS = true;
    static constexpr int D = D_, CH = VBITS == 4 ? 64 : 32, HEAD = CH == 64 ? 2 : 3;
    static constexpr int NT = CH / 16, DS = D / 32, GS = DS / NG;           // tiles, steps of 32 dims, steps of a group
    static constexpr int KRB = D * KB / 8, VRB = D * VBITS / 8;             // bytes of a row
    static constexpr int KW = KRB / 16, VW = VRB / 16;                      // words of a lane's piece of a tile
    // bytes between V's rows in LDS: 16 (8 bits: 8) of them on distinct banks
    static constexpr int VP = VRB == 32 ? 40 : VRB == 48 ? 48 : VRB + 16;
    static constexpr int NP = (NG + NGS - 1) / NGS;                          // groups of a column
    static constexpr int SR = CH + 16, SW = NG * SR;                         // words of a group's scales in LDS, of a chunk's
    static constexpr int VB = CH * VP + 2 * SW * 4;
    static constexpr bool TWO = sizeof(T) == 4, PLUS16 = !TWO && KB == 4;
    // Lane (r, gr): dims 32 s + 8 gr .. + 7 of head r / NGS
    struct Q {
        Eight<T> v[DS];
    };
    // The same as an operand, in the order of the codes
    struct Operand {
        h8 hi[DS], lo[TWO ? DS : 1];
        float sum[NP];  // of the column's groups
        int e;
    };
    // group `p` of column r; where NG is no multiple of NGS, a column without one takes the last again, with a q of 0
    static __device__ __forceinline__ int group_of(int r, int p)
    {
        const int g = p * NGS + r % NGS;
        return NG % NGS == 0 || g < NG ? g : NG - 1;
    }

    static __device__ __forceinline__ void load_q(const T* q, int heads, int lane, Q& x)
    {
        const int h = (lane & 15) / NGS, gr = lane >> 4;
#pragma unroll
        for (int s = 0; s < DS; s++) x.v[s] = h < heads ? *reinterpret_cast<const Eight<T>*>(q + h * D + 32 * s + 8 * gr) : Eight<T>{};
    }
    static __device__ __forceinline__ void prepare(const Q& q, int lane, Operand& x)
    {
        const int r = lane & 15;
        float v[DS][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < DS; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[s][j] = (float)q.v[s].v[j];
                mx = fmaxf(mx, __builtin_fabsf(v[s][j]));
            }
        mx = max_x32(max_x16(mx));
        x.e = mx == 0.0f ? 0 : 137 - (int)(__builtin_bit_cast(uint32_t, mx) >> 23);
#pragma unroll
        for (int p = 0; p < NP; p++) x.sum[p] = 0.0f;
#pragma unroll
        for (int s = 0; s < DS; s++) {
            const bool mine = s / GS % NGS == r % NGS;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int o = KB == 4 ? j / 2 + 4 * (j % 2) : j;
                const float y = mine ? __builtin_ldexpf(v[s][o], x.e) : 0.0f;
                x.hi[s][j] = (f16)y;
                if constexpr (TWO) x.lo[s][j] = (f16)(y - (float)x.hi[s][j]);
                x.sum[s / GS / NGS] += TWO ? (float)x.hi[s][j] + (float)x.lo[TWO ? s : 0][j] : y;
            }
        }
#pragma unroll
        for (int p = 0; p < NP; p++) x.sum[p] = mx == INFINITY ? NAN : sum_x32(sum_x16(x.sum[p]));  // no score of it is a number
    }

    // What a group's codes less their middle are added to
    template <int BITS>
    static __device__ __forceinline__ float middle(uint32_t sm)
    {
        return __builtin_fmaf(pair_scale(sm), CodeMiddle<BITS>, pair_min(sm));
    }

    struct Spot {
        int32_t page, in;
    };
    // Page of the tile of lane's keys in the chunk at c0, and the tile's place in it.
    static __device__ __forceinline__ Spot look(const PagedQArgs& c, int32_t s, int32_t c0, int lane)
    {
        const uint32_t per = (uint32_t)c.P / 16, cap = (uint32_t)c.max_pages * per;
        const uint32_t want = (uint32_t)c0 / 16 + (lane >> 4) % NT, t = want < cap ? want : cap - 1, pg = t / per;
        return Spot{c.table[(int64_t)s * c.max_pages + pg], (int32_t)(t - pg * per)};
    }

    static __device__ __forceinline__ void tile(const PagedQArgs& c, int32_t g, int32_t s, const Q& q0, int32_t c0, int32_t cstep,
                                                int32_t ke, float scale_log2, char* lds, int lane, PagedAcc<D>& acc)
    {
        const int r = lane & 15, gr = lane >> 4;
        uint32_t* const lk = reinterpret_cast<uint32_t*>(lds + CH * VP);
        uint32_t* const lv = lk + SW;
        float minus = -1.0f;
        asm("" : "+s"(minus));
        const CodeMasks masks = code_masks();
        acc.clear();
        float om[NP] = {}, R = -INFINITY, l = 0.0f, ref = 0x1p-30f;
        int es = -30;

        Words<KW> K[NT];
        Words<VW> V[NT];
        Words<NG> S[CH == 64 ? 2 : 1];  // lane = key (32 keys: K's in lanes 0 .. 31, V's in the others)
        int64_t rows[NT];
        bool on;                        // lane's key is one
        auto locate = [&](const Spot& p, int32_t at) {
            const int32_t first = at + 16 * ((lane >> 4) % NT);
            const bool has = p.page >= 0 && p.page < c.pages && first < ke;
            on = has && first + r < ke;
            const int64_t row = has ? ((int64_t)p.page * c.KVH + g) * c.P + p.in * 16 : (int64_t)g * c.P;
#pragma unroll
            for (int t = 0; t < NT; t++) rows[t] = lane_of64((uint64_t)row, 16 * t);
            return row + r;
        };
        auto load_v = [&](int64_t row) {
#pragma unroll
            for (int t = 0; t < NT; t++) V[t] = *reinterpret_cast<const Words<VW>*>(c.vp + rows[t] * VRB + lane * (VW * 4));
            if constexpr (CH == 64) {
                S[0] = *reinterpret_cast<const Words<NG>*>(c.ks + row * NG);
                S[1] = *reinterpret_cast<const Words<NG>*>(c.vs + row * NG);
            } else {
                S[0] = *reinterpret_cast<const Words<NG>*>((lane < 32 ? c.ks : c.vs) + row * NG);
            }
        };
        auto load_k = [&]() {
#pragma unroll
            for (int t = 0; t < NT; t++)
                K[t] = *reinterpret_cast<const Words<KW>*>(c.kp + rows[t] * KRB + (r * KRB + gr * (KRB / 4)));
        };
        if (c0 >= ke) {
            acc.l = 0.0f;
            return;
        }
        Spot spot = look(c, s, c0, lane);
        load_v(locate(spot, c0));
        load_k();
        spot = look(c, s, c0 + cstep, lane);
        Operand q;  // worked out while the first chunk is on its way
        prepare(q0, lane, q);
        // Scores to log2 units: positive (a negative scale turns q's sign), never 0, so that the maximum of the scores is
        // that of the products and -infinity stays.  Scores are below 2^44 and, but for those of queries rounded away, multiples of
        // 2^-48: past these ends all weights are alike, or all but the largest's 0.  A scale that is not finite makes scores NaN.
        const bool fine = scale_log2 - scale_log2 == 0.0f;
        const float kl = fine ? __builtin_amdgcn_fmed3f(__builtin_fabsf(__builtin_ldexpf(scale_log2, -q.e)), 0x1p-100f, 0x1p80f) : 1.0f;
        if (!fine) {
#pragma unroll
            for (int p = 0; p < NP; p++) q.sum[p] = NAN;
        }
        if (scale_log2 < 0.0f) {
#pragma unroll
            for (int x = 0; x < DS; x++) {
                q.hi[x] = -q.hi[x];
                if constexpr (TWO) q.lo[x] = -q.lo[x];
            }
#pragma unroll
            for (int p = 0; p < NP; p++) q.sum[p] = -q.sum[p];
        }
        for (; c0 < ke; c0 += cstep) {
            const uint64_t live = __ballot(on);
            const bool all = CH == 64 ? live == ~0ull : (uint32_t)live == ~0u;
            // ---- V and the scales to LDS
            wave_lds_order();  // after the reads of the chunk before
            float smax = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                uint32_t* to = reinterpret_cast<uint32_t*>(lds + (NT * (lane >> 2) + t) * VP + (lane & 3) * (VRB / 4));
#pragma unroll
                for (int i = 0; i < VW; i++) to[i] = V[t].w[i];
            }
#pragma unroll
            for (int i = 0; i < NG; i++) {
                const uint32_t a = on ? S[0].w[i] : 0u, b = CH == 64 ? (on ? S[CH / 64].w[i] : 0u) : a;
                if constexpr (CH == 64) {
                    lk[i * SR + lane] = a;
                    lv[i * SR + lane] = b;
                } else {
                    (lane < 32 ? lk : lv)[i * SR + lane % 32] = a;
                }
                smax = fmaxf(smax, __builtin_fabsf(pair_scale(b)));
            }
            if (CH == 32 && lane < 32) smax = 0.0f;
            wave_lds_order();
            // ---- the next chunk's V and scales
            load_v(locate(spot, c0 + cstep));
            spot = look(c, s, c0 + 2 * cstep, lane);
            // ---- scores
            f4 sc[NT];
            float cm = -INFINITY;
#pragma unroll
            for (int p = 0; p < NP; p++) {
                f4 part[NT];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float first = PLUS16 ? -16.0f * q.sum[p] : 0.0f;
                    part[t] = f4{first, first, first, first};
#pragma unroll
                    for (int x = p * NGS * GS; x < (p + 1) * NGS * GS && x < DS; x++) {
                        const h8 a = PLUS16   ? codes4_plus_16(K[t].w[x], masks)
                                     : KB == 4 ? codes4(K[t].w[x], masks)
                                               : codes8(K[t].w[2 * x % KW], K[t].w[(2 * x + 1) % KW]);
                        if constexpr (TWO) part[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q.lo[x], part[t], 0, 0, 0);
                        part[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q.hi[x], part[t], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const u4 sm = *reinterpret_cast<const u4*>(lk + group_of(r, p) * SR + 16 * t + 4 * gr);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float y = __builtin_fmaf(PLUS16 ? pair_min(sm[i]) : middle<KB>(sm[i]), q.sum[p], p ? sc[t][i] : 0.0f);
                        sc[t][i] = __builtin_fmaf(pair_scale(sm[i]), part[t][i], y);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (NGS >= 2) sc[t][i] += quad<0xB1>(sc[t][i]);
                    if (NGS >= 4) sc[t][i] += quad<0x4E>(sc[t][i]);
                }
            if (!all) {
                uint64_t bits = live;
                asm volatile("" : "+s"(bits));  // a branch, not 16 selects in every chunk
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (!(bits >> (16 * t + 4 * gr + i) & 1)) sc[t][i] = -INFINITY;
            }
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) cm = fmaxf(cm, sc[t][i]);
            load_k();
            cm = max_x32(max_x16(cm));
            const bool more = (cm - R) * kl > 1.0f;
            if (__any(more || smax > ref)) {  // a new maximum for some head, or a new largest scale
                int en = es;
                if (__any(smax > ref)) {
                    en = (int)(__builtin_bit_cast(uint32_t, group_max(smax, 64)) >> 23) - 126;
                    en = __builtin_amdgcn_readfirstlane(en < 16 ? en : 16);
                    ref = __builtin_ldexpf(1.0f, en);
                }
                const float f = __builtin_amdgcn_exp2f((more ? (R - cm) * kl : 0.0f) + (float)(es - en));
                if (more) R = cm;
                es = en;
                l *= f;
#pragma unroll
                for (int p = 0; p < NP; p++) om[p] *= f;
#pragma unroll
                for (int e = 0; e < D / 16; e++) acc.o[e] *= f;
            }
            const float Rb = R == -INFINITY ? 0.0f : R, up = (float)(14 - es);  // no key yet: every weight is 0
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    sc[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i] - Rb, kl, up));
                    l += sc[t][i];
                }
            // ---- values
#pragma unroll
            for (int p = 0; p < NP; p++) {
                u4 sm[NT], hi[NT / 2], lo[NT / 2];
#pragma unroll
                for (int t = 0; t < NT; t++) sm[t] = *reinterpret_cast<const u4*>(lv + group_of(r, p) * SR + 16 * t + 4 * gr);
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        om[p] = __builtin_fmaf(sc[t][i], middle<VBITS>(sm[t][i]), om[p]);
                // + 0: one instruction that takes the scale as it is
                auto w = [&](int t, int i) { return __builtin_fmaf(sc[t][i], pair_scale(sm[t][i]), 0.0f); };
#pragma unroll
                for (int u = 0; u < NT / 2; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t h, o;
                        if (VBITS == 4) weight_parts(w(2 * u, i), w(2 * u + 1, i), minus, h, o);
                        else weight_parts(w(i / 2, 2 * (i % 2)), w(i / 2, 2 * (i % 2) + 1), minus, h, o);
                        hi[u][i] = h;
                        lo[u][i] = o;
                    }
#pragma unroll
                for (int e = p * NGS * GS * 2; e < (p + 1) * NGS * GS * 2 && e < D / 16; e++) {
                    h8 a[NT / 2];
                    typedef int i2 __attribute__((ext_vector_type(2)));
                    if constexpr (VBITS == 4) {
                        // nibble n of a lane: key 4 gr + n % 4 of tile n / 4
                        const char* src = lds + (16 * gr + 4 * (r & 3) + (r >> 2)) * VP + 8 * e;
                        const i2 w2 = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i2*)(src));
                        a[0] = codes4((uint32_t)w2[0], masks);
                        a[1] = codes4((uint32_t)w2[1], masks);
                    } else {
                        // byte n of a lane: key 4 gr + n % 4 of tile n / 4
                        const char* src = lds + (8 * gr + 2 * (r >> 1 & 3) + (r >> 3)) * VP + 16 * e + 8 * (r & 1);
                        const i2 w2 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i2*)(src));
                        a[0] = codes8((uint32_t)w2[0], (uint32_t)w2[1]);
                    }
#pragma unroll
                    for (int u = 0; u < NT / 2; u++) {
                        acc.o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[u], __builtin_bit_cast(h8, lo[u]), acc.o[e], 0, 0, 0);
                        acc.o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[u], __builtin_bit_cast(h8, hi[u]), acc.o[e], 0, 0, 0);
                    }
                }
            }
        }
        // without the weights' power of two, exactly, so that parts of different ones join by R alone
        const float back = __builtin_ldexpf(1.0f, es);
        float ms[NP];
#pragma unroll
        for (int p = 0; p < NP; p++) ms[p] = sum_x32(sum_x16(om[p])) * back;
#pragma unroll
        for (int e = 0; e < D / 16; e++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc.o[e][i] = __builtin_fmaf(acc.o[e][i], back, ms[e / (2 * GS) / NGS]);
        acc.l = sum_x32(sum_x16(l)) * back;
        acc.m = R * kl;
    }

    // The n heads' sums, from the columns of each dim's group: rows of `pitch` floats and their maxima and sums, which without
    // arrays of their own follow the rows
    static __device__ __forceinline__ void put(const PagedAcc<D>& acc, int lane, int n, float* rows, int pitch, float* wm, float* wl)
    {
        const int r = lane & 15, gr = lane >> 4, h = r / NGS;
        if (h >= n) return;
        float* row = rows + h * pitch;
#pragma unroll
        for (int e = 0; e < D / 16; e++) {
            f4 v = acc.o[e];
            asm("" : "+v"(v));  // here, whatever the column: else the sums go to memory, to be read from there by column
            if (e / (2 * GS) % NGS == r % NGS) *reinterpret_cast<f4*>(row + 16 * e + 4 * gr) = v;
        }
        if (lane % NGS == 0 && gr == 0) {
            (wm ? wm[h] : row[D]) = acc.m;
            (wl ? wl[h] : row[D + 1]) = acc.l;
        }
    }
    // The n heads' outputs
    static __device__ __forceinline__ void store(const PagedAcc<D>& acc, int lane, int n, T* __restrict__ out)
    {
        const int r = lane & 15, gr = lane >> 4, h = r / NGS;
        if (h >= n) return;
        const float inv = acc.l == 0.0f ? 0.0f : 1.0f / acc.l;
#pragma unroll
        for (int e = 0; e < D / 16; e++) {
            f4 v = acc.o[e] * inv;
            asm("" : "+v"(v));  // as above
            if (e / (2 * GS) % NGS == r % NGS) store4(out + h * D + 16 * e + 4 * gr, v);
        }
    }
    static __device__ __forceinline__ void store4(T* to, f4 v)
    {
        typedef T t4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<t4*>(to) = t4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    }
    // A block's sums from its NW waves' (put's rows in os, 16 a wave, D + 4 apart), 4 dims a thread: outputs, or without them a part
    template <int NW>
    static __device__ __forceinline__ void join(T* __restrict__ out, float* __restrict__ part, const float (*wm)[16],
                                                const float (*wl)[16], const float* os, int32_t n)
    {
        constexpr int OP = D + 4;
        for (int idx = threadIdx.x; idx < n * (D / 4); idx += 64 * NW) {
            const int h = idx / (D / 4), d = (idx - h * (D / 4)) * 4;
            float m[NW], M = -INFINITY, den = 0.0f;
#pragma unroll
            for (int i = 0; i < NW; i++) {
                m[i] = wm[i][h];
                M = fmaxf(M, m[i]);
            }
            const float Mb = M == -INFINITY ? 0.0f : M;
            f4 num = {};
#pragma unroll
            for (int i = 0; i < NW; i++) {
                const float f = __builtin_amdgcn_exp2f(m[i] - Mb);
                num += *reinterpret_cast<const f4*>(os + (i * 16 + h) * OP + d) * f;
                den = __builtin_fmaf(f, wl[i][h], den);
            }
            if (out) {
                store4(out + h * D + d, num * (den == 0.0f ? 0.0f : 1.0f / den));
                continue;
            }
            *reinterpret_cast<f4*>(part + h * (D + 4) + d) = num;
            if (d == 0) {
                part[h * (D + 4) + D] = M;
                part[h * (D + 4) + D + 1] = den;
            }
        }
    }
};

// Bytes of LDS a wave: its chunk, then its sums
template <typename TL>
constexpr int kQWaveBytes = TL::VB > 16 * (TL::D + 4) * 4 ? TL::VB : 16 * (TL::D + 4) * 4;

// One tile of one sequence by one block of 1, 2, 4 or 8 waves, each every so many-th chunk, merged through LDS (a wave by itself
// has its sums in registers).
template <typename TL>
__global__ __launch_bounds__(512, 2) void k_attention_paged_q_one(PagedQArgs c, typename TL::T* __restrict__ out,
                                                                  const typename TL::T* __restrict__ q,
                                                                  const int32_t* __restrict__ lens, PagedHeads hd, int32_t H,
                                                                  float scale_log2)
{
    constexpr int D = TL::D, CH = TL::CH, OP = D + 4;
    extern __shared__ __align__(16) char smem[];
    __shared__ float wm[8][16], wl[8][16];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int NW = blockDim.x >> 6;
    const int32_t s = blockIdx.y, len = paged_len(c, lens, s);
    int32_t g, h0, n;
    hd.at(blockIdx.x, g, h0, n);
    const int64_t row0 = (int64_t)s * H + h0;
    typename TL::Q x;
    TL::load_q(q + row0 * D, n, lane, x);
    PagedAcc<D> acc;
    TL::tile(c, g, s, x, w * CH, NW * CH, len, scale_log2, smem + w * kQWaveBytes<TL>, lane, acc);
    typename TL::T* to = out + row0 * D;
    if (NW == 1 || len <= CH) {  // all of it is the first wave's
        if (w == 0) TL::store(acc, lane, n, to);
        return;
    }
    __syncthreads();
    float* os = reinterpret_cast<float*>(smem);
    TL::put(acc, lane, n, os + w * 16 * OP, OP, wm[w], wl[w]);
    __syncthreads();
    if (NW == 8) TL::template join<8>(to, nullptr, wm, wl, os, n);
    else if (NW == 4) TL::template join<4>(to, nullptr, wm, wl, os, n);
    else TL::template join<2>(to, nullptr, wm, wl, os, n);
}
template <typename TL>
__global__ __launch_bounds__(256, 2) void k_attention_paged_q_split(PagedQArgs c, typename TL::T* __restrict__ out,
                                                                    const typename TL::T* __restrict__ q,
                                                                    const int32_t* __restrict__ lens, PagedHeads hd, int32_t H,
                                                                    float scale_log2, int64_t* __restrict__ before_out,
                                                                    float* __restrict__ ws, int32_t VH)
{
    paged_split<TL>(c, out, q, lens, hd, H, scale_log2, before_out, ws, VH);
}

// A launch holds fewer than 2^32 threads: at most 2^22 tokens each (of up to 512).
constexpr int64_t kQTokens = int64_t(1) << 22;

}  // namespace

int launch_rope_append_paged_q(const PagedQArgs& c, void* q_out, const void* q, const void* k, const void* v,
                               const int32_t* seqs, const int32_t* positions, int64_t tokens, int64_t H, const float* rope,
                               int64_t rope_positions, int dtype, void* stream)
{
    const int64_t items = (2 * (int64_t)c.KVH * (c.D / 8) + 63) / 64 * 64 + H * (c.D / 16);
    const int64_t threads = std::min<int64_t>((items + 63) / 64 * 64, tokens > 1024 ? 256 : 512);
    auto go = [&](auto kern, auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        // without seqs token t is sequence t, of fewer than 2^16: one launch
        for (int64_t t = 0; t < tokens; t += kQTokens) {
            const int64_t qd = t * H * c.D, kd = t * c.KVH * c.D;
            hipLaunchKernelGGL(kern, dim3((unsigned)std::min(tokens - t, kQTokens)), dim3((unsigned)threads), 0,
                               static_cast<hipStream_t>(stream), c, (T*)q_out + (q_out ? qd : 0), (const T*)q + (q ? qd : 0),
                               (const T*)k + kd, (const T*)v + kd, seqs ? seqs + t : nullptr, positions + t, (int32_t)H, rope,
                               (int32_t)rope_positions);
        }
    };
    auto dims = [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        c.D == 64 ? go(k_rope_append_paged_q<T, 64>, t) : c.D == 96 ? go(k_rope_append_paged_q<T, 96>, t) : go(k_rope_append_paged_q<T, 128>, t);
    };
    dtype == VVH_F16 ? dims((f16*)nullptr) : dims((float*)nullptr);
    return (int)hipGetLastError();
}

int launch_read_paged_q(const PagedQArgs& c, void* k_out, void* v_out, const int32_t* seqs, const int32_t* positions,
                        int64_t tokens, int dtype, void* stream)
{
    // tokens of a block: as many as leave 1024 blocks of 4 parts (a head's keys or values)
    const int64_t parts = (2 * (int64_t)c.KVH + 3) / 4;
    int64_t each = kReadTokens;
    while (each > 4 && (tokens + each - 1) / each * parts < 1024) each /= 2;
    const int64_t step = std::max<int64_t>(1, kQTokens / parts) * each;  // of a launch: at most 2^22 blocks
    auto go = [&](auto kern, auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        for (int64_t t = 0; t < tokens; t += step) {
            const int64_t n = std::min(tokens - t, step), kd = t * c.KVH * c.D;
            hipLaunchKernelGGL(kern, dim3((unsigned)((n + each - 1) / each), (unsigned)parts), dim3(256), 0,
                               static_cast<hipStream_t>(stream), c, (T*)k_out + (k_out ? kd : 0), (T*)v_out + (v_out ? kd : 0),
                               seqs ? seqs + t : nullptr, positions + t, n, (int32_t)t, (int32_t)each);
        }
    };
    // 8 pieces a lane at a time where a block has as many, else 2 (40 contexts of up to 2000 tokens, 8 heads of 128, 23.6 us, 2
    // at a time 29.7; one of 1500, 2 heads of 64, with 8 4.1, with 2 3.1)
    auto dims = [&](auto* t, auto un) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int UN = decltype(un)::value;
        c.D == 64 ? go(k_read_paged_q<T, 64, UN>, t) : c.D == 96 ? go(k_read_paged_q<T, 96, UN>, t) : go(k_read_paged_q<T, 128, UN>, t);
    };
    auto types = [&](auto un) { dtype == VVH_F16 ? dims((f16*)nullptr, un) : dims((float*)nullptr, un); };
    each == kReadTokens ? types(std::integral_constant<int, 8>{}) : types(std::integral_constant<int, 2>{});
    return (int)hipGetLastError();
}

// Chunks that a block takes by itself, as in paged_kernels.hip
constexpr int64_t kQOneChunks = 16;

AttnPagedPlan attention_paged_q_plan(const PagedQArgs& c, int64_t max_len, int64_t H, int64_t cus)
{
    AttnPagedPlan p{};
    const int64_t G = H / c.KVH;
    p.tiled = true;
    p.tiles = (G + 15) / 16;
    p.GT = (G + p.tiles - 1) / p.tiles;
    // columns of a head: as many of its groups as 16 columns hold
    p.columns = 1;
    while (p.columns * 2 < 2 * (c.D / c.group) && p.GT * p.columns * 2 <= 16) p.columns *= 2;
    const int64_t cap = (int64_t)c.max_pages * c.P, ch = c.vb == 4 ? 64 : 32;
    const int64_t chunks = ((max_len > 0 && max_len < cap ? max_len : cap) + ch - 1) / ch;
    // a wave for each chunk, but no more than the device holds at a time
    p.waves = 1;
    while (p.waves < 8 && p.waves < chunks && p.waves * 2 * c.B * c.KVH * p.tiles <= 8 * cus) p.waves *= 2;
    // Blocks of 4 waves: a chunk a wave where two blocks a CU have as many waves; else one a CU, whose waves have longer runs and
    // leave fewer parts, up to 8 chunks a wave (3 contexts of 30001 keys, fp32, 20.0 -> 18.1 us, 8 of 16000 18.9 -> 17.8, 16 of 8000
    // 20.2 -> 19.4), then two (100 of 8000 93.7 -> 92.4, 40 46.0 -> 44.6, 96 ragged ones 56.8 -> 55.2).
    const int64_t units = chunks * c.B * c.KVH * p.tiles;
    if (chunks > kQOneChunks) p.blocks = std::min<int64_t>((units + 3) / 4, (units <= 8 * cus || units > 32 * cus ? 2 : 1) * cus);
    if (p.blocks > 0) p.ws_floats = paged_before_floats(c.B) + p.blocks * 4 * 2 * p.GT * (c.D + 4);
    return p;
}

template <typename TL>
static void paged_q_go(const AttnPagedPlan& p, const PagedQArgs& c, typename TL::T* out, const typename TL::T* q, const int32_t* lens,
                       int64_t H, float scale_log2, float* ws, hipStream_t s)
{
    const PagedHeads hd{(int32_t)(H / c.KVH), (int32_t)p.GT, (int32_t)p.tiles};
    const int32_t VH = (int32_t)(c.KVH * p.tiles);
    if (p.blocks == 0) {
        hipLaunchKernelGGL((k_attention_paged_q_one<TL>), dim3((unsigned)VH, (unsigned)c.B), dim3((unsigned)(64 * p.waves)),
                           (unsigned)(p.waves * kQWaveBytes<TL>), s, c, out, q, lens, hd, (int32_t)H, scale_log2);
        return;
    }
    int64_t* before = reinterpret_cast<int64_t*>(ws);
    float* parts = ws + paged_before_floats(c.B);
    hipLaunchKernelGGL((k_attention_paged_q_split<TL>), dim3((unsigned)p.blocks), dim3(256), 0, s, c, out, q, lens, hd, (int32_t)H,
                       scale_log2, before, parts, VH);
    // waves of a merge block, if the sequences are alike: about 4 parts a group of lanes, or one where the rows are few (16
    // contexts of 4000 keys, 12 heads of 96, 15.9 -> 15.0 us; but a wave more for each of 7168 rows costs 2.7 us)
    const int64_t W = p.blocks * 4, parts_of = p.blocks / ((int64_t)VH * c.B);
    int64_t nw = 1;
    while (nw < 16 && nw * (256 / TL::D) * (nw * 2 * H * c.B <= 2048 ? 1 : 4) < parts_of) nw *= 2;
    hipLaunchKernelGGL((k_attention_paged_merge<typename TL::T, TL::D, true>), dim3((unsigned)H, (unsigned)c.B), dim3((unsigned)(64 * nw)), 0,
                       s, (int32_t)c.B, out, hd, (int32_t)H, before, parts, VH, (int32_t)W);
}

int launch_attention_paged_q(const AttnPagedPlan& p, const PagedQArgs& c, void* out, const void* q, const int32_t* lens, int64_t H,
                             float scale, float* ws, int dtype, void* stream)
{
    constexpr double most = std::numeric_limits<float>::max();
    const double log2_units = (double)scale * 1.4426950408889634;  // a finite scale stays finite
    const float sl = std::isfinite(scale) ? (float)std::clamp(log2_units, -most, most) : scale;
    auto run = [&](auto* t, auto d, auto ng, auto ngs) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int D = decltype(d)::value, NG = decltype(ng)::value, NGS = decltype(ngs)::value;
        auto go = [&](auto tl) {
            paged_q_go<decltype(tl)>(p, c, (T*)out, (const T*)q, lens, H, sl, ws, static_cast<hipStream_t>(stream));
        };
        c.kb == 4   ? go(PagedQTiles<T, D, NG, NGS, 4, 4>{})
        : c.vb == 4 ? go(PagedQTiles<T, D, NG, NGS, 8, 4>{})
                    : go(PagedQTiles<T, D, NG, NGS, 8, 8>{});
    };
    constexpr std::integral_constant<int, 1> n1{};
    constexpr std::integral_constant<int, 2> n2{};
    constexpr std::integral_constant<int, 3> n3{};
    constexpr std::integral_constant<int, 4> n4{};
    constexpr std::integral_constant<int, 64> d64{};
    constexpr std::integral_constant<int, 96> d96{};
    constexpr std::integral_constant<int, 128> d128{};
    auto columns2 = [&](auto* t, auto d, auto ng) { p.columns == 1 ? run(t, d, ng, n1) : run(t, d, ng, n2); };
    auto columns4 = [&](auto* t, auto d, auto ng) { p.columns == 4 ? run(t, d, ng, n4) : columns2(t, d, ng); };
    auto shape = [&](auto* t) {
        const int ng = c.D / c.group;
        if (c.D == 64) ng == 1 ? run(t, d64, n1, n1) : columns2(t, d64, n2);
        else if (c.D == 96) columns4(t, d96, n3);
        else ng == 1 ? run(t, d128, n1, n1) : ng == 2 ? columns2(t, d128, n2) : columns4(t, d128, n4);
    };
    dtype == VVH_F16 ? shape((f16*)nullptr) : shape((float*)nullptr);
    return (int)hipGetLastError();
}

}  // namespace vvh
