// Linears of 4-bit weights with group scales:
//   out[m][n] = sum_g s[n][g] sum_{k in g} (c[n][k] - z[n][g]) x[m][k] + bias[n] + res[m][n]
// with the codes c two to a byte, scales s in fp16 and zero points z bytes (8
// where there are none).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "device.h"

namespace vvh {

namespace {

// ---------------------------------------------------------------------------
// A wave owns a tile of 16 output channels and takes its weight rows 256 codes (one
// 128-byte line of each) a step; KS waves of a block share a tile's steps, their sums
// are added through LDS in order.  Up to 16 rows of x are a pass, staged in LDS.
//
// Loads: lane l reads the 16-byte piece l % 8 of the lines of rows l / 8 and 8 + l / 8, so
// that an instruction covers 8 whole lines, DEPTH steps ahead of use.  A step's 16 lines go
// through the wave's LDS tile, whose rows a lane reads back as the matrix instruction
// wants them: lane (n, g4) 8 codes of channel n, the four lanes of a channel 32 codes of one
// group, whose sum the instruction gives and the group's scale multiplies in fp32.
// Codes: a nibble in the low bits of an fp16 of exponent 2^10 is 1024 + c (in the second
// nibble 1024 + 16 c); one packed subtraction (or multiply-add by 1 / 16) leaves c - z, exactly.
// The dword of 8 codes gives them in the order 0 4 1 5 2 6 3 7, and x is staged in that order.
// fp32 rows of x are staged as two fp16 planes, high and low parts of x times a power of two that
// puts the step's largest |x| into [2^14, 2^15) (22 bits; the sum of a step is multiplied back).  Up to 8 such
// rows make 16 rows of the operand (FOLD): one instruction then takes both parts.
//
// One fp32 row of 151936 x 896 in groups of 32, 78 MB: 21.3 us, 3.65 TB/s; fp16 in groups of 128, 70 MB, 17.3, 4.1 TB/s; one
// fp16 row of 28672 x 8192, 121 MB, 29.4 us, 4.1 TB/s: bound by HBM and, beside it, the LDS round trips of the codes.  One fp16
// row of 896 x 896: 3.0 us, a launch and two round trips, which one of 17920 x 1536, 14.3 MB, has before and behind its stream:
// 6.3 us.  Rings of 3 and 4 steps: 24.2 and 25.9 us on the first, 28.7 and 28.1 on the third, 8 rows of 9728 x 896 4.8 -> 5.1 and
// 5.4.  Loading the codes straight into the instruction's
// layout (16 pieces of 64 bytes a load, dwords exchanged between lanes) instead of through LDS: 24 -> 29 us on the first.
// ---------------------------------------------------------------------------
constexpr int kQ4Step = 256;     // codes of a row a step
constexpr int kQ4WPitch = 144;   // bytes between rows of the LDS weight tile
constexpr int kQ4SPitch = 12;    // dwords between rows of its scales
constexpr int kQ4Tile = 16 * kQ4WPitch + 16 * kQ4SPitch * 4;
constexpr int kQ4Rows = 16;
constexpr int kQ4Batch = 8;      // pieces of x a wave loads at a time

// How a launch's blocks share out the work: block (slot, pass, split) takes the groups slot, slot +
// slots, ... of `tiles` tiles, 16 rows, and the steps [split * seg, + seg).  Blocks go to the 8 XCDs in
// turn and gridDim.x is a multiple of 8, so a tile's passes and splits are on one, whose L2 then has its weights.
struct Q4Launch {
    int32_t waves, tiles;  // of a block: waves a tile = waves / tiles = 1 << log_ks
    int32_t log_ks;
    int32_t seg;           // steps of a split, whose x is in LDS
    int32_t splits;        // > 1: raw sums to ws[split][M][N], for k_linear_q4_join
    int32_t groups_n, slots;
    int32_t rows;          // of x in LDS: the largest pass
    uint32_t inv_per;      // ceil(2^32 / units of a row of x in LDS)
    int32_t out_f16;
    float* ws;
};

__device__ __forceinline__ h2 q4_h2(uint32_t v) { return __builtin_bit_cast(h2, v); }

// The masks of the code conversion, kept in registers: v_and_or_b32 takes no literal.
struct Q4Masks {
    uint32_t lo, hi, one;
};
__device__ __forceinline__ Q4Masks q4_masks()
{
    Q4Masks k{0x000F000Fu, 0x00F000F0u, 0x64006400u};
    asm("" : "+s"(k.lo), "+s"(k.hi), "+v"(k.one));
    return k;
}
// 8 codes minus their zero point; zl = 1024 + z, zh = 64 + z
__device__ __forceinline__ h8 q4_codes(uint32_t w, h2 zl, h2 zh, const Q4Masks& k)
{
    const h2 sixteenth = {(f16)0.0625f, (f16)0.0625f};
    const uint32_t v = w >> 8;
    const h2 a = q4_h2((w & k.lo) | k.one) - zl;
    const h2 b = __builtin_elementwise_fma(q4_h2((w & k.hi) | k.one), sixteenth, -zh);
    const h2 c = q4_h2((v & k.lo) | k.one) - zl;
    const h2 d = __builtin_elementwise_fma(q4_h2((v & k.hi) | k.one), sixteenth, -zh);
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A wave's stream of a tile's weights: 16 channels from n0 on, a step at a time from memory to registers (issue),
// to its LDS tile (put) and through the matrix instruction (step).
template <int G, bool ZP>
struct Q4Stream {
    static constexpr int PG = kQ4Step / G;          // groups a step
    static constexpr int NS = PG > 4 ? 2 : 1;       // scales a lane loads a step
    static constexpr int DW = G / 32;               // dwords of codes a lane reads a group
    static constexpr int loads = 2 + NS * (ZP ? 2 : 1);  // of a step
    struct Slot {
        u4 a, b;
        uint16_t s[NS];
        uint8_t z[NS];
    };
    const uint8_t *wa, *wb, *zp;
    const uint16_t* sc;
    int32_t K, steps, groups;
    int lane, n, g4;
    char* tile;
    uint32_t* stile;
    Q4Masks masks;

    __device__ __forceinline__ Q4Stream(const Q4Args& a, char* lds, int l)
        : zp(nullptr), K((int32_t)a.K), steps((K + kQ4Step - 1) / kQ4Step), groups(K / G), lane(l), n(l & 15), g4(l >> 4),
          tile(lds), stile(reinterpret_cast<uint32_t*>(lds + 16 * kQ4WPitch)), masks(q4_masks())
    {
    }
    // rows past N are row N - 1, pieces past K the last one (met by zeros in x)
    __device__ __forceinline__ void point(const Q4Args& a, int64_t n0)
    {
        const int64_t last = a.N - 1, ra = n0 + (lane >> 3), rb = ra + 8, rn = n0 + n;
        wa = a.w + (ra < last ? ra : last) * (K / 2);
        wb = a.w + (rb < last ? rb : last) * (K / 2);
        sc = a.scales + (rn < last ? rn : last) * groups;
        if (ZP) zp = a.zeros + (rn < last ? rn : last) * groups;
    }
    __device__ __forceinline__ void issue(Slot& r, int32_t want) const
    {
        const int32_t st = want < steps ? want : steps - 1;  // past the end: never used
        const int32_t at = st * (kQ4Step / 2) + (lane & 7) * 16, last = K / 2 - 16;
        r.a = *reinterpret_cast<const u4*>(wa + (at < last ? at : last));
        r.b = *reinterpret_cast<const u4*>(wb + (at < last ? at : last));
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const int32_t h = st * PG + (g4 * NS + i) % PG, g = h < groups ? h : groups - 1;
            r.s[i] = sc[g];
            if (ZP) r.z[i] = zp[g];
        }
    }
    // st: the step in the slot (a group past the row's end has no sum; its scale, the last group's, may be infinite)
    __device__ __forceinline__ void put(const Slot& r, int32_t st) const
    {
        wave_lds_order();  // after the reads of the step before
        *reinterpret_cast<u4*>(tile + (lane >> 3) * kQ4WPitch + (lane & 7) * 16) = r.a;
        *reinterpret_cast<u4*>(tile + (8 + (lane >> 3)) * kQ4WPitch + (lane & 7) * 16) = r.b;
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const int g = (g4 * NS + i) % PG;  // two lanes the same where there are fewer groups
            uint32_t v = st * PG + g < groups ? r.s[i] : 0;
            if (ZP) v |= (uint32_t)__builtin_bit_cast(uint16_t, (f16)(float)r.z[i]) << 16;
            stile[n * kQ4SPitch + g] = v;
        }
        wave_lds_order();
    }
    // part[r] += the step's sums; xk: the step's x, whose operand rows are at row[r], TWO: and row[r] + plane; FOLD: the two
    // parts of a row are neighbouring rows of the operand, added before the scale
    template <int RT, bool TWO, bool FOLD>
    __device__ __forceinline__ void step(f4 (&part)[RT], const f16* xk, const int32_t (&row)[RT], int32_t plane) const
    {
        uint32_t sv[PG];
#pragma unroll
        for (int g = 0; g < PG; g++) sv[g] = stile[n * kQ4SPitch + g];
#pragma unroll
        for (int g = 0; g < PG; g++) {
            uint32_t w[DW];
            const uint32_t* wr = reinterpret_cast<const uint32_t*>(tile + n * kQ4WPitch) + g * (G / 8) + g4 * DW;
#pragma unroll
            for (int j = 0; j < DW; j++) w[j] = wr[j];
            h2 zl = {(f16)1032.0f, (f16)1032.0f}, zh = {(f16)72.0f, (f16)72.0f};
            if (ZP) {
                const f16 z = q4_h2(sv[g])[1];
                zl = h2{z, z} + h2{(f16)1024.0f, (f16)1024.0f};
                zh = h2{z, z} + h2{(f16)64.0f, (f16)64.0f};
            }
            f4 d[RT] = {};
#pragma unroll
            for (int j = 0; j < DW; j++) {
                const h8 b = q4_codes(w[j], zl, zh, masks);
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    const f16* xp = xk + row[r] + g * G + (g4 * DW + j) * 8;
                    if (TWO) d[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const h8*>(xp + plane), b, d[r], 0, 0, 0);
                    d[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const h8*>(xp), b, d[r], 0, 0, 0);
                }
            }
            const float s = (float)q4_h2(sv[g])[0];
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int i = 0; i < (FOLD ? 2 : 4); i++)
                    part[r][i] = __builtin_fmaf(s, FOLD ? d[r][2 * i] + d[r][2 * i + 1] : d[r][i], part[r][i]);
            // not all of a step's reads at once: registers
            if ((g + 1) % (PG / 2) == 0) __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// bias, residual and rounding of one output
__device__ __forceinline__ void q4_store(const Q4Args& a, bool out_f16, int64_t o, float y)
{
    if (out_f16) {
        if (a.res) y += (float)((const f16*)a.res)[o];
        ((f16*)a.out)[o] = (f16)y;
    } else {
        if (a.res) y += ((const float*)a.res)[o];
        ((float*)a.out)[o] = y;
    }
}

// Channel n's bias, 0 without one: no branch, so that the loads in flight around it are still counted.  (x is 16-byte
// aligned and has a group of 32 values at least.)
__device__ __forceinline__ float q4_bias(const Q4Args& a, int64_t n)
{
    const float b = *(a.bias ? a.bias + (n < a.N ? n : a.N - 1) : (const float*)a.inp);
    return a.bias ? b : 0.0f;
}

// 8 values in the order of the codes: 0 1 2 3 4 5 6 7 -> 0 4 1 5 2 6 3 7
__device__ __forceinline__ u4 q4_order(u4 v)
{
    return u4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
              __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
}

// A wave's 256 values of a row, 4 a lane, as their fp16 parts, in the order of the codes, and their inverse scale.
__device__ __forceinline__ void q4_split(f4 v, int lane, f16* hi_row, f16* lo_row, float* inv)
{
    const float most = group_max(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))), 64);
    // 2^(14 - x) for most in [2^x, 2^(x + 1)), at most 2^126; with an infinity that of the largest finite ones
    const int b = (int)(__builtin_bit_cast(uint32_t, most) >> 23), e = b < 15 ? 15 : b > 254 ? 254 : b;
    const float up = __builtin_bit_cast(float, (uint32_t)(268 - e) << 23);
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int c = 0; c < 2; c++) {
        const float p = v[2 * c] * up, q = v[2 * c + 1] * up;
        const h2 h = {(f16)p, (f16)q};
        h2 l = {(f16)(p - (float)h[0]), (f16)(q - (float)h[1])};
        if (b == 255) l = h2{};  // an infinity is all in its high part
        hi[c] = __builtin_bit_cast(uint32_t, h);
        lo[c] = __builtin_bit_cast(uint32_t, l);
    }
    // lanes of a pair hold values 0-3 and 4-7: the even one stores the high parts, the odd one the low
    const bool odd = lane & 1;
    const uint32_t s0 = odd ? hi[0] : lo[0], s1 = odd ? hi[1] : lo[1];
    const uint32_t r0 = __builtin_amdgcn_mov_dpp((int)s0, 0xB1, 0xF, 0xF, false);
    const uint32_t r1 = __builtin_amdgcn_mov_dpp((int)s1, 0xB1, 0xF, 0xF, false);
    const u4 o = q4_order(odd ? u4{r0, r1, lo[0], lo[1]} : u4{hi[0], hi[1], r0, r1});
    *reinterpret_cast<u4*>((odd ? lo_row : hi_row) + (lane >> 1) * 8) = o;
    *inv = __builtin_bit_cast(float, (uint32_t)(e - 14) << 23);  // every lane the same: no branch
}

template <typename AT, int G, bool ZP, int DEPTH, bool FOLD>
__global__ __launch_bounds__(512) void k_linear_q4(Q4Args a, Q4Launch L)
{
    constexpr bool F32 = sizeof(AT) == 4;
    constexpr int OUT = FOLD ? 2 : 4;               // rows of a lane's sums
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), threads = L.waves * 64;
    const int32_t slot = blockIdx.x, pass = blockIdx.y, split = blockIdx.z;
    if (slot >= L.slots) return;
    const int32_t KS = 1 << L.log_ks, ks = wave & (KS - 1), mytile = wave >> L.log_ks;
    const int64_t m0 = (int64_t)pass * kQ4Rows;
    const int32_t rows = (int32_t)(a.M - m0 < kQ4Rows ? a.M - m0 : kQ4Rows);
    const int32_t K = (int32_t)a.K, steps = (K + kQ4Step - 1) / kQ4Step;
    const int32_t s0 = split * L.seg, s1 = s0 + L.seg < steps ? s0 + L.seg : steps;
    const int32_t mine = (s1 - s0 - ks + KS - 1) >> L.log_ks;   // steps s0 + ks + KS i of every tile are the wave's
    const int32_t turns = mine > DEPTH ? (mine + DEPTH - 1) / DEPTH * DEPTH : DEPTH;  // whole rings, one at least
    const int32_t pitch = L.seg * kQ4Step + 8;      // halves between rows of x in LDS
    f16* xs = reinterpret_cast<f16*>(smem);
    const int32_t plane = L.rows * pitch;           // F32: the low parts' plane is at +plane
    float* xinv = reinterpret_cast<float*>(xs + (F32 ? 2 : 1) * plane);  // F32: [seg][16] inverse scales
    char* tile = reinterpret_cast<char*>(xinv + (F32 ? L.seg * kQ4Rows : 0)) + wave * kQ4Tile;
    const AT* x = (const AT*)a.inp + m0 * a.K;

    Q4Stream<G, ZP> ws(a, tile, lane);
    typename Q4Stream<G, ZP>::Slot ring[DEPTH];
    auto first_channel = [&](int32_t grp) { return ((int64_t)grp * L.tiles + mytile) * 16; };
    auto issue = [&](int u, int32_t i) { ws.issue(ring[u], s0 + ks + (i << L.log_ks)); };

    // ---- x ----
    const int32_t arow = FOLD ? n >> 1 : n, row = arow < rows ? arow : rows - 1;  // past the last: computed and dropped
    // x to LDS.  A unit is 16 bytes of a row: unit i is piece i % per of row i / per (fp32: a wave's unit, 256
    // values of a row, 4 a lane, whose largest the lanes share).  kQ4Batch of them are loaded together; the
    // first batch ahead of the weight ring, whose loads it then does not wait for.
    constexpr int PIECE = F32 ? kQ4Step : 8;            // values a unit
    const int32_t first = F32 ? wave : tid, stride = F32 ? L.waves : threads;
    const int32_t per = L.seg * (kQ4Step / PIECE);
    u4 xr[kQ4Batch];
    auto load_x = [&](int32_t i0) {
#pragma unroll
        for (int j = 0; j < kQ4Batch; j++) {
            const int32_t i = i0 + j * stride;
            if ((F32 ? i : i - first) >= rows * per) break;
            const int32_t m = (int32_t)__umulhi((uint32_t)i, L.inv_per), at = s0 * kQ4Step + (i - m * per) * PIECE + (F32 ? lane * 4 : 0);
            xr[j] = u4{};
            if (m < rows && at < K) xr[j] = *reinterpret_cast<const u4*>(x + (int64_t)m * K + at);
        }
    };
    auto store_x = [&](int32_t i0) {
#pragma unroll
        for (int j = 0; j < kQ4Batch; j++) {
            const int32_t i = i0 + j * stride;
            if ((F32 ? i : i - first) >= rows * per) break;
            const int32_t m = (int32_t)__umulhi((uint32_t)i, L.inv_per), k = (i - m * per) * PIECE;
            if constexpr (!F32) {
                if (m < rows) *reinterpret_cast<u4*>(xs + m * pitch + k) = q4_order(xr[j]);
            } else {
                f16* to = xs + m * pitch + k;
                q4_split(__builtin_bit_cast(f4, xr[j]), lane, to, to + plane, xinv + k / kQ4Step * kQ4Rows + m);
            }
        }
    };
    f4 acc;
    // step i of the wave (last: of the last ring, which may be past its end and then adds nothing)
    auto consume = [&](int u, int32_t i, bool last) {
        const bool is = !last || i < mine;
        const int32_t st = is ? ks + (i << L.log_ks) : 0;  // within x in LDS
        ws.put(ring[u], s0 + st);
        f4 parts[1] = {};
        const int32_t at[1] = {(FOLD && n & 1 ? plane : 0) + row * pitch};
        ws.template step<1, F32 && !FOLD, FOLD>(parts, xs + st * kQ4Step, at, plane);
        const f4 part = parts[0];
        f4 to = acc;
        if constexpr (FOLD) {
            const float* inv = xinv + st * kQ4Rows + 2 * g4;
#pragma unroll
            for (int j = 0; j < 2; j++) to[j] = __builtin_fmaf(part[j], inv[j], acc[j]);
        } else if constexpr (F32) {
            const f4 inv = *reinterpret_cast<const f4*>(xinv + st * kQ4Rows + 4 * g4);  // rows past the last: dropped
#pragma unroll
            for (int j = 0; j < 4; j++) to[j] = __builtin_fmaf(part[j], inv[j], acc[j]);
        } else {
            to = acc + part;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) acc[j] = is ? to[j] : acc[j];
    };

    load_x(first);
    float bias = q4_bias(a, first_channel(slot) + n), bias_next = 0.0f;
    ws.point(a, first_channel(slot));
#pragma unroll
    for (int u = 0; u < DEPTH; u++) issue(u, u);
    store_x(first);
    // Waits that are there anyway, said once more where every path has had them: x's registers are free, the ring still on
    // its way
    wait_loads<DEPTH * Q4Stream<G, ZP>::loads>();
    for (int32_t i = kQ4Batch * stride; i < rows * per; i += kQ4Batch * stride) {
        load_x(first + i);
        store_x(first + i);
        wait_loads<0>();
    }
    lds_barrier();
    for (int32_t grp = slot;; grp += L.slots) {
        const bool next = grp + L.slots < L.groups_n;
        acc = f4{};
        // The ring is refilled with this tile's steps, at their end with the next tile's first ones (no work of a step ahead
        // of the one before it: registers).  No branch around its loads but the last: waits count what is in flight.
        int32_t i = 0;
        for (; i + DEPTH < turns; i += DEPTH)
#pragma unroll
            for (int u = 0; u < DEPTH; u++) {
                consume(u, i + u, false);
                __builtin_amdgcn_sched_barrier(0);
                issue(u, i + u + DEPTH);
            }
        if (next) {
            bias_next = q4_bias(a, first_channel(grp + L.slots) + n);
            ws.point(a, first_channel(grp + L.slots));
#pragma unroll
            for (int u = 0; u < DEPTH; u++) {
                consume(u, i + u, true);
                __builtin_amdgcn_sched_barrier(0);
                issue(u, u);
            }
        } else {
#pragma unroll
            for (int u = 0; u < DEPTH; u++) {
                if (u > 0 && i + u >= mine) break;  // no loads follow
                consume(u, i + u, u == 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // the sums of the tile's waves, through their weight tiles
        if (KS > 1) {
            wave_lds_order();
            *reinterpret_cast<f4*>(tile + lane * 16) = acc;
            lds_barrier();
            if (ks == 0)
                for (int i = 1; i < KS; i++) acc += *reinterpret_cast<const f4*>(tile + i * kQ4Tile + lane * 16);
            if (next) lds_barrier();  // read before the next tile's weights
        }
        const int64_t n1 = first_channel(grp) + n;
        if (ks == 0 && n1 < a.N) {
#pragma unroll
            for (int i = 0; i < OUT; i++) {
                if (OUT * g4 + i >= rows) break;
                const int64_t o = (m0 + OUT * g4 + i) * a.N + n1;
                if (L.splits > 1) L.ws[(int64_t)split * a.M * a.N + o] = acc[i];
                else q4_store(a, L.out_f16, o, acc[i] + bias);
            }
        }
        if (!next) break;
        bias = bias_next;
    }
}

// Many rows over many channels: a block takes 8 tiles, a wave each, and up to 16 RT rows, and x goes through LDS a step
// at a time: two buffers, the next step's x on its way from memory while the waves work on this one, a barrier a step.
// A wave's codes meet RT operands of x.  Against the kernel above, which needs all of x before it begins: 13 rows of 17920 x
// 1536 9.0 -> 8.0 us, 32 13.2 -> 10.0, 64 18.2 -> 14.8 (fp32 32.7 -> 26.5), 64 rows of 151936 x 896 69.9 -> 52; up to 4 rows
// it is slower (1 of 28672 x 8192 31 -> 38), and with few blocks (76: 8 rows of 9728 x 896 4.7 -> 5.6).  The steps' latency
// bounds it (13 rows: 14.9 MB, 1.9 TB/s), and from 32 rows on the LDS reads of x, 8 KB for 16 rows and a step of a wave.
// Nothing in the loop branches on a lane: a branch costs 50 registers here, and waits past it take every load for pending.
template <typename AT, int G, bool ZP, int RT>
__global__ __launch_bounds__(512) void k_linear_q4_rows(Q4Args a, int32_t pass_rows, int32_t groups_n, int32_t out_f16, int32_t seg,
                                                        float* __restrict__ parts)
{
    constexpr bool F32 = sizeof(AT) == 4;
    constexpr int R = 16 * RT, PITCH = kQ4Step + 8, NX = F32 ? 2 * RT : RT, PLANE = R * PITCH, BUF = (F32 ? 2 : 1) * PLANE;
    constexpr int DEPTH = 2;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int32_t grp = blockIdx.x;
    if (grp >= groups_n) return;
    const int64_t m0 = (int64_t)blockIdx.y * pass_rows, n0 = ((int64_t)grp * 8 + wave) * 16;
    const int32_t rows = (int32_t)(a.M - m0 < pass_rows ? a.M - m0 : pass_rows), K = (int32_t)a.K;
    f16* xs = reinterpret_cast<f16*>(smem);                        // [2][planes][R][PITCH]
    float* xinv = reinterpret_cast<float*>(xs + 2 * BUF);          // F32: [2][R]
    Q4Stream<G, ZP> ws(a, reinterpret_cast<char*>(xinv + (F32 ? 2 * R : 0)) + wave * kQ4Tile, lane);
    typename Q4Stream<G, ZP>::Slot ring[DEPTH];
    const int32_t s0 = blockIdx.z * seg, s1 = s0 + seg < ws.steps ? s0 + seg : ws.steps;  // the split's steps
    const AT* x = (const AT*)a.inp + m0 * a.K;
    const int32_t xrow = F32 ? wave : tid >> 5, xat = F32 ? lane * 4 : (tid & 31) * 8;
    constexpr int XROWS = F32 ? 8 : 16;  // rows the block loads at a time
    u4 xr[NX];  // x of the next step
    // rows past the last are the last, values past K the row's last ones, stored as 0 (no branch around the loads, so that
    // waits count what is in flight)
    constexpr int XV = 16 / (int)sizeof(AT);  // values a load
    auto load_x = [&](int32_t st) {
        const int32_t at = st * kQ4Step + xat;
#pragma unroll
        for (int j = 0; j < NX; j++) {
            const int32_t m = xrow + XROWS * j;
            xr[j] = *reinterpret_cast<const u4*>(x + (int64_t)(m < rows ? m : rows - 1) * K + (at < K ? at : K - XV));
        }
    };
    auto store_x = [&](int32_t st, int buf) {
        const bool is = st * kQ4Step + xat < K;
#pragma unroll
        for (int j = 0; j < NX; j++) {
            const int32_t m = xrow + XROWS * j;
            f16* to = xs + buf * BUF + m * PITCH;
            const u4 v = is ? xr[j] : u4{};
            if constexpr (F32) q4_split(__builtin_bit_cast(f4, v), lane, to, to + PLANE, xinv + buf * R + m);
            else *reinterpret_cast<u4*>(to + xat) = q4_order(v);
        }
    };
    int32_t row[RT];                                // rows of the operand past the last are computed and dropped
#pragma unroll
    for (int r = 0; r < RT; r++) row[r] = (r * 16 + n < rows ? r * 16 + n : rows - 1) * PITCH;

    f4 acc[RT] = {};
    auto consume = [&](int u, int32_t st) {
        const int buf = u & 1;
        ws.put(ring[u], st);
        if constexpr (F32) {
            f4 part[RT] = {};
            ws.template step<RT, true, false>(part, xs + buf * BUF, row, PLANE);
#pragma unroll
            for (int r = 0; r < RT; r++) {
                const f4 inv = *reinterpret_cast<const f4*>(xinv + buf * R + r * 16 + 4 * g4);  // rows past the last: dropped
#pragma unroll
                for (int i = 0; i < 4; i++) acc[r][i] = __builtin_fmaf(part[r][i], inv[i], acc[r][i]);
            }
        } else {
            ws.template step<RT, false, false>(acc, xs + buf * BUF, row, PLANE);
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    load_x(s0);
    const float bias = q4_bias(a, n0 + n);
    ws.point(a, n0);
    ws.issue(ring[0], s0);
    store_x(s0, 0);
    load_x(s0 + 1);
    ws.issue(ring[1], s0 + 1);
    lds_barrier();
    int32_t st = s0;
    for (; st + DEPTH < s1; st += DEPTH)
#pragma unroll
        for (int u = 0; u < DEPTH; u++) {
            consume(u, st + u);
            ws.issue(ring[u], st + u + DEPTH);
            store_x(st + u + 1, (u + 1) & 1);
            load_x(st + u + 2);
            lds_barrier();
        }
#pragma unroll
    for (int u = 0; u < DEPTH; u++) {
        if (st + u >= s1) break;
        consume(u, st + u);
        if (st + u + 1 < s1) {
            store_x(st + u + 1, (u + 1) & 1);
            lds_barrier();
        }
    }
    if (n0 + n >= a.N) return;
#pragma unroll
    for (int e = 0; e < 4 * RT; e++) {
        const int m = e / 4 * 16 + 4 * g4 + e % 4;
        if (m >= rows) break;
        const int64_t o = (m0 + m) * a.N + n0 + n;
        if (parts) parts[blockIdx.z * a.M * a.N + o] = acc[e / 4][e % 4];  // for k_linear_q4_join
        else q4_store(a, out_f16, o, acc[e / 4][e % 4] + bias);
    }
}

// The sums of the splits, in order, then bias and residual; also K = 0 (no splits).
template <typename OT>
__global__ __launch_bounds__(256) void k_linear_q4_join(Q4Args a, const float* __restrict__ ws, int32_t splits)
{
    const int64_t all = a.M * a.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        float y = 0.0f;
#pragma unroll 4
        for (int32_t s = 0; s < splits; s++) y += ws[s * all + i];
        y += a.bias ? a.bias[i % a.N] : 0.0f;
        ((OT*)a.out)[i] = (OT)(y + (a.res ? (float)((const OT*)a.res)[i] : 0.0f));
    }
}

constexpr int64_t kQ4Lds = 160 * 1024;

int64_t q4_lds(const Q4Plan& p, int64_t rows, bool f32)
{
    return (f32 ? 2 : 1) * rows * (p.seg * kQ4Step + 8) * 2 + (f32 ? p.seg * kQ4Rows * 4 : 0) +
           p.waves * kQ4Tile;
}

}  // namespace

Q4Plan linear_q4_plan(const Q4Args& a, int act, int64_t cus)
{
    const bool f32 = act == VVH_F32;
    const int64_t tiles = (a.N + 15) / 16, steps = (a.K + kQ4Step - 1) / kQ4Step, passes = (a.M + kQ4Rows - 1) / kQ4Rows,
                  rows = std::min<int64_t>(a.M, kQ4Rows);
    Q4Plan p{};
    if (steps == 0) return p;
    // x a step at a time, passes of `most` rows, `parts` shares of k
    const int64_t groups = (a.N + 127) / 128, n16 = (a.M + 15) / 16, n32 = (a.M + 31) / 32;
    auto stepwise = [&](int64_t most, int64_t parts) {
        const int64_t n = (a.M + most - 1) / most;
        p.rows = (a.M + n - 1) / n;
        p.seg = (steps + parts - 1) / parts;
        p.splits = (steps + p.seg - 1) / p.seg;
        p.ws_floats = p.splits > 1 ? p.splits * a.M * a.N : 0;
        return p;
    };
    // 5 / 8 of a device of blocks, and at most 12 parts to join
    const int64_t parts = std::min<int64_t>({(cus * 5 / 8 + groups * n16 - 1) / (groups * n16), 12, steps});
    // where the blocks of 8 tiles fill half the device and there are rows to share the codes
    if (a.M > (f32 ? 8 : 4) && groups * n16 >= cus / 2) {
        // k in two from 12 steps on, where the second launch is made up for: 16 rows of 16384 channels, whole and shared, 6 steps 7.5
        // and 8.9 us, 11 steps 11.15 and 11.27, 14 steps 13.1 and 11.9, 20 steps 17.6 and 14.1; 64 rows of 4000 the same but 11 steps
        // 11.0 and 10.7
        if (parts > 1 && steps >= 12) return stepwise(16, parts);
        // passes of 16 or 32 rows, by the blocks a CU takes and what these cost (17920 x 1536: 1, 2, 3 of 16 rows 8.0, 11.7,
        // 15.5 us; 1, 2 of 32 rows 9.3, 14.7); fp32 x of 32 rows leaves a CU one block (19.6 us, of 16 18.6)
        const int64_t c16 = (groups * n16 + cus - 1) / cus, c32 = (groups * n32 + cus - 1) / cus;
        return stepwise(!f32 && 7 * c32 < 5 * c16 ? 32 : 16, 1);
    }
    p.splits = 1;
    p.ks = 1;
    p.waves = 8;
    p.seg = std::max<int64_t>(2, steps);
    // 5 to 16 fp32 rows up to 96 KB: a block that needs more has a CU for itself (16 rows of 1536 x 1536, 121 KB, 9.1 us, a step at a
    // time 6.8); below it whole is faster for most (6 rows of 1536 x 1792, 67 KB, 5.7 and 6.8; 16 of 1536 x 768, 73 KB, 6.3 and 6.7;
    // 16 of 1536 x 1024, 89 KB, 7.0 and 6.2)
    const int64_t most = f32 && rows > 4 ? 96 * 1024 : kQ4Lds;
    while (q4_lds(p, rows, f32) > most) {
        p.splits++;
        p.seg = std::max<int64_t>(2, (steps + p.splits - 1) / p.splits);
    }
    // where x does not fit (16 rows of 1536 x 8960 10.7 -> 8.7 us, 64 18.1 -> 13.7; fp32 17 rows of 1536 x 1536 8.6 -> 7.0); x that
    // fits stays whole (17 rows of 4000 x 4096 9.0, in 3 shares 10.7)
    if (a.M > 4 && p.splits > 1) return stepwise(16, parts);
    while (p.ks < 8 && p.ks < p.seg && tiles * passes * p.splits * p.ks < (rows > 4 ? 4 : 8) * cus) p.ks *= 2;
    p.waves = rows > 4 ? 8 : std::max<int64_t>(4, p.ks);
    p.splits = (steps + p.seg - 1) / p.seg;
    p.ws_floats = p.splits > 1 ? p.splits * a.M * a.N : 0;
    return p;
}

int launch_linear_q4(const Q4Plan& p, const Q4Args& a, int act, int out, float* ws, int64_t cus, void* stream)
{
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool f32 = act == VVH_F32;
    if (p.rows > 0) {
        const int64_t groups = (a.N + 127) / 128, rt = (p.rows + 15) / 16, planes = f32 ? 2 : 1;
        const int64_t lds = 2 * planes * rt * 16 * (kQ4Step + 8) * 2 + (f32 ? 2 * rt * 16 * 4 : 0) + 8 * kQ4Tile;
        const dim3 grid((unsigned)((groups + 7) / 8 * 8), (unsigned)((a.M + p.rows - 1) / p.rows), (unsigned)p.splits);
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, grid, dim3(512), (size_t)lds, st, a, (int32_t)p.rows, (int32_t)groups, (int32_t)(out == VVH_F16),
                               (int32_t)p.seg, p.splits > 1 ? ws : nullptr);
        };
        auto go_rt = [&](auto* t, auto z, auto g) {
            using AT = std::remove_pointer_t<decltype(t)>;
            constexpr bool ZP = decltype(z)::value;
            constexpr int G = decltype(g)::value;
            if constexpr (sizeof(AT) == 2) {
                if (rt == 2) return go(k_linear_q4_rows<AT, G, ZP, 2>);
            }
            go(k_linear_q4_rows<AT, G, ZP, 1>);
        };
        auto go_group = [&](auto* t, auto z) {
            if (a.group == 32) go_rt(t, z, std::integral_constant<int, 32>{});
            else if (a.group == 64) go_rt(t, z, std::integral_constant<int, 64>{});
            else go_rt(t, z, std::integral_constant<int, 128>{});
        };
        auto go_type = [&](auto* t) { a.zeros ? go_group(t, std::true_type{}) : go_group(t, std::false_type{}); };
        f32 ? go_type((float*)nullptr) : go_type((f16*)nullptr);
    } else if (p.splits > 0) {
        const int64_t tiles = (a.N + 15) / 16, passes = (a.M + kQ4Rows - 1) / kQ4Rows, rows = std::min<int64_t>(a.M, kQ4Rows);
        const int64_t per = p.seg * (f32 ? 1 : kQ4Step / 8), lds = q4_lds(p, rows, f32);
        const int64_t tpb = p.waves / p.ks, groups = (tiles + tpb - 1) / tpb;
        // Blocks of a group are enough where x costs little to stage; else a block takes several groups with the
        // x it has, while the blocks still fill the device
        const int64_t fit = std::max<int64_t>(1, std::min(kQ4Lds / lds, 32 / p.waves));
        const int64_t worth = (rows * (f32 ? 4 : 2) + tpb - 1) / tpb, full = groups * passes * p.splits / (fit * cus);
        const int64_t turns = std::max<int64_t>(1, std::min(worth, full)), slots = (groups + turns - 1) / turns;
        const dim3 grid((unsigned)((slots + 7) / 8 * 8), (unsigned)passes, (unsigned)p.splits);
        Q4Launch L{(int32_t)p.waves, (int32_t)tpb, 0, (int32_t)p.seg, (int32_t)p.splits, (int32_t)groups, (int32_t)slots, (int32_t)rows,
                   (uint32_t)(((uint64_t(1) << 32) + per - 1) / per), out == VVH_F16, ws};
        while ((1 << L.log_ks) < p.ks) L.log_ks++;
        const bool one = (p.seg + p.ks - 1) / p.ks == 1 && turns == 1;  // a single step a wave
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, grid, dim3((unsigned)(64 * p.waves)), (size_t)lds, st, a, L);
        };
        auto go_fold = [&](auto* t, auto z, auto g, auto depth) {
            using AT = std::remove_pointer_t<decltype(t)>;
            constexpr bool ZP = decltype(z)::value;
            constexpr int G = decltype(g)::value, DEPTH = decltype(depth)::value;
            if constexpr (sizeof(AT) == 4) {
                if (rows <= 8) return go(k_linear_q4<AT, G, ZP, DEPTH, true>);
            }
            go(k_linear_q4<AT, G, ZP, DEPTH, false>);
        };
        auto go_depth = [&](auto* t, auto z, auto g) {
            one ? go_fold(t, z, g, std::integral_constant<int, 1>{}) : go_fold(t, z, g, std::integral_constant<int, 2>{});
        };
        auto go_group = [&](auto* t, auto z) {
            if (a.group == 32) go_depth(t, z, std::integral_constant<int, 32>{});
            else if (a.group == 64) go_depth(t, z, std::integral_constant<int, 64>{});
            else go_depth(t, z, std::integral_constant<int, 128>{});
        };
        auto go_type = [&](auto* t) { a.zeros ? go_group(t, std::true_type{}) : go_group(t, std::false_type{}); };
        f32 ? go_type((float*)nullptr) : go_type((f16*)nullptr);
    }
    if (p.splits != 1) {
        const dim3 grid((unsigned)std::min<int64_t>((a.M * a.N + 255) / 256, 65536));
        if (out == VVH_F16) hipLaunchKernelGGL(k_linear_q4_join<f16>, grid, dim3(256), 0, st, a, ws, (int32_t)p.splits);
        else hipLaunchKernelGGL(k_linear_q4_join<float>, grid, dim3(256), 0, st, a, ws, (int32_t)p.splits);
    }
    return (int)hipGetLastError();
}

}  // namespace vvh
