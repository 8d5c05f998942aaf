// attention.hip — attention over whole packed sequences with grouped heads and a relative position bias learned by buckets:
// mi_attention_dev and mi_attention_backward_dev (include/mi355rag.h has the formulas).
//
// All products are 32x32x16 MFMAs on 16-bit operands with fp32 accumulators, in the form that puts ONE row of the softmax on a
// lane: S^T = K Q^T has keys on the accumulator rows and the query on the lane, so maximum and sum over keys are in-register
// work, and the bf16 / fp16 P^T that falls out of the accumulators is, register for register, the B operand of O^T = V^T P^T
// (accumulator row 8 g + 4 h + i of lane half h is operand element k = 4 (g & 1) + i of 16-key step g >> 1; the V^T operand is
// read with the same permutation of keys by the hardware transpose read, so no value crosses a lane).
#include <float.h>
#include <math.h>
#include <atomic>
#include "attention.h"
#include "kernels.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short tr4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) tr4_t tr4_lds_t;

#define AT_LOG2E 1.4426950408889634f
#define AT_LN2 0.6931471805599453f
#define AT_KT 64                       // rows of the staged operand per tile

template <bool F16> __device__ __forceinline__ f32x16 at_mfma(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// two fp32 values, each rounded to nearest even
template <bool F16> __device__ __forceinline__ uint32_t at_pack2(float lo, float hi)
{
    if constexpr (F16) {
        f16x2 v;
        v[0] = (_Float16)lo;
        v[1] = (_Float16)hi;
        return __builtin_bit_cast(uint32_t, v);
    } else {
        bf16x2 v;
        v[0] = (__bf16)lo;
        v[1] = (__bf16)hi;
        return __builtin_bit_cast(uint32_t, v);
    }
}
__device__ __forceinline__ float at_max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// the two 16-bit values of a word
template <bool F16> __device__ __forceinline__ float at_lo(uint32_t w)
{
    if constexpr (F16) return (float)__builtin_bit_cast(f16x2, w)[0];
    else return __builtin_bit_cast(float, w << 16);
}
template <bool F16> __device__ __forceinline__ float at_hi(uint32_t w)
{
    if constexpr (F16) return (float)__builtin_bit_cast(f16x2, w)[1];
    else return __builtin_bit_cast(float, w & 0xFFFF0000u);
}
// the value of the same lane in the other half of the wave
__device__ __forceinline__ float at_other_half(float x) { return __shfl_xor(x, 32, 64); }
__device__ __forceinline__ f32x16 at_zero16()
{
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.0f;
    return z;
}

// ---------------------------------------------------------------- work items
// Blocks go to the 8 XCDs round robin by their linear id, and each XCD has its own L2.  A unit is a head, or, where the heads
// are no multiple of 8, every parts-th tile of a head; an XCD owns units_per_xcd consecutive units, so the query heads of one key
// head read its K and V through one L2, and every XCD has the same mix of tiles (a causal sequence's last tiles are its longest).
__device__ __forceinline__ bool at_work(const mi_attn_args& p, int& head, int& t)
{
    const int xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
    const int u = xcd * p.units_per_xcd + idx / p.tiles_per_unit;
    head = u / p.parts;
    t = (idx % p.tiles_per_unit) * p.parts + u % p.parts;
    return t < p.tiles;
}

// Tile t of the token axis -> sequence and tile of it.  Tiles of sequence i start at offsets[i] / BM + i: an upper bound of the
// tiles before it that needs no prefix sum; the surplus finds no rows.  64 lanes probe 64 sequences at a time.  With zero_tail
// the rows behind the last sequence are one more "sequence" (tail = true).  Offsets are clamped to [0, tokens], so whatever
// they hold, start and len stay inside the tensors.
template <int BM>
__device__ __forceinline__ bool at_find(const mi_attn_args& p, int t, int& start, int& len, int& tile, bool& tail)
{
    tail = false;
    if (!p.offsets) {
        const int per = (p.uniform_len + BM - 1) / BM;
        const int i = t / per;
        if (i >= p.nseq) return false;
        tile = t - i * per;
        start = i * p.uniform_len;
        len = p.uniform_len;
        return true;
    }
    const int lane = threadIdx.x & 63, T = (int)p.tokens;
    auto first = [&](int i) { int o = p.offsets[i]; o = o < 0 ? 0 : o > T ? T : o; return o; };
    int lo = 0, hi = p.nseq + (p.zero_tail ? 1 : 0);
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) >> 6, i = lo + lane * step;
        const bool below = i < hi && first(i) / BM + i <= t;
        const int n = __popcll(__builtin_amdgcn_ballot_w64(below));
        if (n == 0) return false;
        lo += (n - 1) * step;
        hi = hi < lo + step ? hi : lo + step;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    start = first(lo);
    tile = t - (start / BM + lo);
    if (tile < 0) return false;
    int end = T;
    if (lo < p.nseq) end = first(lo + 1);
    else if (p.zero_tail) tail = true;
    else return false;                                // (no sequences at all)
    len = end - start;
    start = __builtin_amdgcn_readfirstlane(start);
    len = __builtin_amdgcn_readfirstlane(len);
    return tile * BM < len;
}

// ---------------------------------------------------------------- tiles in LDS
// A tile is 64 rows of DP elements (head_dim rounded up to 32, 64 or 128), 16-byte chunks XOR-swizzled within the row so that both
// reads are free of bank conflicts (64 banks, 256 bytes a cycle): 16 consecutive rows at one chunk (operand rows, ds_read_b128) and
// 4 consecutive rows at 4 chunks (the transpose read, 32 lanes).  LDS-DMA writes lane i's 16 bytes at base + 16 i, so the swizzle is on
// the source side.
template <int DP> struct AtTile {
    static constexpr int RP = DP * 2;                 // row pitch, bytes
    static constexpr int BYTES = AT_KT * RP;
    static __device__ __forceinline__ int f(int row)
    {
        if constexpr (DP == 32) return (row >> 2) & 3;
        else if constexpr (DP == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        else return ((row & 3) << 2) | ((row >> 2) & 3);
    }
};

__device__ __forceinline__ void at_dma16(const void* src, unsigned lds_addr)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(src), "s"(lds_addr) : "memory", "m0");
}
__device__ __forceinline__ void at_dma16(unsigned off, const char* base, unsigned lds_addr)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "s"(lds_addr) : "memory", "m0");
}

// One operand's DMA: rows r0 .. r0 + 63 of a sequence (clamped to its last row) into the tile at lds_addr, by NW waves.
// Chunks beyond head_dim repeat the last one: their products meet zeros of the other operand, or columns that are not stored.
// Rows that the key mask takes out are staged as zeros: they may hold anything (0 x NaN in the product would not be 0).
// A whole tile costs no vector instruction but the loads: scalar bases, one constant 32-bit lane offset (64 rows are below 2^31 bytes).
__device__ const uint4 at_zero_chunk = {0, 0, 0, 0};
template <int DP, int NW> struct AtStage {
    static constexpr int LPR = DP / 8;                // lanes per row
    static constexpr int RPI = 64 / LPR;              // rows per instruction
    static constexpr int NI = AT_KT / (RPI * NW);
    const char* base;                                 // row 0 of the sequence (uniform)
    int pitch;                                        // bytes between rows
    int row0, chunk;                                  // this lane's row in instruction 0 and its bytes in the row
    unsigned off;
    int last;                                         // the sequence's last row
    __device__ __forceinline__ void init(const mi_attn_rows& x, int start, int len, int head, int hd, int wave, int lane)
    {
        row0 = wave * RPI + lane / LPR;
        int c = (lane % LPR) ^ AtTile<DP>::f(row0);
        const int most = (hd >> 3) - 1;
        chunk = (c < most ? c : most) * 16;
        base = reinterpret_cast<const char*>(x.p + (int64_t)start * x.ts + (int64_t)head * x.hs);
        pitch = (int)(x.ts * 2);
        off = (unsigned)(row0 * pitch + chunk);
        last = len - 1;
    }
    __device__ __forceinline__ void issue(int r0, unsigned lds_addr, int wave, const int32_t* mask = nullptr) const
    {
        const char* const at = base + (int64_t)r0 * pitch;
        if (!mask && r0 + AT_KT - 1 <= last) {
#pragma unroll
            for (int i = 0; i < NI; ++i) at_dma16(off, at + (int64_t)i * RPI * NW * pitch, lds_addr + (unsigned)((i * NW + wave) * 1024));
            return;
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            int row = row0 + i * RPI * NW;
            row = row < last - r0 ? row : last - r0;
            const char* src = at + (int64_t)row * pitch + chunk;
            if (mask && mask[r0 + row] == 0) src = reinterpret_cast<const char*>(&at_zero_chunk);
            at_dma16(src, lds_addr + (unsigned)((i * NW + wave) * 1024));
        }
    }
};
// everything outstanding has landed and been read, on every wave
__device__ __forceinline__ void at_sync()
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Operand rows straight from memory: row's chunks 2 s + half, s = 0 .. DP / 16 - 1, zero beyond head_dim.
template <int DP>
__device__ __forceinline__ void at_load_rows(u32x4 (&f)[DP / 16], const mi_attn_rows& x, int64_t token, int head, int hd, int half)
{
    const uint16_t* r = x.p + token * x.ts + (int64_t)head * x.hs;
    const int most = (hd >> 3) - 1;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int c = 2 * s + half;
        const u32x4 v = *reinterpret_cast<const u32x4*>(r + (c < most ? c : most) * 8);
        f[s] = c <= most ? v : u32x4{0, 0, 0, 0};
    }
}
// ... and a 32-row operand block of a tile: lane's row 32 st + col
template <int DP>
__device__ __forceinline__ u32x4 at_rows(const char* tile, int st, int s, int col, int half)
{
    return *reinterpret_cast<const u32x4*>(tile + (32 * st + col) * AtTile<DP>::RP + (((2 * s + half) ^ AtTile<DP>::f(col)) << 4));
}
// The transposed operand: columns 32 dt + col of the tile for the 16 rows 16 ks .., in the accumulators' order of rows: element j
// is row 16 ks + 8 (j >> 2) + 4 half + (j & 3).  In a 16-lane group lane 4 a + b supplies the address of row a, columns 4 b ..,
// and lane i receives column i of the 4 rows.
template <int DP>
__device__ __forceinline__ u32x4 at_cols(const char* tile, int ks, int dt, int lane)
{
    const int r = 4 * (lane >> 5) + ((lane & 15) >> 2);                // + 16 ks (+ 8: f differs)
    const int c = 4 * dt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const char* const a = tile + (16 * ks + r) * AtTile<DP>::RP + 8 * (lane & 1);
    const tr4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr4_lds_t*)(a + ((c ^ AtTile<DP>::f(r)) << 4)));
    const tr4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr4_lds_t*)(a + ((c ^ AtTile<DP>::f(r + 8)) << 4) + 8 * AtTile<DP>::RP));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
// DP columns of one row from transposed accumulators (column 32 dt + 8 g + 4 half + i), times f, as 16-bit elements
template <int DP, bool F16>
__device__ __forceinline__ void at_store_row(const mi_attn_rows& x, int64_t token, int head, int hd, int half, const f32x16 (&acc)[DP / 32], float f)
{
    uint16_t* r = x.p + token * x.ts + (int64_t)head * x.hs;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * dt + 8 * g + 4 * half;
            if (hd == DP || d < hd) {
                uint2 o;
                o.x = at_pack2<F16>(acc[dt][4 * g + 0] * f, acc[dt][4 * g + 1] * f);
                o.y = at_pack2<F16>(acc[dt][4 * g + 2] * f, acc[dt][4 * g + 3] * f);
                *reinterpret_cast<uint2*>(r + d) = o;
            }
        }
}
// ... and as fp32, row `row` of a [rows][head_dim] array
template <int DP>
__device__ __forceinline__ void at_store_part(float* x, int64_t row, int hd, int half, const f32x16 (&acc)[DP / 32], float f)
{
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * dt + 8 * g + 4 * half;
            if (d < hd) *reinterpret_cast<float4*>(x + row * hd + d) = make_float4(acc[dt][4 * g] * f, acc[dt][4 * g + 1] * f, acc[dt][4 * g + 2] * f, acc[dt][4 * g + 3] * f);
        }
}
__device__ __forceinline__ void at_zero_rows(const mi_attn_rows& x, int64_t token0, int rows, int head, int hd)
{
    const int per = hd >> 3;
    for (int i = threadIdx.x; i < rows * per; i += blockDim.x)
        *reinterpret_cast<u32x4*>(x.p + (token0 + i / per) * x.ts + (int64_t)head * x.hs + (i % per) * 8) = u32x4{0, 0, 0, 0};
}

// ---------------------------------------------------------------- relative position bias
// In LDS as a vector over r = key - query, [-(reach + AT_PAD), reach + AT_PAD]: a 64 x 32 tile of scores that touches |r| < reach
// stays inside it, any other tile lies in one bucket.  Values are in log2 units.
// A finite bias counts as at most 4096 in size.  Beyond that it only says "never" or "always" (exp(-4096) is 0 beside any other
// score), and a running reference near the type's lowest value would swallow the scores of the keys that come after it; at 4096
// fp32 still resolves a score to 2^-12, half of fp16's step in p.
#define AT_PAD 96
#define AT_BIAS_MOST 4096.0f
__host__ __device__ __forceinline__ int at_bucket(const mi_attn_args& p, int r)
{
    const int d = p.two_sided ? (r < 0 ? -r : r) : (r < 0 ? -r : 0);
    int b = d;
    if (d >= p.exact) {
        b = p.exact;
        for (int t = 0; t < p.nborder; ++t) b += d >= p.border[t] ? 1 : 0;
    }
    return b + (p.two_sided && r > 0 ? p.side : 0);
}
__device__ __forceinline__ float at_bias(const mi_attn_args& p, int head, int r)
{
    const float x = p.table[(int64_t)at_bucket(p, r) * p.heads + head];
    return (fabsf(x) <= FLT_MAX ? fminf(fmaxf(x, -AT_BIAS_MOST), AT_BIAS_MOST) : x) * AT_LOG2E;
}
__device__ __forceinline__ void at_fill_bias(const mi_attn_args& p, int head, float* vec)
{
    const int R = p.reach + AT_PAD;
    for (int i = threadIdx.x; i < 2 * R + 1; i += blockDim.x) vec[i] = at_bias(p, head, i - R);
}

// Which of the 64 keys at k0 are keys of the sequence that the mask leaves (bit = key - k0); the wave's lanes ask for one each.
__device__ __forceinline__ uint64_t at_keys(const int32_t* mask, int k0, int len, int lane)
{
    if (!mask && k0 + AT_KT <= len) return ~0ull;
    const int key = k0 + lane;
    return __builtin_amdgcn_ballot_w64(key < len && (!mask || mask[key < len ? key : len - 1] != 0));
}
// ... and of the 32 of block st those that this lane's query attends, bit 8 g + i for its register 4 g + i; ahead = query - k0
__device__ __forceinline__ uint32_t at_allowed(const mi_attn_args& p, uint64_t keys, int st, int ahead, int half)
{
    uint32_t ok = (uint32_t)(keys >> (32 * st));
    if (p.causal) {
        const int lim = ahead - 32 * st;                               // the last attended key of the block
        ok = lim >= 31 ? ok : lim < 0 ? 0u : ok & ((2u << lim) - 1u);
    }
    return ok >> (4 * half);
}

// ---------------------------------------------------------------- forward
// One block per (head, 128 QB query rows), four waves of 32 QB queries; K and V tiles of 64 keys by LDS-DMA, double-buffered, one
// barrier per tile.  The running maximum is an exponent reference that only has to keep exp2 in range: it moves, and O and l are
// rescaled, when a tile's maximum exceeds it by more than 2^8.
template <int DP, bool F16, bool BIAS, int QB>
__global__ __launch_bounds__(256, DP == 32 ? 4 : DP == 64 ? 3 : 2) void attn_fwd_kernel(const mi_attn_args p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int BM = 128 * QB, TB = AtTile<DP>::BYTES;
    float* const vec = reinterpret_cast<float*>(lds + 4 * TB);
    int head, t, start, len, tile;
    bool tail;
    if (!at_work(p, head, t) || !at_find<BM>(p, t, start, len, tile, tail)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    if (tail) {
        const int n = len - tile * BM < BM ? len - tile * BM : BM;
        at_zero_rows(p.out, start + tile * BM, n, head, p.hd);
        if (p.lse) for (int i = threadIdx.x; i < n; i += 256) p.lse[(int64_t)head * p.tokens + start + tile * BM + i] = -INFINITY;
        return;
    }
    if (p.causal) tile = (len + BM - 1) / BM - 1 - tile;               // the longest rows first
    const int qw = tile * BM + wave * 32 * QB;                         // this wave's first query
    const int kend = p.causal ? (tile * BM + BM < len ? tile * BM + BM : len) : len;

    u32x4 qf[QB][DP / 16];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        const int q = qw + 32 * b + col;
        at_load_rows<DP>(qf[b], p.q, start + (q < len ? q : len - 1), head, p.hd, half);
    }
    const int kvh = head / p.group;
    AtStage<DP, 4> ks, vs;
    ks.init(p.k, start, len, kvh, p.hd, wave, lane);
    vs.init(p.v, start, len, kvh, p.hd, wave, lane);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
    const int32_t* const mask = p.key_mask ? p.key_mask + start : nullptr;
    ks.issue(0, lds0, wave, mask);
    vs.issue(0, lds0 + TB, wave, mask);
    if constexpr (BIAS) at_fill_bias(p, head, vec);

    f32x16 O[QB][DP / 32];
    float m[QB], thr[QB], l[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) O[b][dt] = at_zero16();
        m[b] = 0.0f;
        thr[b] = -INFINITY;                                            // no finite score seen yet
        l[b] = 0.0f;
    }
    const int R = p.reach + AT_PAD;
    for (int k0 = 0, buf = 0; k0 < kend; k0 += AT_KT, buf ^= 1) {
        at_sync();                                                     // this tile has landed, the other buffer has been read
        if (k0 + AT_KT < kend) {
            ks.issue(k0 + AT_KT, lds0 + (buf ^ 1) * 2 * TB, wave, mask);
            vs.issue(k0 + AT_KT, lds0 + (buf ^ 1) * 2 * TB + TB, wave, mask);
        }
        if (qw >= len || (p.causal && k0 > qw + 32 * QB - 1)) continue;  // nothing for this wave (it has met the barrier)
        const char* const Kt = lds + buf * 2 * TB;
        const char* const Vt = Kt + TB;
        const uint64_t keys = at_keys(mask, k0, len, lane);
        const bool masked = ~keys != 0 || (p.causal && k0 + AT_KT - 1 > qw);

        f32x16 S[QB][2];
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                const u32x4 kf = at_rows<DP>(Kt, st, s, col, half);
#pragma unroll
                for (int b = 0; b < QB; ++b) S[b][st] = at_mfma<F16>(kf, qf[b][s], s == 0 ? at_zero16() : S[b][st]);
            }
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            const int q = qw + 32 * b + col;
            const float c = p.scale_log2;
            // x = score in log2 units, less the reference
            if constexpr (BIAS) {
                const int rlo = k0 - (qw + 32 * b + 31), rhi = k0 + AT_KT - 1 - (qw + 32 * b);
                if (rhi <= -p.reach || rlo >= p.reach) {
                    const float far = vec[rhi <= -p.reach ? 0 : 2 * R] - m[b];
#pragma unroll
                    for (int st = 0; st < 2; ++st)
#pragma unroll
                        for (int i = 0; i < 16; ++i) S[b][st][i] = __builtin_fmaf(S[b][st][i], c, far);
                } else {
                    const float* bv = vec + (k0 + 4 * half - q + R);
#pragma unroll
                    for (int st = 0; st < 2; ++st)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            S[b][st][i] = __builtin_fmaf(S[b][st][i], c, bv[32 * st + 8 * (i >> 2) + (i & 3)] - m[b]);
                }
            } else {
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int i = 0; i < 16; ++i) S[b][st][i] = __builtin_fmaf(S[b][st][i], c, -m[b]);
            }
            if (masked) {
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    const uint32_t ok = at_allowed(p, keys, st, q - k0, half);
#pragma unroll
                    for (int i = 0; i < 16; ++i) S[b][st][i] = (ok >> (8 * (i >> 2) + (i & 3))) & 1u ? S[b][st][i] : -INFINITY;
                }
            }
            float top = S[b][0][0];
#pragma unroll
            for (int i = 1; i < 15; i += 2) top = at_max3(top, S[b][0][i], S[b][0][i + 1]);
            top = at_max3(top, S[b][0][15], S[b][1][0]);
#pragma unroll
            for (int i = 1; i < 15; i += 2) top = at_max3(top, S[b][1][i], S[b][1][i + 1]);
            top = fmaxf(top, S[b][1][15]);
            if (__builtin_amdgcn_ballot_w64(top > thr[b]) != 0) {
                top = fmaxf(top, at_other_half(top));                  // both halves of a query move alike
                const bool move = top > thr[b];
                const float up = move ? top : 0.0f;
                const float alpha = move ? (thr[b] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(-up)) : 1.0f;
                m[b] += up;
                if (move) thr[b] = 8.0f;
                l[b] *= alpha;
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt) O[b][dt] = O[b][dt] * alpha;
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int i = 0; i < 16; ++i) S[b][st][i] -= up;
            }
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    S[b][st][i] = __builtin_amdgcn_exp2f(S[b][st][i]);
                    l[b] += S[b][st][i];
                }
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            u32x4 pf[QB];
#pragma unroll
            for (int b = 0; b < QB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    pf[b][i] = at_pack2<F16>(S[b][kk >> 1][8 * (kk & 1) + 2 * i], S[b][kk >> 1][8 * (kk & 1) + 2 * i + 1]);
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) {
                const u32x4 vf = at_cols<DP>(Vt, kk, dt, lane);
#pragma unroll
                for (int b = 0; b < QB; ++b) O[b][dt] = at_mfma<F16>(vf, pf[b], O[b][dt]);
            }
        }
    }
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        const int q = qw + 32 * b + col;
        const float sum = l[b] + at_other_half(l[b]);
        if (q < len) {
            at_store_row<DP, F16>(p.out, start + q, head, p.hd, half, O[b], sum == 0.0f ? 0.0f : 1.0f / sum);
            if (p.lse && half == 0)
                p.lse[(int64_t)head * p.tokens + start + q] = sum == 0.0f ? -INFINITY : (m[b] + __builtin_amdgcn_logf(sum)) * AT_LN2;
        }
    }
}

// ---------------------------------------------------------------- backward
// P is rebuilt from the saved log-sum-exp.  fp16 only: p is scaled by 2^12 on its way into the 16-bit operand of dV (a row of
// thousands of keys has p near fp16's subnormals), and ds = p (dp - D) takes the scale back out.
template <bool F16> struct AtPScale { static constexpr float log2 = F16 ? 12.0f : 0.0f, up = F16 ? 4096.0f : 1.0f, down = F16 ? 1.0f / 4096.0f : 1.0f; };

// D = sum_j p dp of every row.  rowsum(dout * out) is the same sum, but takes over the rounding of p and out in the forward pass,
// which shows in rows of few keys (20 causal rows: dq and dk 1.65 x the plain rounding of their values, 1.4 with D exact) and in
// the table's gradient, a sum of many ds that nearly cancel.  So with a bias, for rows of up to 128 keys, and for up to 512 where
// a mask may leave few of them, the sum is made from the scores, in fp32; other rows take the dot product.
template <int DP, bool F16, bool BIAS>
__global__ __launch_bounds__(256, 2) void attn_delta_kernel(const mi_attn_args p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int BM = 128, TB = AtTile<DP>::BYTES;
    float* const vec = reinterpret_cast<float*>(lds + 4 * TB);
    int head, t, start, len, tile;
    bool tail;
    if (!at_work(p, head, t) || !at_find<BM>(p, t, start, len, tile, tail) || tail || tile * BM >= len) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    if (p.causal) tile = (len + BM - 1) / BM - 1 - tile;
    const int qw = tile * BM + wave * 32, q = qw + col;
    const int kend = p.causal ? (tile * BM + BM < len ? tile * BM + BM : len) : len;
    const int64_t tok = start + (q < len ? q : len - 1);
    const int32_t* const mask = p.key_mask ? p.key_mask + start : nullptr;
    u32x4 df[DP / 16], qf[DP / 16];                                    // qf: rows of out, or of q
    at_load_rows<DP>(df, p.dout, tok, head, p.hd, half);
    float a = 0.0f, c = 0.0f;
    if (!BIAS && kend > (mask ? 512 : 128)) {
        at_load_rows<DP>(qf, p.out, tok, head, p.hd, half);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a = __builtin_fmaf(at_lo<F16>(df[s][j]), at_lo<F16>(qf[s][j]), a);
                a = __builtin_fmaf(at_hi<F16>(df[s][j]), at_hi<F16>(qf[s][j]), a);
            }
        c = half == 0 ? 1.0f : 0.0f;
    } else {
        at_load_rows<DP>(qf, p.q, tok, head, p.hd, half);
        AtStage<DP, 4> ks, vs;
        ks.init(p.k, start, len, head / p.group, p.hd, wave, lane);
        vs.init(p.v, start, len, head / p.group, p.hd, wave, lane);
        const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
        ks.issue(0, lds0, wave, mask);
        vs.issue(0, lds0 + TB, wave, mask);
        if constexpr (BIAS) at_fill_bias(p, head, vec);
        float nl = p.lse[(int64_t)head * p.tokens + tok] * AT_LOG2E;
        if (nl == -INFINITY) nl = INFINITY;                            // a row that attends nothing: p = 0
        const int R = p.reach + AT_PAD;
        for (int k0 = 0, buf = 0; k0 < kend; k0 += AT_KT, buf ^= 1) {
            at_sync();
            if (k0 + AT_KT < kend) {
                ks.issue(k0 + AT_KT, lds0 + (buf ^ 1) * 2 * TB, wave, mask);
                vs.issue(k0 + AT_KT, lds0 + (buf ^ 1) * 2 * TB + TB, wave, mask);
            }
            if (qw >= len || (p.causal && k0 > qw + 31)) continue;
            const char* const Kt = lds + buf * 2 * TB;
            const uint64_t keys = at_keys(mask, k0, len, lane);
            const bool masked = ~keys != 0 || (p.causal && k0 + AT_KT - 1 > qw);
            const int rlo = k0 - (qw + 31), rhi = k0 + AT_KT - 1 - qw;
            const bool near = BIAS && rhi > -p.reach && rlo < p.reach;
            const float far = BIAS && !near ? vec[rhi <= -p.reach ? 0 : 2 * R] - nl : -nl;
            const float* const bv = vec + (k0 + 4 * half - q + R);
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                f32x16 S = at_zero16(), dP = at_zero16();
#pragma unroll
                for (int s = 0; s < DP / 16; ++s) S = at_mfma<F16>(at_rows<DP>(Kt, st, s, col, half), qf[s], S);
#pragma unroll
                for (int s = 0; s < DP / 16; ++s) dP = at_mfma<F16>(at_rows<DP>(Kt + TB, st, s, col, half), df[s], dP);
                if (near) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) S[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], p.scale_log2, bv[32 * st + 8 * (i >> 2) + (i & 3)] - nl));
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) S[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], p.scale_log2, far));
                }
                if (masked) {
                    const uint32_t ok = at_allowed(p, keys, st, q - k0, half);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const bool on = (ok >> (8 * (i >> 2) + (i & 3))) & 1u;
                        S[i] = on ? S[i] : 0.0f;
                        dP[i] = on ? dP[i] : 0.0f;
                    }
                }
                float a1 = 0.0f, c1 = 0.0f;                            // (short chains: a long row's sums stay exact to fp32's last bits)
#pragma unroll
                for (int i = 0; i < 16; ++i) { a1 = __builtin_fmaf(S[i], dP[i], a1); c1 += S[i]; }
                a += a1;
                c += c1;
            }
        }
    }
    a += at_other_half(a);
    c += at_other_half(c);
    if (half == 0 && q < len) p.delta[(int64_t)head * p.tokens + tok] = c == 0.0f ? a : a / c;
}

// dQ: one block per (head, 128 query rows), like the forward pass: S^T = K Q^T and dP^T = V dO^T with the query on the lane,
// dQ^T += K^T dS^T.
//
// BIAS: the table's gradient is the sum of ds along the diagonals r = key - query.  A 32 x 32 block of ds goes through a skewed
// image in LDS, element (key, query) at [query][key - query + 31], so that lane l finds a diagonal in column l (the positions a row
// never writes hold the zeros they started with); the 63 sums are added to the wave's vector over r.  A tile of one bucket adds
// in registers.  Every sum has one owner and a fixed order.  @DQ_BIAS@
template <int DP, bool F16, bool BIAS>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(const mi_attn_args p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int BM = 128, TB = AtTile<DP>::BYTES;
    const int R = p.reach + AT_PAD, nvec = 2 * R + 1;
    float* const skew0 = reinterpret_cast<float*>(lds + 4 * TB);       // BIAS: [4][32][64], the waves' images
    float* const vec = skew0 + 4 * 32 * 64;                            // the bias over r
    float* const dvec0 = vec + nvec;                                   // [4][nvec], the waves' sums over r
    int head, t, start, len, tile;
    bool tail;
    if (!at_work(p, head, t)) return;
    float* const part = BIAS ? p.partial + ((int64_t)head * p.tiles + t) * MI_ATTN_MAX_BUCKETS : nullptr;
    if (!at_find<BM>(p, t, start, len, tile, tail) || tail || tile * BM >= len) {
        if (BIAS && (int)threadIdx.x < MI_ATTN_MAX_BUCKETS) part[threadIdx.x] = 0.0f;
        if (tail) at_zero_rows(p.dq, start + tile * BM, len - tile * BM < BM ? len - tile * BM : BM, head, p.hd);
        return;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    if (p.causal) tile = (len + BM - 1) / BM - 1 - tile;
    const int qw = tile * BM + wave * 32, q = qw + col;
    const int kend = p.causal ? (tile * BM + BM < len ? tile * BM + BM : len) : len;
    const int kvh = head / p.group;

    AtStage<DP, 4> ks, vs;
    ks.init(p.k, start, len, kvh, p.hd, wave, lane);
    vs.init(p.v, start, len, kvh, p.hd, wave, lane);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
    const int32_t* const mask = p.key_mask ? p.key_mask + start : nullptr;
    ks.issue(0, lds0, wave, mask);
    vs.issue(0, lds0 + TB, wave, mask);

    u32x4 qf[DP / 16], df[DP / 16];
    const int64_t tok = start + (q < len ? q : len - 1);
    at_load_rows<DP>(qf, p.q, tok, head, p.hd, half);
    at_load_rows<DP>(df, p.dout, tok, head, p.hd, half);
    const float D = p.delta[(int64_t)head * p.tokens + tok];
    float nl = p.lse[(int64_t)head * p.tokens + tok] * AT_LOG2E;
    if (nl == -INFINITY || q >= len) nl = INFINITY;                    // a row that attends nothing, or is none: p = 0

    float* const skew = skew0 + wave * 32 * 64;
    float* const dvec = dvec0 + wave * nvec;
    float farS[2] = {0.0f, 0.0f};                                      // sums of the tiles of one bucket, before and behind
    if constexpr (BIAS) {
        at_fill_bias(p, head, vec);
#pragma unroll
        for (int i = 0; i < 32; ++i) skew[i * 64 + lane] = 0.0f;
        for (int i = lane; i < nvec; i += 64) dvec[i] = 0.0f;
    }
    f32x16 dQ[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) dQ[dt] = at_zero16();

    for (int k0 = 0, buf = 0; k0 < kend; k0 += AT_KT, buf ^= 1) {
        at_sync();
        if (k0 + AT_KT < kend) {
            ks.issue(k0 + AT_KT, lds0 + (buf ^ 1) * 2 * TB, wave, mask);
            vs.issue(k0 + AT_KT, lds0 + (buf ^ 1) * 2 * TB + TB, wave, mask);
        }
        if (qw >= len || (p.causal && k0 > qw + 31)) continue;
        const char* const Kt = lds + buf * 2 * TB;
        const uint64_t keys = at_keys(mask, k0, len, lane);
        const bool masked = ~keys != 0 || (p.causal && k0 + AT_KT - 1 > qw);
        const int rlo = k0 - (qw + 31), rhi = k0 + AT_KT - 1 - qw;
        const bool near = BIAS && rhi > -p.reach && rlo < p.reach;
        const float far = BIAS && !near ? vec[rhi <= -p.reach ? 0 : 2 * R] - nl : -nl;
        const float* const bv = vec + (k0 + 4 * half - q + R);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            f32x16 S = at_zero16(), dP = at_zero16();
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) S = at_mfma<F16>(at_rows<DP>(Kt, st, s, col, half), qf[s], S);
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) dP = at_mfma<F16>(at_rows<DP>(Kt + TB, st, s, col, half), df[s], dP);
            if (near) {
#pragma unroll
                for (int i = 0; i < 16; ++i) S[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], p.scale_log2, bv[32 * st + 8 * (i >> 2) + (i & 3)] - nl));
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) S[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], p.scale_log2, far));
            }
            // ds, over dp
#pragma unroll
            for (int i = 0; i < 16; ++i) dP[i] = S[i] * (dP[i] - D);
            if (masked) {
                const uint32_t ok = at_allowed(p, keys, st, q - k0, half);
#pragma unroll
                for (int i = 0; i < 16; ++i) dP[i] = (ok >> (8 * (i >> 2) + (i & 3))) & 1u ? dP[i] : 0.0f;
            }
            if constexpr (BIAS) {
                if (near) {
                    float* const at = skew + col * 63 + 31 + 4 * half;
#pragma unroll
                    for (int i = 0; i < 16; ++i) at[8 * (i >> 2) + (i & 3)] = dP[i];
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[i & 3] += skew[i * 64 + lane];
                    if (lane < 63) dvec[rlo + 32 * st + R + lane] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                } else {
                    float sum[2] = {0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[i & 1] += dP[i];
                    farS[0] += rhi <= -p.reach ? sum[0] + sum[1] : 0.0f;
                    farS[1] += rhi <= -p.reach ? 0.0f : sum[0] + sum[1];
                }
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                u32x4 sf;
#pragma unroll
                for (int i = 0; i < 4; ++i) sf[i] = at_pack2<F16>(dP[8 * kk + 2 * i], dP[8 * kk + 2 * i + 1]);
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt) dQ[dt] = at_mfma<F16>(at_cols<DP>(Kt, 2 * st + kk, dt, lane), sf, dQ[dt]);
            }
        }
    }
    if (q < len) at_store_row<DP, F16>(p.dq, start + q, head, p.hd, half, dQ, p.scale);
    if constexpr (BIAS) {
        // lane b of each wave sums the wave's diagonals of bucket b, then one wave adds the waves
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) {
            farS[0] += __shfl_xor(farS[0], s, 64);
            farS[1] += __shfl_xor(farS[1], s, 64);
        }
        if (lane == 0) {
            dvec[0] += farS[0];
            dvec[2 * R] += farS[1];
        }
        float sum = 0.0f;
        if (lane < p.buckets) {
            const bool ahead = p.two_sided && lane >= p.side;          // r > 0
            const int i = ahead ? lane - p.side : lane;
            int lo = i < p.exact ? i : i == p.exact ? p.exact : p.border[i - p.exact - 1];           // distances lo .. hi
            int hi = i < p.exact ? i : i - p.exact < p.nborder ? p.border[i - p.exact] - 1 : R;
            if (ahead && lo == 0) lo = 1;                              // distance 0 is not ahead
            for (int d = lo; d <= hi; ++d) sum += dvec[ahead ? R + d : R - d];
            if (!p.two_sided && lane == 0)
                for (int d = 1; d <= R; ++d) sum += dvec[R + d];       // one-sided: whatever is ahead counts as distance 0
        }
        at_sync();
        skew0[wave * 64 + lane] = sum;
        at_sync();
        if (wave == 0) part[lane] = (skew0[lane] + skew0[64 + lane]) + (skew0[128 + lane] + skew0[192 + lane]);
    }
}

// dK, dV: one block per (key head, share of its query heads, 128 keys), a wave per 32 keys, over the tiles of 64 query rows of
// the share's heads: S = Q K^T and dP = dO V^T with the key on the lane, dV^T += dO^T P, dK^T += Q^T dS.  Where one block per key
// head and tile would leave CUs idle the group's heads are shared out over `splits` blocks, whose fp32 sums attn_join_kernel
// adds in the heads' order.
template <int DP, bool F16, bool BIAS>
__global__ __launch_bounds__(256, DP == 128 ? 1 : 2) void attn_dkv_kernel(const mi_attn_args p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int BM = 128, TB = AtTile<DP>::BYTES;
    float* const rowv = reinterpret_cast<float*>(lds + 4 * TB);        // [2][lse | D][64]
    float* const vec = rowv + 256;
    int kvh, t, start, len, tile;
    bool tail;
    if (!at_work(p, kvh, t) || !at_find<BM>(p, t, start, len, tile, tail)) return;
    const int share = kvh % p.splits, heads = p.group / p.splits;      // (units are key heads x shares)
    kvh /= p.splits;
    const int head0 = kvh * p.group + share * heads;
    if (tail) {
        if (share != 0) return;
        const int n = len - tile * BM < BM ? len - tile * BM : BM;
        at_zero_rows(p.dk, start + tile * BM, n, kvh, p.hd);
        at_zero_rows(p.dv, start + tile * BM, n, kvh, p.hd);
        return;
    }
    if (tile * BM >= len) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int kw = tile * BM + wave * 32, key = kw + col;
    const int64_t ktok = start + (key < len ? key : len - 1);
    u32x4 kf[DP / 16], vf[DP / 16];
    at_load_rows<DP>(kf, p.k, ktok, kvh, p.hd, half);
    at_load_rows<DP>(vf, p.v, ktok, kvh, p.hd, half);
    const bool on = key < len && (!p.key_mask || p.key_mask[ktok] != 0);

    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
    const int qfirst = p.causal ? tile * BM / AT_KT * AT_KT : 0;       // earlier queries attend no key of this block
    const int nq = (len - qfirst + AT_KT - 1) / AT_KT, n = nq * heads;
    AtStage<DP, 4> qs, ds;
    float rowreg = 0.0f;
    auto issue = [&](int it, int buf) __attribute__((always_inline)) {
        const int head = head0 + it / nq, q0 = qfirst + it % nq * AT_KT;
        qs.init(p.q, start, len, head, p.hd, wave, lane);
        ds.init(p.dout, start, len, head, p.hd, wave, lane);
        qs.issue(q0, lds0 + buf * 2 * TB, wave);
        ds.issue(q0, lds0 + buf * 2 * TB + TB, wave);
        if (wave < 2) {                                                // wave 0: log-sum-exp in log2 units, wave 1: D
            const int q = q0 + lane;
            const int64_t i = (int64_t)head * p.tokens + start + (q < len ? q : len - 1);
            if (wave == 0) {
                const float x = p.lse[i] * AT_LOG2E;
                rowreg = q < len && x != -INFINITY ? x - AtPScale<F16>::log2 : INFINITY;
            } else {
                rowreg = q < len ? p.delta[i] * AtPScale<F16>::down : 0.0f;
            }
        }
    };
    f32x16 dK[DP / 32], dV[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) { dK[dt] = at_zero16(); dV[dt] = at_zero16(); }
    issue(0, 0);
    const int R = p.reach + AT_PAD;
    int bias_head = -1;
    for (int it = 0, buf = 0; it < n; ++it, buf ^= 1) {
        if (wave < 2) rowv[buf * 128 + wave * 64 + lane] = rowreg;
        const int head = head0 + it / nq, q0 = qfirst + it % nq * AT_KT;
        if constexpr (BIAS) {
            if (head != bias_head) {
                if (bias_head >= 0) at_sync();                         // the last head's vector has been read
                at_fill_bias(p, head, vec);
                bias_head = head;
            }
        }
        at_sync();
        if (it + 1 < n) issue(it + 1, buf ^ 1);
        if (kw >= len || (p.causal && q0 + AT_KT - 1 < kw)) continue;
        const char* const Qt = lds + buf * 2 * TB;
        const char* const Dt = Qt + TB;
        const bool diag = p.causal && q0 < kw + 31;
        const int rlo = kw - (q0 + AT_KT - 1), rhi = kw + 31 - q0;
        const bool near = BIAS && rhi > -p.reach && rlo < p.reach;
        const float far = BIAS && !near ? vec[rhi <= -p.reach ? 0 : 2 * R] : 0.0f;
        const int at = key - q0 - 4 * half + R;
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            f32x16 S = at_zero16(), dP = at_zero16();
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) S = at_mfma<F16>(at_rows<DP>(Qt, st, s, col, half), kf[s], S);
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) dP = at_mfma<F16>(at_rows<DP>(Dt, st, s, col, half), vf[s], dP);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 nl = *reinterpret_cast<const float4*>(rowv + buf * 128 + 32 * st + 8 * g + 4 * half);
                const float4 Dr = *reinterpret_cast<const float4*>(rowv + buf * 128 + 64 + 32 * st + 8 * g + 4 * half);
                const float nls[4] = {nl.x, nl.y, nl.z, nl.w}, Drs[4] = {Dr.x, Dr.y, Dr.z, Dr.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 4 * g + e;
                    const float b = near ? vec[at - 32 * st - 8 * g - e] : far;
                    S[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], p.scale_log2, b - nls[e]));
                    dP[i] = S[i] * __builtin_fmaf(dP[i], AtPScale<F16>::down, -Drs[e]);
                }
            }
            if (diag) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const bool ok = q0 + 32 * st + 8 * (i >> 2) + 4 * half + (i & 3) >= key;
                    S[i] = ok ? S[i] : 0.0f;
                    dP[i] = ok ? dP[i] : 0.0f;
                }
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                u32x4 pf, sf;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    pf[i] = at_pack2<F16>(S[8 * kk + 2 * i], S[8 * kk + 2 * i + 1]);
                    sf[i] = at_pack2<F16>(dP[8 * kk + 2 * i], dP[8 * kk + 2 * i + 1]);
                }
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt) {
                    dV[dt] = at_mfma<F16>(at_cols<DP>(Dt, 2 * st + kk, dt, lane), pf, dV[dt]);
                    dK[dt] = at_mfma<F16>(at_cols<DP>(Qt, 2 * st + kk, dt, lane), sf, dK[dt]);
                }
            }
        }
    }
    if (key < len) {
        if (!on) {                                                     // a masked key (the products above ran on its column alone)
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) { dK[dt] = at_zero16(); dV[dt] = at_zero16(); }
        }
        if (p.splits == 1) {
            at_store_row<DP, F16>(p.dk, start + key, kvh, p.hd, half, dK, p.scale);
            at_store_row<DP, F16>(p.dv, start + key, kvh, p.hd, half, dV, AtPScale<F16>::down);
        } else {
            at_store_part<DP>(p.parts_kv, ((int64_t)(2 * share) * p.tokens + start + key) * (p.heads / p.group) + kvh, p.hd, half, dK, p.scale);
            at_store_part<DP>(p.parts_kv, ((int64_t)(2 * share + 1) * p.tokens + start + key) * (p.heads / p.group) + kvh, p.hd, half, dV, AtPScale<F16>::down);
        }
    }
}

// dk and dv from the shares' sums ([share][dk | dv][token][key head][head_dim] fp32), 8 elements a thread
template <bool F16>
__global__ __launch_bounds__(256) void attn_join_kernel(const mi_attn_args p)
{
    const int per = p.hd >> 3, kvh = p.heads / p.group;
    const int64_t n = p.tokens * kvh * per, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int64_t row = i / per, token = row / kvh;
    if (p.offsets && (token < p.offsets[0] || token >= p.offsets[p.nseq])) return;   // no sequence's: left, or zeroed by the tail's block
    const mi_attn_rows& x = blockIdx.y ? p.dv : p.dk;
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int s = 0; s < p.splits; ++s) {
        const float4* src = reinterpret_cast<const float4*>(p.parts_kv + (((int64_t)(2 * s + blockIdx.y) * p.tokens) * kvh + row) * p.hd + (i % per) * 8);
        const float4 a = src[0], b = src[1];
        sum[0] += a.x; sum[1] += a.y; sum[2] += a.z; sum[3] += a.w;
        sum[4] += b.x; sum[5] += b.y; sum[6] += b.z; sum[7] += b.w;
    }
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = at_pack2<F16>(sum[2 * j], sum[2 * j + 1]);
    *reinterpret_cast<u32x4*>(x.p + token * x.ts + (row % kvh) * x.hs + (i % per) * 8) = o;
}

// dT[b][head] = the sum of the blocks' partial sums, in the tiles' order within each of 16 strides
__global__ __launch_bounds__(1024) void attn_dtable_kernel(const mi_attn_args p)
{
    __shared__ float red[16][64];
    const int b = threadIdx.x & 63, s = threadIdx.x >> 6, head = blockIdx.x;
    float sum = 0.0f;
    for (int t = s; t < p.tiles; t += 16) sum += p.partial[((int64_t)head * p.tiles + t) * MI_ATTN_MAX_BUCKETS + b];
    red[s][b] = sum;
    __syncthreads();
    if (s == 0 && b < p.buckets) {
        for (int i = 1; i < 16; ++i) sum += red[i][b];
        p.dtable[(int64_t)b * p.heads + head] = sum;
    }
}

// ---------------------------------------------------------------- launch
static int gcd_int(int a, int b) { while (b) { const int t = a % b; a = b; b = t; } return a; }

// The grid over `heads` heads and tiles of BM rows (see at_work).
static unsigned at_schedule(mi_attn_args* a, int heads, int BM)
{
    const int64_t tiles = a->offsets ? a->tokens / BM + a->nseq + (a->zero_tail ? 1 : 0)
                                     : (int64_t)a->nseq * ((a->uniform_len + BM - 1) / BM);
    const int g = gcd_int(heads, 8);
    a->tiles = (int)tiles;
    a->parts = 8 / g;
    a->units_per_xcd = heads * a->parts / 8;
    a->tiles_per_unit = (int)((tiles + a->parts - 1) / a->parts);
    return (unsigned)((int64_t)heads * a->parts * a->tiles_per_unit);
}

// Leave for more than the default 64 KB of dynamic LDS, asked for once per kernel and device.
template <auto KERNEL>
static int at_lds(size_t bytes)
{
    static std::atomic<uint64_t> done{0};
    if (bytes <= 64 * 1024) return MI_OK;
    int dev = 0;
    MI_HIP(hipGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return MI_OK;
    MI_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
    return MI_OK;
}

template <int DP, bool F16>
static int launch_fwd(hipStream_t st, mi_attn_args& a)
{
    const unsigned grid = at_schedule(&a, a.heads, 128);
    size_t smem = 4 * AtTile<DP>::BYTES;
    if (grid == 0) return MI_OK;
    if (a.table) {
        smem += (2 * (size_t)(a.reach + AT_PAD) + 1) * sizeof(float);
        MI_TRY((at_lds<&attn_fwd_kernel<DP, F16, true, 1>>(smem)));
        attn_fwd_kernel<DP, F16, true, 1><<<grid, 256, smem, st>>>(a);
    } else {
        MI_TRY((at_lds<&attn_fwd_kernel<DP, F16, false, 1>>(smem)));
        attn_fwd_kernel<DP, F16, false, 1><<<grid, 256, smem, st>>>(a);
    }
    MI_HIP(hipGetLastError());
    return MI_OK;
}

int mi_launch_attention(hipStream_t st, mi_attn_args a, int dtype)
{
    const bool f16 = dtype == MI_DTYPE_F16;
    if (a.hd <= 32) return f16 ? launch_fwd<32, true>(st, a) : launch_fwd<32, false>(st, a);
    if (a.hd <= 64) return f16 ? launch_fwd<64, true>(st, a) : launch_fwd<64, false>(st, a);
    return f16 ? launch_fwd<128, true>(st, a) : launch_fwd<128, false>(st, a);
}

// Shares of a group's query heads in the dK / dV kernel: the fewest that give AT_DKV_BLOCKS blocks (two per CU, four rounds, so
// that a causal sequence's long first tiles even out), all heads at most.  1 x 8,191 causal, 8 heads on 2 key heads of 128:
// 128 blocks 1,620 us, 512 blocks @DKV_SPLIT@ us.
#define AT_DKV_BLOCKS 2048
static int at_dkv_splits(const mi_attn_args& a)
{
    const int64_t blocks = (int64_t)(a.heads / a.group) * (a.tokens / 128 + a.nseq);
    for (int s = 1; s < a.group; ++s)
        if (a.group % s == 0 && blocks * s >= AT_DKV_BLOCKS) return s;
    return a.group;
}

size_t mi_attn_backward_bytes(const mi_attn_args& a)
{
    const size_t delta = mi_round_up((int64_t)a.heads * a.tokens * 4, 256);
    const int splits = at_dkv_splits(a);
    const size_t join = splits > 1 ? (size_t)mi_round_up((int64_t)splits * 2 * a.tokens * (a.heads / a.group) * a.hd * 4, 256) : 0;
    const int64_t tiles = a.offsets ? a.tokens / 128 + a.nseq + 1 : (int64_t)a.nseq * ((a.uniform_len + 127) / 128);
    return delta + join + (a.table ? (size_t)(a.heads * tiles) * MI_ATTN_MAX_BUCKETS * 4 : 0);
}

template <int DP, bool F16, bool BIAS>
static int launch_dq(hipStream_t st, mi_attn_args& a)
{
    const unsigned grid = at_schedule(&a, a.heads, 128);
    if (grid == 0) return MI_OK;
    const size_t smem = 4 * AtTile<DP>::BYTES + (BIAS ? (4 * 32 * 64 + 5 * (2 * (size_t)(a.reach + AT_PAD) + 1)) * 4 : 0);
    MI_TRY((at_lds<&attn_dq_kernel<DP, F16, BIAS>>(smem)));
    attn_dq_kernel<DP, F16, BIAS><<<grid, 256, smem, st>>>(a);
    MI_HIP(hipGetLastError());
    return MI_OK;
}

template <int DP, bool F16, bool BIAS>
static int launch_delta(hipStream_t st, mi_attn_args& a)
{
    const unsigned grid = at_schedule(&a, a.heads, 128);
    if (grid == 0) return MI_OK;
    const size_t smem = 4 * AtTile<DP>::BYTES + (BIAS ? (size_t)(2 * (a.reach + AT_PAD) + 1) * 4 : 0);
    MI_TRY((at_lds<&attn_delta_kernel<DP, F16, BIAS>>(smem)));
    attn_delta_kernel<DP, F16, BIAS><<<grid, 256, smem, st>>>(a);
    MI_HIP(hipGetLastError());
    return MI_OK;
}

template <int DP, bool F16>
static int launch_bwd(hipStream_t st, mi_attn_args& a)
{
    if (a.table) MI_TRY((launch_delta<DP, F16, true>(st, a)));
    else MI_TRY((launch_delta<DP, F16, false>(st, a)));
    if (a.table) MI_TRY((launch_dq<DP, F16, true>(st, a)));
    else MI_TRY((launch_dq<DP, F16, false>(st, a)));
    if (a.table) {
        attn_dtable_kernel<<<(unsigned)a.heads, 1024, 0, st>>>(a);
        MI_HIP(hipGetLastError());
    }
    const unsigned grid = at_schedule(&a, a.heads / a.group * a.splits, 128);
    if (grid == 0) return MI_OK;
    const size_t smem = 4 * AtTile<DP>::BYTES + 1024 + (a.table ? (size_t)(2 * (a.reach + AT_PAD) + 1) * 4 : 0);
    if (a.table) {
        MI_TRY((at_lds<&attn_dkv_kernel<DP, F16, true>>(smem)));
        attn_dkv_kernel<DP, F16, true><<<grid, 256, smem, st>>>(a);
    } else {
        MI_TRY((at_lds<&attn_dkv_kernel<DP, F16, false>>(smem)));
        attn_dkv_kernel<DP, F16, false><<<grid, 256, smem, st>>>(a);
    }
    MI_HIP(hipGetLastError());
    if (a.splits > 1) {
        attn_join_kernel<F16><<<dim3((unsigned)((a.tokens * (a.heads / a.group) * (a.hd >> 3) + 255) / 256), 2), 256, 0, st>>>(a);
        MI_HIP(hipGetLastError());
    }
    return MI_OK;
}

int mi_launch_attention_backward(hipStream_t st, mi_attn_args a, int dtype, void* workspace)
{
    a.delta = (float*)workspace;
    a.splits = at_dkv_splits(a);
    a.parts_kv = (float*)((char*)workspace + mi_round_up((int64_t)a.heads * a.tokens * 4, 256));
    a.partial = (float*)((char*)a.parts_kv + (a.splits > 1 ? mi_round_up((int64_t)a.splits * 2 * a.tokens * (a.heads / a.group) * a.hd * 4, 256) : 0));
    const bool f16 = dtype == MI_DTYPE_F16;
    if (a.hd <= 32) return f16 ? launch_bwd<32, true>(st, a) : launch_bwd<32, false>(st, a);
    if (a.hd <= 64) return f16 ? launch_bwd<64, true>(st, a) : launch_bwd<64, false>(st, a);
    return f16 ? launch_bwd<128, true>(st, a) : launch_bwd<128, false>(st, a);
}

// ---------------------------------------------------------------- arguments
int mi_attn_buckets(const char* who, mi_attn_args* a, int buckets, int max_distance, int bidirectional)
{
    const int n = bidirectional ? buckets / 2 : buckets, m = n / 2;
    MI_REQUIRE(buckets >= (bidirectional ? 4 : 2) && buckets <= MI_ATTN_MAX_BUCKETS && (!bidirectional || buckets % 2 == 0),
               "%s: num_buckets %d must be %s, at most %d", who, buckets, bidirectional ? "even and at least 4" : "at least 2", MI_ATTN_MAX_BUCKETS);
    MI_REQUIRE(max_distance > m && max_distance <= MI_ATTN_MAX_DISTANCE, "%s: max_distance %d must be above %d (the distances with a bucket each) and at most %d",
               who, max_distance, m, MI_ATTN_MAX_DISTANCE);
    a->buckets = buckets;
    a->two_sided = bidirectional ? 1 : 0;
    a->side = n;
    a->exact = m;
    a->nborder = n - m - 1;
    // border t: the least whole d with d^(n - m) >= max_distance^t m^(n - m - t).  Found in floating point; a real border within
    // 1e-12 of a whole number (far below the distance of any other border from one, for these sizes) is that number.
    int reach = m;
    for (int t = 1; t <= a->nborder; ++t) {
        const double x = m * exp((double)t / (n - m) * log((double)max_distance / m));
        int d = (int)ceil(x * (1.0 - 1e-12));
        if (d < m) d = m;
        a->border[t - 1] = d;
        if (d > reach) reach = d;
    }
    a->reach = reach;
    return MI_OK;
}

static int fill_rows(const char* who, const char* what, const mi_attention_rows* r, int64_t tokens, int heads, int hd, mi_attn_rows* out)
{
    MI_REQUIRE(r && (r->ptr || tokens == 0), "%s: %s is NULL", who, what);
    MI_REQUIRE(((uintptr_t)r->ptr & 15) == 0, "%s: %s is not 16-byte aligned", who, what);
    MI_REQUIRE(r->token_stride % 8 == 0 && r->head_stride % 8 == 0, "%s: strides of %s (%lld, %lld) must be multiples of 8 elements", who, what,
               (long long)r->token_stride, (long long)r->head_stride);
    MI_REQUIRE(r->token_stride < ((int64_t)1 << 24), "%s: token stride of %s, %lld, is not below 2^24 elements", who, what, (long long)r->token_stride);
    MI_REQUIRE(r->token_stride >= 0 && r->head_stride >= 0 && (tokens <= 1 || r->token_stride >= hd) && (heads <= 1 || r->head_stride >= hd),
               "%s: strides of %s (%lld, %lld) let rows of %d elements overlap", who, what, (long long)r->token_stride, (long long)r->head_stride, hd);
    out->p = (uint16_t*)r->ptr;
    out->ts = r->token_stride;
    out->hs = r->head_stride;
    return MI_OK;
}

// Everything both directions check; fills the fields they share.
static int fill_args(const char* who, mi_ctx* ctx, const mi_attention_config* c, int64_t tokens, int64_t nseq, const int32_t* offsets,
                     const int32_t* key_mask, const mi_attention_rows* q, const mi_attention_rows* k, const mi_attention_rows* v,
                     const float* table, mi_attn_args* a)
{
    MI_REQUIRE(ctx && c, "%s: NULL argument", who);
    MI_REQUIRE(c->dtype == MI_DTYPE_BF16 || c->dtype == MI_DTYPE_F16, "%s: dtype %d is not MI_DTYPE_BF16 or MI_DTYPE_F16", who, c->dtype);
    MI_REQUIRE(c->heads > 0 && c->heads <= 65535 && c->kv_heads > 0 && c->heads % c->kv_heads == 0, "%s: heads %d must be a positive multiple of kv_heads %d", who, c->heads, c->kv_heads);
    MI_REQUIRE(c->head_dim > 0 && c->head_dim % 8 == 0 && c->head_dim <= 128, "%s: head_dim %d must be a multiple of 8 up to 128", who, c->head_dim);
    MI_REQUIRE(c->scale > 0.0f && c->scale <= FLT_MAX / 2, "%s: scale must be positive and finite", who);
    MI_REQUIRE(tokens >= 0 && tokens < ((int64_t)1 << 31) - 4096, "%s: %lld tokens out of range", who, (long long)tokens);
    MI_REQUIRE(nseq >= 0 && nseq < ((int64_t)1 << 24), "%s: %lld sequences out of range", who, (long long)nseq);
    MI_REQUIRE(offsets || (nseq == 0 ? tokens == 0 : tokens % nseq == 0), "%s: %lld tokens are not %lld sequences of one length", who, (long long)tokens, (long long)nseq);
    MI_TRY(fill_rows(who, "q", q, tokens, c->heads, c->head_dim, &a->q));
    MI_TRY(fill_rows(who, "k", k, tokens, c->kv_heads, c->head_dim, &a->k));
    MI_TRY(fill_rows(who, "v", v, tokens, c->kv_heads, c->head_dim, &a->v));
    if (c->num_buckets != 0) {
        MI_TRY(mi_attn_buckets(who, a, c->num_buckets, c->max_distance, c->bidirectional));
        MI_REQUIRE(table, "%s: num_buckets is %d and bias_table is NULL", who, c->num_buckets);
    } else {
        MI_REQUIRE(!table, "%s: a bias_table without buckets", who);
    }
    a->table = table;
    a->offsets = offsets;
    a->key_mask = key_mask;
    a->tokens = tokens;
    a->nseq = (int)nseq;
    a->uniform_len = offsets || nseq == 0 ? 0 : (int)(tokens / nseq);
    a->heads = c->heads;
    a->group = c->heads / c->kv_heads;
    a->hd = c->head_dim;
    a->causal = c->causal != 0;
    a->zero_tail = c->zero_tail != 0;
    a->scale = c->scale;
    a->scale_log2 = c->scale * AT_LOG2E;
    // one launch: heads x tiles of at least 64 rows, below 2^31 blocks
    MI_REQUIRE((tokens / 64 + nseq + 9) * (int64_t)c->heads < ((int64_t)1 << 31) - 1, "%s: %lld tokens x %d heads are too many for one call", who, (long long)tokens, c->heads);
    return MI_OK;
}

extern "C" int mi_attention_dev(mi_ctx* ctx, const mi_attention_config* cfg, int64_t tokens, int64_t nseq, const int32_t* offsets_dev,
                                const int32_t* key_mask_dev, const mi_attention_rows* q, const mi_attention_rows* k,
                                const mi_attention_rows* v, const float* bias_table_dev, const mi_attention_rows* out, float* lse_dev,
                                void* stream)
{
    mi_attn_args a;
    MI_TRY(fill_args("mi_attention_dev", ctx, cfg, tokens, nseq, offsets_dev, key_mask_dev, q, k, v, bias_table_dev, &a));
    MI_TRY(fill_rows("mi_attention_dev", "out", out, tokens, cfg->heads, cfg->head_dim, &a.out));
    if (tokens == 0) return MI_OK;
    a.lse = lse_dev;
    DeviceGuard guard(mi_ctx_device(ctx));
    return mi_launch_attention(mi_pick_stream(stream, mi_ctx_stream(ctx)), a, cfg->dtype);
}

extern "C" int mi_attention_backward_workspace(const mi_attention_config* cfg, int64_t tokens, int64_t nseq, int packed, size_t* bytes)
{
    MI_REQUIRE(cfg && bytes, "mi_attention_backward_workspace: NULL argument");
    MI_REQUIRE(cfg->heads > 0 && cfg->kv_heads > 0 && cfg->heads % cfg->kv_heads == 0 && cfg->head_dim > 0 && tokens >= 0 && nseq >= 0 && (packed || nseq == 0 || tokens % nseq == 0), "mi_attention_backward_workspace: bad argument");
    mi_attn_args a;
    static const int32_t some = 0;
    static const float one = 0.0f;
    if (cfg->num_buckets != 0) {
        MI_TRY(mi_attn_buckets("mi_attention_backward_workspace", &a, cfg->num_buckets, cfg->max_distance, cfg->bidirectional));
        a.table = &one;
    }
    a.offsets = packed ? &some : nullptr;
    a.heads = cfg->heads;
    a.group = cfg->heads / cfg->kv_heads;
    a.hd = cfg->head_dim;
    a.tokens = tokens;
    a.nseq = (int)nseq;
    a.uniform_len = packed || nseq == 0 ? 0 : (int)(tokens / nseq);
    *bytes = mi_attn_backward_bytes(a);
    return MI_OK;
}

extern "C" int mi_attention_backward_dev(mi_ctx* ctx, const mi_attention_config* cfg, int64_t tokens, int64_t nseq,
                                         const int32_t* offsets_dev, const int32_t* key_mask_dev, const mi_attention_rows* q,
                                         const mi_attention_rows* k, const mi_attention_rows* v, const float* bias_table_dev,
                                         const mi_attention_rows* out, const float* lse_dev, const mi_attention_rows* dout,
                                         const mi_attention_rows* dq, const mi_attention_rows* dk, const mi_attention_rows* dv,
                                         float* dbias_table_dev, void* workspace_dev, size_t workspace_bytes, void* stream)
{
    const char* who = "mi_attention_backward_dev";
    mi_attn_args a;
    MI_TRY(fill_args(who, ctx, cfg, tokens, nseq, offsets_dev, key_mask_dev, q, k, v, bias_table_dev, &a));
    MI_TRY(fill_rows(who, "out", out, tokens, cfg->heads, cfg->head_dim, &a.out));
    MI_TRY(fill_rows(who, "dout", dout, tokens, cfg->heads, cfg->head_dim, &a.dout));
    MI_TRY(fill_rows(who, "dq", dq, tokens, cfg->heads, cfg->head_dim, &a.dq));
    MI_TRY(fill_rows(who, "dk", dk, tokens, cfg->kv_heads, cfg->head_dim, &a.dk));
    MI_TRY(fill_rows(who, "dv", dv, tokens, cfg->kv_heads, cfg->head_dim, &a.dv));
    MI_REQUIRE(tokens == 0 || lse_dev, "%s: lse is NULL (the forward pass writes it)", who);
    MI_REQUIRE(!bias_table_dev == !dbias_table_dev, "%s: dbias_table goes with bias_table", who);
    const size_t need = mi_attn_backward_bytes(a);
    MI_REQUIRE(need == 0 || (workspace_dev && ((uintptr_t)workspace_dev & 255) == 0), "%s: workspace is NULL or not 256-byte aligned", who);
    MI_REQUIRE(workspace_bytes >= need, "%s: workspace of %zu bytes, %zu are needed", who, workspace_bytes, need);
    a.lse = const_cast<float*>(lse_dev);
    a.dtable = dbias_table_dev;
    DeviceGuard guard(mi_ctx_device(ctx));
    return mi_launch_attention_backward(mi_pick_stream(stream, mi_ctx_stream(ctx)), a, cfg->dtype, workspace_dev);
}

extern "C" int mi_attention_buckets(int num_buckets, int max_distance, int bidirectional, int64_t n, const int64_t* rel, int32_t* out)
{
    MI_REQUIRE(n >= 0 && (n == 0 || (rel && out)), "mi_attention_buckets: NULL argument");
    mi_attn_args a;
    MI_TRY(mi_attn_buckets("mi_attention_buckets", &a, num_buckets, max_distance, bidirectional));
    for (int64_t i = 0; i < n; ++i) {
        const int64_t far = 2 * MI_ATTN_MAX_DISTANCE, r = rel[i] < -far ? -far : rel[i] > far ? far : rel[i];
        out[i] = at_bucket(a, (int)r);
    }
    return MI_OK;
}
