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
#include <type_traits>
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

template <int V> using at_int = std::integral_constant<int, V>;
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
// Grid: x = 8 XCDs x the XCD's units, y and z = a unit's tiles, so nothing is divided, and the units of an XCD take the same tiles
// at the same time: the heads of a key head share K and V, neighbouring heads of 32 cache lines.  (All tiles of a unit
// before the next: 13 causal prompts up to 2,039, 32 heads on 8 of 128, 92 -> 77 us; 24 passages, 12 heads of 64, dQ 65 -> 61 us.)
__device__ __forceinline__ int at_unit(const mi_attn_args& p) { return (blockIdx.x & 7) * p.units_per_xcd + (blockIdx.x >> 3); }
__device__ __forceinline__ bool at_work(const mi_attn_args& p, int& head, int& t)
{
    const int u = at_unit(p);
    head = u >> p.parts_log2;
    t = (int)((blockIdx.z * gridDim.y + blockIdx.y) << p.parts_log2) + (u & ((1 << p.parts_log2) - 1));
    return t < p.tiles;
}
// x / d for x < 2^16 and m = ceil(2^32 / d)
__device__ __forceinline__ int at_div(int x, uint32_t m) { return m ? (int)__umulhi((uint32_t)x, m) : x; }

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

// A pointer that is the same on every lane, in scalar registers (hipcc may have moved it to vector ones)
__device__ __forceinline__ const char* at_uniform(const char* x)
{
    const uint64_t u = (uint64_t)x;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
    return (const char*)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ void at_dma16(const void* src, unsigned lds_addr)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(src), "s"(lds_addr) : "memory", "m0");
}
__device__ __forceinline__ void at_dma4(const void* src, unsigned lds_addr)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" :: "v"(src), "s"(lds_addr) : "memory", "m0");
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
    const char* at;                                   // the next tile's row 0 (uniform): tiles are requested in order
    int pitch;                                        // bytes between rows
    int row0, chunk;                                  // this lane's row in instruction 0 and its bytes in the row
    unsigned off;
    int left;                                         // rows from `at` to the sequence's last one
    __device__ __forceinline__ void init(const mi_attn_rows& x, int start, int first, int len, int head, int hd, int wave, int lane)
    {
        row0 = wave * RPI + lane / LPR;
        int c = (lane % LPR) ^ AtTile<DP>::f(row0);
        const int most = (hd >> 3) - 1;
        chunk = (c < most ? c : most) * 16;
        at = at_uniform(reinterpret_cast<const char*>(x.p + (int64_t)(start + first) * x.ts + (int64_t)head * x.hs));
        pitch = __builtin_amdgcn_readfirstlane((int)(x.ts * 2));
        off = (unsigned)(row0 * pitch + chunk);
        left = len - 1 - first;
    }
    // the next 64 rows to lds_addr; keys: which of them are keys
    __device__ __forceinline__ void issue(unsigned lds_addr, int wave, uint64_t keys = ~0ull)
    {
        lds_addr += wave * 1024;
        if (keys == ~0ull && left >= AT_KT - 1) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                at_dma16(off, at, lds_addr + (unsigned)(i * NW * 1024));
                at += RPI * NW * pitch;               // (below 2^31)
            }
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = row0 + i * RPI * NW, row = r < left ? r : left;
                const char* src = at + (int64_t)row * pitch + chunk;
                if (!((keys >> r) & 1)) src = reinterpret_cast<const char*>(&at_zero_chunk);
                at_dma16(src, lds_addr + (unsigned)(i * NW * 1024));
            }
            at += (int64_t)AT_KT * pitch;
        }
        left -= AT_KT;
    }
};
// Everything a wave issued but its last AHEAD x PER loads has landed and what it read from LDS is in registers, on every wave.
template <int PER>
__device__ __forceinline__ void at_arrive(int ahead)
{
    if (ahead >= 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * PER) : "memory");
    else if (ahead == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PER) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// everything outstanding has landed and been read, on every wave
__device__ __forceinline__ void at_sync()
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// Which keys of a sequence the mask leaves, 64 a word.  The block reads the mask once, ahead of everything: so tiles without a key
// are left out at the end (a padded batch's padding) and whole ones in front take the code without a mask.
#define AT_WORDS 256                                  // tiles whose words are kept; later ones are asked for as they come
struct AtKeys {
    const int32_t* mask;                              // from the sequence's first row on, or NULL
    const uint64_t* words;
    int len, lane;
    int full, some;                                   // leading tiles of 64 keys each; tiles up to the last one with a key
    __device__ __forceinline__ uint64_t load(int t) const
    {
        const int key = t * AT_KT + lane;
        return __builtin_amdgcn_ballot_w64(key < len && mask[key < len ? key : len - 1] != 0);
    }
    __device__ __forceinline__ uint64_t tile(int t) const
    {
        if (!mask) return ~0ull;
        if (t >= AT_WORDS) return load(t);
        const uint64_t w = words[t];
        return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(w >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)w);
    }
    // waves: of the block, all of them call
    __device__ __forceinline__ void init(const int32_t* key_mask, uint64_t* w, int start, int n, int kend, int wave, int waves, int l)
    {
        mask = key_mask ? key_mask + start : nullptr;
        words = w;
        len = n;
        lane = l;
        some = (kend + AT_KT - 1) / AT_KT;
        full = some;
        if (!mask) return;
        const int tiles = some < AT_WORDS ? some : AT_WORDS;
        for (int t = wave; t < tiles; t += waves) {
            const uint64_t k = load(t);
            if (lane == 0) w[t] = k;
        }
        at_sync();
        full = 0;
        int last = 0;
        for (int t = 0; t < tiles; t += 64) {
            const uint64_t k = t + lane < tiles ? w[t + lane] : 0;
            const uint64_t whole = __builtin_amdgcn_ballot_w64(k == ~0ull), any = __builtin_amdgcn_ballot_w64(k != 0);
            if (full == t) full += ~whole ? __builtin_ctzll(~whole) : 64;
            if (any) last = t + 64 - __builtin_clzll(any);
        }
        if (some <= AT_WORDS) some = last;
    }
};
// The K and V tiles of a sequence through NB pairs of buffers: tile t + NB - 1 is requested when every wave is done with tile t - 1.
// (With two buffers a tile has one tile's computing to arrive, about 0.5 us at head size 32, and memory takes longer.)
template <int DP, int NB> struct AtPipe {
    static constexpr int PAIR = 2 * AtTile<DP>::BYTES, BYTES = NB * PAIR, PER = 2 * AtStage<DP, 4>::NI;
    AtStage<DP, 4> a, b;
    AtKeys* keys;
    unsigned lds0;
    int n, wave, buf;
    __device__ __forceinline__ void issue(int t, int slot)
    {
        const uint64_t k = keys->tile(t);
        a.issue(lds0 + slot * PAIR, wave, k);
        b.issue(lds0 + slot * PAIR + PAIR / 2, wave, k);
    }
    __device__ __forceinline__ void start(const char* lds, AtKeys* k, int w)
    {
        lds0 = (unsigned)(size_t)(const __attribute__((address_space(3))) char*)lds;
        n = k->some;
        keys = k;
        wave = w;
        buf = NB - 1;
#pragma unroll
        for (int t = 0; t < NB - 1; ++t) if (t < n) issue(t, t);
    }
    // tile t has landed; returns its place
    __device__ __forceinline__ int next(int t)
    {
        const int left = n - 1 - t;
        at_arrive<PER>(left < NB - 2 ? left : NB - 2);
        if (t + NB - 1 < n) issue(t + NB - 1, buf);                    // over tile t - 1
        buf = buf + 1 == NB ? 0 : buf + 1;
        return buf * PAIR;
    }
};
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
// stays inside it, any other tile lies in one bucket.  Values are times `unit`: log2(e), to be added to scaled scores, or 1 / scale, to be
// the C operand of a score block's first product.
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
        for (int t = 0; t < p.nborder; t += 8)                         // (the array ends in values beyond any distance)
#pragma unroll
            for (int j = 0; j < 8; ++j) b += d >= p.border[t + j] ? 1 : 0;
    }
    return b + (p.two_sided && r > 0 ? p.side : 0);
}
__device__ __forceinline__ float at_bias(const mi_attn_args& p, int head, int r, float unit)
{
    const float x = p.table[(int64_t)at_bucket(p, r) * p.heads + head];
    return (fabsf(x) <= FLT_MAX ? fminf(fmaxf(x, -AT_BIAS_MOST), AT_BIAS_MOST) : x) * unit;
}
__device__ __forceinline__ void at_fill_bias(const mi_attn_args& p, int head, float unit, float shift, float* vec)
{
    const int R = p.reach + AT_PAD;
    for (int i = threadIdx.x; i < 2 * R + 1; i += blockDim.x) vec[i] = at_bias(p, head, i - R, unit) + shift;
}

// Calls f(i, attended) for the registers of a block of scores, 32 keys from k on, one query a lane (register 4 g + i is key
// k + 8 g + 4 half + i), where not all are attended; keys: the block's keys (all, without a mask).
template <class F>
__device__ __forceinline__ void at_unattended(const mi_attn_args& p, bool mask, uint32_t keys, int k, int qw, int q, int len, int half, F&& f)
{
    if (k + 32 <= len && !(p.causal && k + 31 > qw) && keys == 0xFFFFFFFFu) return;
    int lim = len - 1 - k;                                             // the last attended key but for the mask
    if (p.causal && q - k < lim) lim = q - k;
    lim -= 4 * half;
    if (mask) {
        uint32_t ok = keys >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) f(i, 8 * (i >> 2) + (i & 3) <= lim && ((ok >> (8 * (i >> 2) + (i & 3))) & 1u));
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) f(i, 8 * (i >> 2) + (i & 3) <= lim);
    }
}

// The first of a score block's products, on the bias where it is not one value for the tile: 8 g + i steps on from bv
template <bool F16>
__device__ __forceinline__ f32x16 at_first(bool near, const float* bv, int step, u32x4 a, u32x4 b)
{
    if (near) {
        f32x16 C;
#pragma unroll
        for (int i = 0; i < 16; ++i) C[i] = bv[step * (8 * (i >> 2) + (i & 3))];
        return at_mfma<F16>(a, b, C);
    }
    return at_mfma<F16>(a, b, at_zero16());
}

// ---------------------------------------------------------------- forward
#define AT_BUFFERS(DP) ((DP) == 32 ? 4 : (DP) == 64 ? 3 : 2)          // what leaves LDS for as many blocks as the registers do
// One block per (head, 128 / KS query rows): four waves, each 32 queries by every KS-th 32-key block of the K and V tiles, which come by
// LDS-DMA, 64 keys at a time, one barrier per tile.  With KS = 2 the two waves of a query join their sums through LDS at the end:
// half the time per tile and twice the blocks, for calls of few blocks.  Bound: head size 128 by the products (16,384 tokens causal, 16
// heads on 2, 1,061 us, 1,036 TFLOP/s of the 1,127 a large fp16 product reaches), 32 and 64 by the exponentials and what
// goes with them (400 chunks up to 256 tokens, 12 heads of 32, bias: 68 us; 64 x 512 padded, 12 heads of 64: 67 us).
template <int DP, bool F16, bool BIAS, int KS>
__global__ __launch_bounds__(256, DP == 32 ? 4 : DP == 64 ? 3 : 2) void attn_fwd_kernel(const mi_attn_args p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int BM = 128 / KS, TB = AtTile<DP>::BYTES, NS = 2 / KS, NB = AT_BUFFERS(DP);
    float* const vec = reinterpret_cast<float*>(lds + NB * 2 * TB);
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
    const int qw = tile * BM + (KS == 1 ? wave : wave & 1) * 32, q = qw + col;   // this wave's queries
    const int s0 = KS == 1 ? 0 : wave >> 1;                            // its first 32-key block of a tile
    const int kend = p.causal ? (tile * BM + BM < len ? tile * BM + BM : len) : len;

    u32x4 qf[DP / 16];
    at_load_rows<DP>(qf, p.q, start + (q < len ? q : len - 1), head, p.hd, half);
    const int kvh = at_div(head, p.group_inv);
    __shared__ uint64_t words[AT_WORDS];
    AtKeys keys;
    keys.init(p.key_mask, words, start, len, kend, wave, 4, lane);
    const bool mask = keys.mask != nullptr;
    AtPipe<DP, NB> pipe;
    pipe.a.init(p.k, start, 0, len, kvh, p.hd, wave, lane);
    pipe.b.init(p.v, start, 0, len, kvh, p.hd, wave, lane);
    pipe.start(lds, &keys, wave);
    if constexpr (BIAS) at_fill_bias(p, head, AT_LOG2E, F16 ? 8.0f : 0.0f, vec);

    f32x16 O[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) O[dt] = at_zero16();
    // the reference starts at a usual place and stays while the first tile's maximum lies within 2^8 of it; bf16 has fp32's range,
    // fp16 takes it 2^8 lower so that the sum is at least 1, and p up to 2^15
    constexpr float REF0 = F16 ? -8.0f : 0.0f, HIGH = F16 ? 15.0f : 8.0f, LOW = F16 ? 0.0f : -8.0f;
    // Rows of up to 64 keys take their maximum: its p is then 1, which rounding to 16 bits leaves, and a row of one key is that key's
    // v (sequences of a few tokens: out 1.1 - 1.2 x as far off as its own rounding alone; from the fixed reference 1.4 - 1.6; the first rows
    // of 16,384 causal ones are half of its error, too: 1.45 -> 1.3).
    const float high = (p.causal && qw + 32 < kend ? qw + 32 : kend) <= AT_KT ? -INFINITY : HIGH;
    float m = 0.0f, low = LOW, l = 0.0f;                               // reference = REF0 + m; low = -inf once a finite score has been seen
    bool moved = false;                                                // some lane's m is not 0
    const int R = p.reach + AT_PAD;
    const float c = p.scale_log2;
    // One tile, in the forms that the loops below need: with and without unattended keys, with the bias one value (FAR) or many,
    // from which m is taken or, while it is 0 on every lane, not.  Each is a straight run of code in a loop of its own: where
    // forms meet in one loop hipcc copies O for each.
    constexpr int FAR = 0, NEAR0 = 1, NEARM = 2;
    auto compute = [&](auto masked_, auto form_, int k0, const char* Kt) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked_)::value;
        constexpr int FORM = decltype(form_)::value;
        const int kw = k0 + 32 * s0;
        const uint64_t on = MASKED ? keys.tile(k0 / AT_KT) : 0;
        const float less = BIAS ? vec[kw < qw ? 0 : 2 * R] - m : -REF0 - m;
        f32x16 S[NS];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) S[n] = at_mfma<F16>(at_rows<DP>(Kt, s0 + n, s, col, half), qf[s], s == 0 ? at_zero16() : S[n]);
        const float* const bv = vec + (kw + 4 * half - q + R);         // (less the reference's start)
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            int lim = 0;                                               // the last attended key but for the mask
            uint32_t ok = 0;
            if constexpr (MASKED) {
                lim = len - 1 - kw - 32 * n;
                if (p.causal && q - kw - 32 * n < lim) lim = q - kw - 32 * n;
                lim -= 4 * half;
                ok = (uint32_t)(on >> (32 * (s0 + n))) >> (4 * half);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = 8 * (i >> 2) + (i & 3);
                S[n][i] = __builtin_fmaf(S[n][i], c, FORM == FAR ? less : FORM == NEARM ? bv[32 * n + r] - m : bv[32 * n + r]);
                if constexpr (MASKED) S[n][i] = r <= lim && (!mask || ((ok >> r) & 1u)) ? S[n][i] : -INFINITY;
            }
        }
        float top = S[0][0];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int i = n == 0 ? 1 : 0; i + 1 < 16; i += 2) top = at_max3(top, S[n][i], S[n][i + 1]);
        top = fmaxf(top, S[0][15]);
        if (__builtin_amdgcn_ballot_w64(top > high || top < low) != 0) {
            top = fmaxf(top, at_other_half(top));                      // both halves of a query move alike
            low = fminf(low, at_other_half(low));
            const bool move = top > high || (top < low && top > -INFINITY);
            const float up = move ? top : 0.0f;
            const float alpha = low > -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(-up);   // (nothing summed before the first)
            m += up;
            moved = true;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) O[dt] = O[dt] * alpha;
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) S[n][i] -= up;
        }
        low = top > -INFINITY ? -INFINITY : low;
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                S[n][i] = __builtin_amdgcn_exp2f(S[n][i]);
                l += S[n][i];
            }
#pragma unroll
        for (int kk = 0; kk < 2 * NS; ++kk) {
            u32x4 pf;
#pragma unroll
            for (int i = 0; i < 4; ++i) pf[i] = at_pack2<F16>(S[kk >> 1][8 * (kk & 1) + 2 * i], S[kk >> 1][8 * (kk & 1) + 2 * i + 1]);
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) O[dt] = at_mfma<F16>(at_cols<DP>(Kt + TB, 2 * s0 + kk, dt, lane), pf, O[dt]);
        }
    };
    // tiles: [0, far0) all before the bias's reach, [far0, far1) within it, [far1, plain) behind it, [plain, live) with unattended
    // keys, [live, all) nothing for this wave but the barriers
    const int all = pipe.n, lim = p.causal && qw + 1 < len ? qw + 1 : len;
    int live = 0, plain = 0, far0 = 0, far1 = 0;
    if (qw < len) {
        const int end = p.causal && qw + 32 < kend ? qw + 32 : kend;
        live = end <= 32 * s0 ? 0 : (end - 32 * s0 + AT_KT - 1) / AT_KT;
        if (live > all) live = all;
        plain = lim < 32 * (NS + s0) ? 0 : (lim - 32 * (NS + s0)) / AT_KT + 1;
        if (plain > live) plain = live;
        if (mask && plain > keys.full) plain = keys.full;
        if constexpr (BIAS) {
            const int x = qw - p.reach - 32 * (NS + s0) + 1, y = qw + 31 + p.reach - 32 * s0;   // before: k0 <= x; behind: k0 >= y
            far0 = x < 0 ? 0 : x / AT_KT + 1;
            far1 = (y + AT_KT - 1) / AT_KT;
        }
    }
    const int end0 = BIAS ? (far0 < plain ? far0 : plain) : plain, end1 = far1 < plain ? far1 : plain;
    auto run = [&](auto masked_, auto form_, int t) __attribute__((always_inline)) { compute(masked_, form_, t * AT_KT, lds + pipe.next(t)); };
    using std::false_type;
    using std::true_type;
    int t2 = 0;
    for (; t2 < end0; ++t2) run(false_type{}, at_int<FAR>{}, t2);
    if constexpr (BIAS) {
        for (; t2 < end1 && !moved; ++t2) run(false_type{}, at_int<NEAR0>{}, t2);
        for (; t2 < end1; ++t2) run(false_type{}, at_int<NEARM>{}, t2);
        for (; t2 < plain; ++t2) run(false_type{}, at_int<FAR>{}, t2);
        for (; t2 < live; ++t2) {
            if (t2 < far0 || t2 >= far1) run(true_type{}, at_int<FAR>{}, t2);
            else run(true_type{}, at_int<NEARM>{}, t2);
        }
    } else {
        for (; t2 < live; ++t2) run(true_type{}, at_int<FAR>{}, t2);
    }
    for (; t2 < all; ++t2) (void)pipe.next(t2);
    float sum = l + at_other_half(l);
    if constexpr (KS == 2) {
        // waves 2 and 3 hand over reference, sum and O; rows of 64 lanes, one register each
        low = fminf(low, at_other_half(low));
        at_sync();
        float* const x = reinterpret_cast<float*>(lds) + (wave & 1) * (DP / 2 + 3) * 64 + lane;
        if (wave >= 2) {
            x[0] = m;
            x[64] = sum;
            x[128] = low;
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[(3 + 16 * dt + i) * 64] = O[dt][i];
        }
        at_sync();
        if (wave >= 2) return;
        const float m2 = x[0], sum2 = x[64], low2 = x[128];
        // a side without a finite score has summed nothing (or NaN): the other side's reference stands
        const float mm = low > -INFINITY ? m2 : low2 > -INFINITY ? m : fmaxf(m, m2);
        const float f1 = low > -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mm), f2 = low2 > -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m2 - mm);
        m = mm;
        sum = sum * f1 + sum2 * f2;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) O[dt][i] = O[dt][i] * f1 + x[(3 + 16 * dt + i) * 64] * f2;
    }
    if (q < len) {
        at_store_row<DP, F16>(p.out, start + q, head, p.hd, half, O, sum == 0.0f ? 0.0f : 1.0f / sum);
        if (p.lse && half == 0)
            p.lse[(int64_t)head * p.tokens + start + q] = sum == 0.0f ? -INFINITY : (REF0 + m + __builtin_amdgcn_logf(sum)) * AT_LN2;
    }
}

// ---------------------------------------------------------------- backward
// P is rebuilt from the saved log-sum-exp.  fp16 only: p is scaled by 2^12 on its way into the 16-bit operand of dV (a row of
// thousands of keys has p near fp16's subnormals), and ds = p (dp - D) takes the scale back out.
template <bool F16> struct AtPScale { static constexpr float log2 = F16 ? 12.0f : 0.0f, down = F16 ? 1.0f / 4096.0f : 1.0f; };

// the largest of a block's 16 sizes (three steps deep: as one chain of eight it held up the short calls)
__device__ __forceinline__ float at_size(const f32x16& x)
{
    float m[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) m[i] = at_max3(fabsf(x[3 * i]), fabsf(x[3 * i + 1]), fabsf(x[3 * i + 2]));
    return fmaxf(at_max3(m[0], m[1], m[2]), at_max3(m[3], m[4], fabsf(x[15])));
}

// The power of two that ds is carried with into the 16-bit operand of dQ and dK, fp16 only: with dout as a loss's mean leaves it (1e-3,
// 4,096 keys) ds lies in fp16's subnormals and its rounding was 8 times the result's own; with large v and dout it is beyond 65,504.  One
// power for each lane's sum (a query's dQ, a key's dK).  It starts where no ds that counts is lost, and where a block's largest would pass
// 2^15 with it, it falls to put that at 2^10 .. 2^11: at a lane's first block, and then for a ds 2^5 times as large as any before.  So a ds
// is off by 2^-11 of itself or by 2^-35 of the lane's largest.  (Bounded by |dp - D| instead, which is there earlier, the rows and keys
// whose p are all tiny would lose theirs.)  bf16 has fp32's range and does without.  The check costs the fp16 kernels 1 - 7 % (24 passages up
// to 511, 12 heads of 64, bias: dQ 62.5 -> 64.6 us, dK / dV 40.5 -> 41.8; 9 prompts up to 2,048, 16 heads on 4 of 128: 117 -> 121).
template <bool F16> struct AtDsScale {
    static constexpr float START = F16 ? 0x1p60f : 1.0f;               // (|dp| < 2^41: finite)
    float up = START;
    // ds: N blocks, times `up` already.  What the lane has summed goes along, and also(f) takes the change to what makes the next ds.
    template <int N, int M, class Also>
    __device__ __forceinline__ void fit(f32x16 (&ds)[N], f32x16 (&sum)[M], Also&& also)
    {
        if constexpr (F16) {
            float top = at_size(ds[0]);
#pragma unroll
            for (int n = 1; n < N; ++n) top = fmaxf(top, at_size(ds[n]));
            if (__builtin_amdgcn_ballot_w64(top > 0x1p15f) != 0) {
                top = fmaxf(top, at_other_half(top));                  // both halves of a lane's sum move alike
                const float f = top > 0x1p15f && top < INFINITY ? __builtin_amdgcn_ldexpf(0x1p11f, -__builtin_amdgcn_frexp_expf(top)) : 1.0f;
                up *= f;
#pragma unroll
                for (int n = 0; n < N; ++n) ds[n] = ds[n] * f;
#pragma unroll
                for (int m = 0; m < M; ++m) sum[m] = sum[m] * f;
                also(f);
            }
        }
    }
    // the sum without the power
    template <int M> __device__ __forceinline__ void down(f32x16 (&sum)[M], float f = 1.0f) const
    {
        if constexpr (F16) {
            f /= up;
#pragma unroll
            for (int m = 0; m < M; ++m) sum[m] = sum[m] * f;
        }
    }
};

#define AT_DQ_BUFFERS(DP, BIAS) ((BIAS) ? ((DP) == 32 ? 3 : 2) : AT_BUFFERS(DP))
// dQ: one block per (head, 128 query rows), like the forward pass: S^T = K Q^T and dP^T = V dO^T with the query on the lane,
// dQ^T += K^T dS^T, with ds = p (dp - D).
//
// D = sum_j p dp of a row.  rowsum(dout * out) is the same sum, but takes over the rounding of p and out in the forward pass,
// which shows in rows of few keys (20 causal rows: dq and dk 1.65 x the plain rounding of their values, 1.4 with D exact) and in
// the table's gradient, a sum of many ds that nearly cancel.  So with a bias, for rows of up to 128 keys, and for up to 512 where
// a mask may leave few of them, a first pass over the keys makes the sum from the scores, in fp32 (its tiles are still in LDS for
// the second where they fit); other rows take the dot product.  D and the rows' log-sum-exp in log2 units, +inf for a row that
// attends nothing, are left for the dK / dV kernel.  A kernel of its own for D
// was slower: 8 queries of 5 - 31 tokens (12 heads of 32, bias) 14.3 -> 10.2 us, 96 chunks up to 256 67 -> 59, 24 passages up to 511
// (12 x 64) 73 -> 65, 9 causal prompts up to 2,048 (16 x 128, no bias) 87 -> 78.
//
// BIAS: the table's gradient is the sum of ds along the diagonals r = key - query.  A 32 x 32 block of ds goes through a skewed
// image in LDS, element (key, query) at [query][key - query + 31], so that lane l finds a diagonal in column l (the positions a row
// never writes hold the zeros they started with); the 63 sums are added to the wave's vector over r.  A tile of one bucket adds
// in registers.  Every sum has one owner and a fixed order.  (LDS float atomics, the direct form, took 122 clocks a wave instruction;
// diagonals as rows of 36 floats, read 16 bytes a lane, the same time.)
template <int DP, bool F16, bool BIAS, int KS>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(const mi_attn_args p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int BM = 128 / KS, TB = AtTile<DP>::BYTES, NB = AT_DQ_BUFFERS(DP, BIAS);
    const int R = p.reach + AT_PAD, nvec = 2 * R + 1;
    float* const skew0 = reinterpret_cast<float*>(lds + NB * 2 * TB);       // BIAS: [4][32][64], the waves' images
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
    const int qw = tile * BM + (KS == 1 ? wave : wave & 1) * 32, q = qw + col, s0 = KS == 1 ? 0 : wave >> 1;   // as in attn_fwd_kernel
    const int kend = p.causal ? (tile * BM + BM < len ? tile * BM + BM : len) : len;
    const int kvh = at_div(head, p.group_inv);

    __shared__ uint64_t words[AT_WORDS];
    __shared__ float pair[4][2][64];
    AtKeys keys;
    keys.init(p.key_mask, words, start, len, kend, wave, 4, lane);
    const bool mask = keys.mask != nullptr;
    AtPipe<DP, NB> pipe;
    pipe.a.init(p.k, start, 0, len, kvh, p.hd, wave, lane);
    pipe.b.init(p.v, start, 0, len, kvh, p.hd, wave, lane);
    pipe.start(lds, &keys, wave);

    u32x4 qf[DP / 16], df[DP / 16];
    const int64_t tok = start + (q < len ? q : len - 1);
    at_load_rows<DP>(qf, p.q, tok, head, p.hd, half);
    at_load_rows<DP>(df, p.dout, tok, head, p.hd, half);
    float nl = p.lse[(int64_t)head * p.tokens + tok] * AT_LOG2E;
    if (nl == -INFINITY || q >= len) nl = INFINITY;                    // p = 0

    float* const skew = skew0 + wave * 32 * 64;
    float* const dvec = dvec0 + wave * nvec;
    float farS[2] = {0.0f, 0.0f};                                      // sums of the tiles of one bucket, before and behind
    if constexpr (BIAS) {
        at_fill_bias(p, head, p.scale_inv, 0.0f, vec);
#pragma unroll
        for (int i = 0; i < 32; ++i) skew[i * 64 + lane] = 0.0f;
        for (int i = lane; i < nvec; i += 64) dvec[i] = 0.0f;
    }

    // calls use(tile, K tile, 32-key block, p, dp, ...) with p = 0 and dp = 0 where a key is not attended
    auto walk = [&](auto use) __attribute__((always_inline)) {
        for (int k0 = 0; k0 < pipe.n * AT_KT; k0 += AT_KT) {
            const char* const Kt = lds + pipe.next(k0 / AT_KT);
            if (qw >= len || (p.causal && k0 + 32 * s0 > qw + 31)) continue;
            const uint64_t on = keys.tile(k0 / AT_KT);
            const int rlo = k0 - (qw + 31), rhi = k0 + AT_KT - 1 - qw;
            const bool near = BIAS && rhi > -p.reach && rlo < p.reach;
            const float far = BIAS && !near ? __builtin_fmaf(vec[rhi <= -p.reach ? 0 : 2 * R], p.scale_log2, -nl) : -nl;
            const float* const bv = vec + (k0 + 4 * half - q + R);
#pragma unroll
            for (int st = s0; st < (KS == 1 ? 2 : s0 + 1); ++st) {
                if (st > 0 && (k0 + 32 >= kend || (p.causal && k0 + 32 > qw + 31))) break;
                f32x16 S = at_first<F16>(near, bv + 32 * st, 1, at_rows<DP>(Kt, st, 0, col, half), qf[0]), dP = at_zero16();
#pragma unroll
                for (int s = 1; s < DP / 16; ++s) S = at_mfma<F16>(at_rows<DP>(Kt, st, s, col, half), qf[s], S);
#pragma unroll
                for (int s = 0; s < DP / 16; ++s) dP = at_mfma<F16>(at_rows<DP>(Kt + TB, st, s, col, half), df[s], dP);
#pragma unroll
                for (int i = 0; i < 16; ++i) S[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], p.scale_log2, far));
                at_unattended(p, mask, (uint32_t)(on >> (32 * st)), k0 + 32 * st, qw, q, len, half, [&](int i, bool yes) __attribute__((always_inline)) {
                    S[i] = yes ? S[i] : 0.0f;
                    dP[i] = yes ? dP[i] : 0.0f;
                });
                use(Kt, st, S, dP, near, rlo, rhi);
            }
        }
    };

    float D = 0.0f, fix = 1.0f;                                        // fix: over the sum of p as it is rebuilt (the saved log-sum-exp is off by up to 5e-7)
    if (!BIAS && kend > (mask ? 512 : 128)) {
        u32x4 of[DP / 16];
        at_load_rows<DP>(of, p.out, tok, head, p.hd, half);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                D = __builtin_fmaf(at_lo<F16>(df[s][j]), at_lo<F16>(of[s][j]), D);
                D = __builtin_fmaf(at_hi<F16>(df[s][j]), at_hi<F16>(of[s][j]), D);
            }
        D += at_other_half(D);
    } else {
        float c = 0.0f;
        walk([&](const char*, int, const f32x16& S, const f32x16& dP, bool, int, int) __attribute__((always_inline)) {
            float a1 = 0.0f, c1 = 0.0f;                                // (short chains: a long row's sums stay exact to fp32's last bits)
#pragma unroll
            for (int i = 0; i < 16; ++i) { a1 = __builtin_fmaf(S[i], dP[i], a1); c1 += S[i]; }
            D += a1;
            c += c1;
        });
        D += at_other_half(D);
        c += at_other_half(c);
        if (KS == 2) {
            pair[wave][0][lane] = D;
            pair[wave][1][lane] = c;
        }
        at_sync();                                                     // (every wave is done with the tiles)
        if (KS == 2) {
            D += pair[wave ^ 2][0][lane];
            c += pair[wave ^ 2][1][lane];
        }
        if (c != 0.0f) fix = 1.0f / c;
        D *= fix;
        if (pipe.n < NB) {
            pipe.buf = NB - 1;                                         // all tiles are where they were
        } else {
            pipe.a.init(p.k, start, 0, len, kvh, p.hd, wave, lane);
            pipe.b.init(p.v, start, 0, len, kvh, p.hd, wave, lane);
            pipe.start(lds, &keys, wave);
        }
    }
    if (half == 0 && q < len && (KS == 1 || wave < 2)) {
        p.delta[(int64_t)head * p.tokens + tok] = D;
        p.lse2[(int64_t)head * p.tokens + tok] = nl;
    }

    // ds = p fix (dp - D), times the power of two but with a bias.  LATE: `fix` waits for the end, in LDS: a register more would leave head
    // size 64 two blocks a CU (100 x 512, 12 heads: 175 -> 219 us).
    AtDsScale<F16> sc;
    constexpr bool LATE = F16 && !BIAS && KS == 1;
    if constexpr (LATE) pair[wave][0][lane] = fix;
    else if constexpr (F16 && !BIAS) fix *= sc.START;
    float Df = LATE ? D * sc.START : D * fix;
    f32x16 dQ[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) dQ[dt] = at_zero16();
    walk([&](const char* Kt, int st, const f32x16& S, f32x16& dP, bool near, int rlo, int rhi) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) dP[i] = S[i] * __builtin_fmaf(dP[i], LATE ? sc.up : fix, -Df);   // ds
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
        f32x16 ds[1] = {F16 && BIAS ? dP * sc.up : dP};                // (the table's sums take it as it is)
        sc.fit(ds, dQ, [&](float f) __attribute__((always_inline)) {
            if constexpr (!BIAS) {
                if constexpr (!LATE) fix *= f;
                Df *= f;
            }
        });
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            u32x4 sf;
#pragma unroll
            for (int i = 0; i < 4; ++i) sf[i] = at_pack2<F16>(ds[0][8 * kk + 2 * i], ds[0][8 * kk + 2 * i + 1]);
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) dQ[dt] = at_mfma<F16>(at_cols<DP>(Kt, 2 * st + kk, dt, lane), sf, dQ[dt]);
        }
    });
    sc.down(dQ, LATE ? pair[wave][0][lane] : 1.0f);
    if constexpr (KS == 2) {
        at_sync();
        float* const x = reinterpret_cast<float*>(lds) + (wave & 1) * (DP / 2) * 64 + lane;
        if (wave >= 2) {
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[(16 * dt + i) * 64] = dQ[dt][i];
        }
        at_sync();
        if (wave < 2) {
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) dQ[dt][i] += x[(16 * dt + i) * 64];
        }
    }
    if (q < len && (KS == 1 || wave < 2)) at_store_row<DP, F16>(p.dq, start + q, head, p.hd, half, dQ, p.scale);
    if constexpr (BIAS) {
        // The diagonals of a wave by buckets: those of the outermost buckets across the lanes (one-sided, whatever is ahead counts as
        // distance 0), then lane b those of bucket b, four at a time.  One lane after another over the outermost ones took 3 us a block.
        for (int d = p.reach + lane; d <= R; d += 64) farS[0] += dvec[R - d];
        for (int d = (p.two_sided ? p.reach : 1) + lane; d <= R; d += 64) farS[1] += dvec[R + d];
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) {
            farS[0] += __shfl_xor(farS[0], s, 64);
            farS[1] += __shfl_xor(farS[1], s, 64);
        }
        float sum = 0.0f;
        if (lane < p.buckets) {
            const bool ahead = p.two_sided && lane >= p.side;          // r > 0
            const int i = ahead ? lane - p.side : lane;
            int lo = i <= p.exact ? i : p.border[i - p.exact - 1];     // distances lo .. hi
            const int hi = i < p.exact ? i : (i - p.exact < p.nborder ? p.border[i - p.exact] : p.reach) - 1;
            if (ahead && lo == 0) lo = 1;                              // distance 0 is not ahead
            const float* const at = dvec + R;
            const int sign = ahead ? 1 : -1;
            float part4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int d = lo; d <= hi; d += 4)
#pragma unroll
                for (int e = 0; e < 4; ++e) part4[e] += d + e <= hi ? at[sign * (d + e <= hi ? d + e : hi)] : 0.0f;
            sum = (part4[0] + part4[1]) + (part4[2] + part4[3]);
            if (lane == p.side - 1) sum += farS[0];
            if (lane == (p.two_sided ? p.buckets - 1 : 0)) sum += farS[1];
        }
        at_sync();
        skew0[wave * 64 + lane] = sum;
        at_sync();
        if (wave == 0) part[lane] = (skew0[lane] + skew0[64 + lane]) + (skew0[128 + lane] + skew0[192 + lane]);
    }
}

// dT[b][head] = the sum of the blocks' partial sums, in the tiles' order within each of WAVES strides.  Run by blocks of the dK / dV
// launch behind its tiles (attn_dq_kernel has ended by then): the grid's row of tiles number dtable_row, a head a block.
template <int WAVES>
__device__ __forceinline__ bool at_dtable(const mi_attn_args& p)
{
    const int row = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    if (row != p.dtable_row) return row > p.dtable_row;
    __shared__ float red[WAVES][64];
    const int b = threadIdx.x & 63, s = threadIdx.x >> 6;
    for (int head = at_unit(p); head < p.heads; head += 8 * p.units_per_xcd) {
        float sum = 0.0f;
        for (int t = s; t < p.dq_tiles; t += WAVES) sum += p.partial[((int64_t)head * p.dq_tiles + t) * MI_ATTN_MAX_BUCKETS + b];
        red[s][b] = sum;
        __syncthreads();
        if (s == 0 && b < p.buckets) {
            for (int i = 1; i < WAVES; ++i) sum += red[i][b];
            p.dtable[(int64_t)b * p.heads + head] = sum;
        }
        __syncthreads();
    }
    return true;
}

// dK, dV: one block per (key head, share of its query heads, 128 keys), a wave per 32 keys, over the tiles of 64 query rows of
// the share's heads: S = Q K^T and dP = dO V^T with the key on the lane, dV^T += dO^T P, dK^T += Q^T dS.  Where one block per key
// head and tile would leave CUs idle the group's heads are shared out over `splits` blocks, whose fp32 sums attn_join_kernel
// adds in the heads' order.  96 chunks up to 256 tokens (12 heads of 32, bias) take 33 us, a document of 4,000 (8 heads of 64) 68.
template <int DP, bool F16, bool BIAS, int KS>
__global__ __launch_bounds__(256, 2) void attn_dkv_kernel(const mi_attn_args p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int BM = 128 / KS, TB = AtTile<DP>::BYTES, NB = AT_BUFFERS(DP), PER = 2 * AtStage<DP, 4>::NI + 1;
    float* const rowv = reinterpret_cast<float*>(lds + NB * 2 * TB);   // [NB][lse in log2 units | D][64]
    float* const vec = rowv + NB * 128;
    if (BIAS && at_dtable<4>(p)) return;
    int kvh, t, start, len, tile;
    bool tail;
    if (!at_work(p, kvh, t) || !at_find<BM>(p, t, start, len, tile, tail)) return;
    const int unit = kvh, heads = p.share_heads;                       // (units are key heads x shares)
    kvh = at_div(unit, p.splits_inv);
    const int share = unit - kvh * p.splits;
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
    // with KS = 2 two waves share 32 keys and take every other 32 rows
    const int kw = tile * BM + (KS == 1 ? wave : wave & 1) * 32, key = kw + col, s0 = KS == 1 ? 0 : wave >> 1;
    const int64_t ktok = start + (key < len ? key : len - 1);
    u32x4 kf[DP / 16], vf[DP / 16];
    at_load_rows<DP>(kf, p.k, ktok, kvh, p.hd, half);
    at_load_rows<DP>(vf, p.v, ktok, kvh, p.hd, half);
    const bool on = key < len && (!p.key_mask || p.key_mask[ktok] != 0);

    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
    const int qfirst = p.causal ? tile * BM / AT_KT * AT_KT : 0;       // earlier queries attend no key of this block
    const int nq = (len - qfirst + AT_KT - 1) / AT_KT, n = nq * heads;
    AtStage<DP, 4> qs, ds;
    int ihead = head0 - 1, iq = nq;                                    // the tile requested last: its head, its number
    const float* rows = nullptr;
    auto issue = [&](int slot) __attribute__((always_inline)) {
        if (++iq >= nq) {
            iq = 0;
            ++ihead;
            qs.init(p.q, start, qfirst, len, ihead, p.hd, wave, lane);
            ds.init(p.dout, start, qfirst, len, ihead, p.hd, wave, lane);
            rows = (wave & 1 ? p.delta : p.lse2) + (int64_t)ihead * p.tokens + start;
        }
        qs.issue(lds0 + slot * 2 * TB, wave);
        ds.issue(lds0 + slot * 2 * TB + TB, wave);
        // 64 values of each row vector: even waves the log-sum-exp, odd ones D (waves 2 and 3 the same again)
        const int q = qfirst + iq * AT_KT + lane;
        at_dma4(rows + (q < len ? q : len - 1), lds0 + NB * 2 * TB + (unsigned)(slot * 128 + (wave & 1) * 64) * 4);
    };
    f32x16 dK[DP / 32], dV[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) { dK[dt] = at_zero16(); dV[dt] = at_zero16(); }
    AtDsScale<F16> sc;
    float dsf = AtPScale<F16>::down * sc.START;                        // ds = (p 2^12) (dp - D) dsf
    if (F16 && !on) dsf = 0.0f;                                        // a masked key: whatever its p, nothing to keep in range
#pragma unroll
    for (int t2 = 0; t2 < NB - 1; ++t2) if (t2 < n) issue(t2);
    const int R = p.reach + AT_PAD;
    int bias_head = -1;
    int head = head0, q0 = qfirst - AT_KT;
    for (int it = 0, buf = NB - 1; it < n; ++it) {
        q0 += AT_KT;
        if (q0 >= len) {
            q0 = qfirst;
            ++head;
        }
        if constexpr (BIAS) {
            if (head != bias_head) {
                if (bias_head >= 0) at_sync();                         // the last head's vector has been read
                at_fill_bias(p, head, p.scale_inv, 0.0f, vec);
                bias_head = head;
            }
        }
        at_arrive<PER>(n - 1 - it < NB - 2 ? n - 1 - it : NB - 2);
        if (it + NB - 1 < n) issue(buf);
        buf = buf + 1 == NB ? 0 : buf + 1;
        if (kw >= len || (p.causal && q0 + AT_KT - 1 < kw)) continue;
        const char* const Qt = lds + buf * 2 * TB;
        const char* const Dt = Qt + TB;
        const int rlo = kw - (q0 + AT_KT - 1), rhi = kw + 31 - q0;
        const bool near = BIAS && rhi > -p.reach && rlo < p.reach;
        const float add = AtPScale<F16>::log2 + (BIAS && !near ? vec[rhi <= -p.reach ? 0 : 2 * R] * p.scale_log2 : 0.0f);
        const int at = key - q0 - 4 * half + R;
#pragma unroll
        for (int st = s0; st < (KS == 1 ? 2 : s0 + 1); ++st) {
            if ((q0 + 32 * st >= len || (p.causal && q0 + 32 * st + 31 < kw))) continue;
            f32x16 S = at_first<F16>(near, vec + at - 32 * st, -1, at_rows<DP>(Qt, st, 0, col, half), kf[0]), X[1] = {at_zero16()};
            f32x16& dP = X[0];
#pragma unroll
            for (int s = 1; s < DP / 16; ++s) S = at_mfma<F16>(at_rows<DP>(Qt, st, s, col, half), kf[s], S);
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
                    S[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], p.scale_log2, add - nls[e]));
                    dP[i] = S[i] * ((dP[i] - Drs[e]) * dsf);
                }
            }
            if ((p.causal && q0 + 32 * st < kw + 31) || q0 + 32 * st + 32 > len) {   // rows that do not attend, or are none
                const int first = p.causal ? key - q0 - 32 * st - 4 * half : -AT_KT, end = len - q0 - 32 * st - 4 * half;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = 8 * (i >> 2) + (i & 3);
                    const bool ok = r >= first && r < end;
                    S[i] = ok ? S[i] : 0.0f;
                    dP[i] = ok ? dP[i] : 0.0f;
                }
            }
            sc.fit(X, dK, [&](float f) __attribute__((always_inline)) { dsf *= f; });
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
    sc.down(dK);
    if constexpr (KS == 2) {
        at_sync();
        float* const x = reinterpret_cast<float*>(lds) + (wave & 1) * DP * 64 + lane;
        if (wave >= 2) {
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    x[(32 * dt + i) * 64] = dK[dt][i];
                    x[(32 * dt + 16 + i) * 64] = dV[dt][i];
                }
        }
        at_sync();
        if (wave >= 2) return;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                dK[dt][i] += x[(32 * dt + i) * 64];
                dV[dt][i] += x[(32 * dt + 16 + i) * 64];
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

// The same at head sizes above 64, where dK, dV, K and V of 32 keys (192 registers and what the products need) leave a SIMD one wave,
// which nothing overlaps with: 1 x 8,191 causal, 8 heads of 128, 412 us where this form takes 362 us.  Eight waves, two to 32 keys: wave A
// makes S and P and sums dV, wave B makes dP and dS and sums dK.  P goes from A to B through LDS in fp32, each register to the same
// lane's; a SIMD has one wave of either kind, so one's exponentials run beside the other's products.  Two barriers a tile: it has
// landed, P is there.
template <bool F16, bool BIAS>
__global__ __launch_bounds__(512, 2) void attn_dkv_pair_kernel(const mi_attn_args p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int DP = 128, BM = 128, TB = AtTile<DP>::BYTES, NB = 2, PER = 2 * AtStage<DP, 8>::NI + 1;
    float* const rowv = reinterpret_cast<float*>(lds + NB * 2 * TB);   // [NB][lse in log2 units | D][64]
    float4* const pass = reinterpret_cast<float4*>(rowv + NB * 128);   // [4 pairs][8][64 lanes]
    float* const vec = reinterpret_cast<float*>(pass + 4 * 8 * 64);
    if (BIAS && at_dtable<8>(p)) return;
    int kvh, t, start, len, tile;
    bool tail;
    if (!at_work(p, kvh, t) || !at_find<BM>(p, t, start, len, tile, tail)) return;
    const int unit = kvh, heads = p.share_heads;                       // (units are key heads x shares)
    kvh = at_div(unit, p.splits_inv);
    const int share = unit - kvh * p.splits;
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
    const int col = lane & 31, half = lane >> 5, pair = wave & 3;
    const bool first = wave < 4;                                       // wave A
    const int kw = tile * BM + pair * 32, key = kw + col;
    const int64_t ktok = start + (key < len ? key : len - 1);
    u32x4 wf[DP / 16];                                                 // K or V
    at_load_rows<DP>(wf, first ? p.k : p.v, ktok, kvh, p.hd, half);
    const bool on = key < len && (!p.key_mask || p.key_mask[ktok] != 0);

    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
    const int qfirst = p.causal ? tile * BM / AT_KT * AT_KT : 0;       // earlier queries attend no key of this block
    const int nq = (len - qfirst + AT_KT - 1) / AT_KT, n = nq * heads;
    AtStage<DP, 8> qs, ds;
    int ihead = head0 - 1, iq = nq;                                    // the tile requested last: its head, its number
    const float* rows = nullptr;
    auto issue = [&](int slot) __attribute__((always_inline)) {
        if (++iq >= nq) {
            iq = 0;
            ++ihead;
            qs.init(p.q, start, qfirst, len, ihead, p.hd, wave, lane);
            ds.init(p.dout, start, qfirst, len, ihead, p.hd, wave, lane);
            rows = (wave & 1 ? p.delta : p.lse2) + (int64_t)ihead * p.tokens + start;
        }
        qs.issue(lds0 + slot * 2 * TB, wave);
        ds.issue(lds0 + slot * 2 * TB + TB, wave);
        // 64 values of each row vector: even waves the log-sum-exp, odd ones D (the others the same again)
        const int q = qfirst + iq * AT_KT + lane;
        at_dma4(rows + (q < len ? q : len - 1), lds0 + NB * 2 * TB + (unsigned)(slot * 128 + (wave & 1) * 64) * 4);
    };
    f32x16 acc[DP / 32];                                               // dV^T or dK^T
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = at_zero16();
    issue(0);
    const int R = p.reach + AT_PAD;
    int bias_head = -1, head = head0, q0 = qfirst - AT_KT, buf = NB - 1;
    // the next tile has landed; the one behind it is requested
    auto next = [&](int it) __attribute__((always_inline)) {
        q0 += AT_KT;
        if (q0 >= len) {
            q0 = qfirst;
            ++head;
        }
        if constexpr (BIAS) {
            if (head != bias_head) {
                if (bias_head >= 0) at_sync();                         // the last head's vector has been read
                at_fill_bias(p, head, AT_LOG2E, AtPScale<F16>::log2, vec);
                bias_head = head;
            }
        }
        at_arrive<PER>(0);
        if (it + 1 < n) issue(buf);
        buf ^= 1;
        return lds + buf * 2 * TB;
    };
    auto there = [&]() __attribute__((always_inline)) {                // what a wave wrote to LDS is there for the others
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto sum_half = [&](const char* rows_t, int st, const f32x16& X) __attribute__((always_inline)) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            u32x4 f;
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = at_pack2<F16>(X[8 * kk + 2 * i], X[8 * kk + 2 * i + 1]);
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = at_mfma<F16>(at_cols<DP>(rows_t, 2 * st + kk, dt, lane), f, acc[dt]);
        }
    };
    auto sum_up = [&](const char* rows_t, const f32x16 (&X)[2]) __attribute__((always_inline)) {
        sum_half(rows_t, 0, X[0]);
        sum_half(rows_t, 1, X[1]);
    };
    float4* const mine = pass + pair * 8 * 64 + lane;
    if (first) {
        for (int it = 0; it < n; ++it) {
            const char* const Qt = next(it);
            const bool idle = kw >= len || (p.causal && q0 + AT_KT - 1 < kw);
            f32x16 S[2];
            if (!idle) {
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int s = 0; s < DP / 16; ++s) S[st] = at_mfma<F16>(at_rows<DP>(Qt, st, s, col, half), wf[s], s == 0 ? at_zero16() : S[st]);
                const int rlo = kw - (q0 + AT_KT - 1), rhi = kw + 31 - q0;
                const bool near = BIAS && rhi > -p.reach && rlo < p.reach;
                const float add = BIAS ? (near ? 0.0f : vec[rhi <= -p.reach ? 0 : 2 * R]) : AtPScale<F16>::log2;
                const float* const bv = vec + (key - q0 - 4 * half + R);
                const bool edge = (p.causal && q0 < kw + 31) || q0 + AT_KT > len;      // rows that do not attend, or are none
                const int lo = p.causal ? key - q0 - 4 * half : -AT_KT, hi = len - q0 - 4 * half;
#pragma unroll
                for (int st = 0; st < 2; ++st) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float4 nl = *reinterpret_cast<const float4*>(rowv + buf * 128 + 32 * st + 8 * g + 4 * half);
                        const float nls[4] = {nl.x, nl.y, nl.z, nl.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int i = 4 * g + e, r = 32 * st + 8 * g + e;
                            const float b = BIAS && near ? bv[-r] : add;
                            S[st][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[st][i], p.scale_log2, b - nls[e]));
                            if (edge) S[st][i] = r >= lo && r < hi ? S[st][i] : 0.0f;
                        }
                        mine[(4 * st + g) * 64] = make_float4(S[st][4 * g], S[st][4 * g + 1], S[st][4 * g + 2], S[st][4 * g + 3]);
                    }
                }
            }
            there();
            if (!idle) sum_up(Qt + TB, S);
        }
    } else {
        AtDsScale<F16> sc;
        float dsf = AtPScale<F16>::down * sc.START;                    // as in attn_dkv_kernel
        if (F16 && !on) dsf = 0.0f;
        for (int it = 0; it < n; ++it) {
            const char* const Qt = next(it);
            const bool idle = kw >= len || (p.causal && q0 + AT_KT - 1 < kw);
            f32x16 dP[2];
            if (!idle) {
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int s = 0; s < DP / 16; ++s) dP[st] = at_mfma<F16>(at_rows<DP>(Qt + TB, st, s, col, half), wf[s], s == 0 ? at_zero16() : dP[st]);
                if constexpr (F16) {
#pragma unroll
                    for (int st = 0; st < 2; ++st)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const float4 Dr = *reinterpret_cast<const float4*>(rowv + buf * 128 + 64 + 32 * st + 8 * g + 4 * half);
                            const float Drs[4] = {Dr.x, Dr.y, Dr.z, Dr.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) dP[st][4 * g + e] = (dP[st][4 * g + e] - Drs[e]) * dsf;
                        }
                }
            }
            there();
            if constexpr (F16) {
                // the power of two is looked after 32 rows at a time, so that one half's products run beside the other's check
                if (!idle) {
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        f32x16 x[1];
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const float4 P = mine[(4 * st + g) * 64];
                            const float Ps[4] = {P.x, P.y, P.z, P.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[0][4 * g + e] = Ps[e] * dP[st][4 * g + e];
                        }
                        sc.fit(x, acc, [&](float f) __attribute__((always_inline)) {
                            dsf *= f;
                            if (st == 0) dP[1] = dP[1] * f;
                        });
                        sum_half(Qt, st, x[0]);
                    }
                }
            } else if (!idle) {
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float4 Dr = *reinterpret_cast<const float4*>(rowv + buf * 128 + 64 + 32 * st + 8 * g + 4 * half), P = mine[(4 * st + g) * 64];
                        const float Drs[4] = {Dr.x, Dr.y, Dr.z, Dr.w}, Ps[4] = {P.x, P.y, P.z, P.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) dP[st][4 * g + e] = Ps[e] * ((dP[st][4 * g + e] - Drs[e]) * AtPScale<F16>::down);
                    }
                sum_up(Qt, dP);
            }
        }
        sc.down(acc);
    }
    if (key < len) {
        if (!on) {                                                     // a masked key (the products above ran on its column alone)
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = at_zero16();
        }
        const float f = first ? AtPScale<F16>::down : p.scale;
        if (p.splits == 1) at_store_row<DP, F16>(first ? p.dv : p.dk, start + key, kvh, p.hd, half, acc, f);
        else at_store_part<DP>(p.parts_kv, ((int64_t)(2 * share + (first ? 1 : 0)) * p.tokens + start + key) * at_div(p.heads, p.group_inv) + kvh, p.hd, half, acc, f);
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

// ---------------------------------------------------------------- launch
static int gcd_int(int a, int b) { while (b) { const int t = a % b; a = b; b = t; } return a; }

// The grid over `heads` heads and tiles of BM rows (see at_work), and `more` rows of blocks behind them.
static dim3 at_schedule(mi_attn_args* a, int heads, int BM, int more = 0)
{
    const int64_t tiles = a->offsets ? a->tokens / BM + a->nseq + (a->zero_tail ? 1 : 0)
                                     : (int64_t)a->nseq * ((a->uniform_len + BM - 1) / BM);
    const int g = gcd_int(heads, 8);
    a->tiles = (int)tiles;
    a->parts_log2 = g == 8 ? 0 : g == 4 ? 1 : g == 2 ? 2 : 3;
    a->units_per_xcd = heads / g;
    a->dtable_row = (int)((tiles + 8 / g - 1) >> a->parts_log2);
    const unsigned rows = (unsigned)(a->dtable_row + more), z = (rows + 65534) / 65535;
    return dim3((unsigned)(8 * a->units_per_xcd), z ? (rows + z - 1) / z : 0, z);
}
static uint32_t inv32(int d) { return d <= 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + d - 1) / d); }

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
    MI_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, 156 * 1024));   // (160 KB less the mask words)
    if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
    return MI_OK;
}

// Two waves to a row where 128-row blocks are fewer than four to a CU.  Forward: 432 blocks (2 causal documents up to 4,099, 8 heads of
// 64, bias) 76 -> 56 us, 520 (8,191, 8 heads of 128) 178 -> 160 us; 1,500 blocks (prompts up to 2,039, 32 heads of 128) 75 ->
// 87 us, 2,048 (16,384, 16 heads of 128) 1,066 -> 1,243 us, 8,900 (chunks up to 256, 12 heads of 32) 67 -> 83 us.  Backward: 256
// blocks (a document of 4,000, 8 heads of 64, bias) dQ 98 -> 73 us, dK / dV 99 -> 68 us; 512 (8,191, 8 heads of 128) dQ 255 -> 228 us.
// (Blocks are counted, not their work: a batch of short sequences is split like one document, and with up to 32 keys the second wave of a
// row has nothing to do.)
static bool at_few(const mi_attn_args& a, int heads) { return (int64_t)heads * (a.tokens / 128 + a.nseq) < 1024; }

template <int DP, bool F16, bool BIAS, int KS>
static int launch_fwd(hipStream_t st, mi_attn_args& a)
{
    const dim3 grid = at_schedule(&a, a.heads, 128 / KS);
    if (grid.y == 0) return MI_OK;
    size_t smem = AT_BUFFERS(DP) * 2 * AtTile<DP>::BYTES + (BIAS ? (2 * (size_t)(a.reach + AT_PAD) + 1) * 4 : 0);
    if (KS == 2 && smem < (size_t)2 * (DP / 2 + 3) * 64 * 4) smem = (size_t)2 * (DP / 2 + 3) * 64 * 4;
    MI_TRY((at_lds<&attn_fwd_kernel<DP, F16, BIAS, KS>>(smem)));
    attn_fwd_kernel<DP, F16, BIAS, KS><<<grid, 256, smem, st>>>(a);
    MI_HIP(hipGetLastError());
    return MI_OK;
}

template <int DP, bool F16>
static int launch_fwd(hipStream_t st, mi_attn_args& a)
{
    const bool split = at_few(a, a.heads);
    if (a.table) return split ? launch_fwd<DP, F16, true, 2>(st, a) : launch_fwd<DP, F16, true, 1>(st, a);
    return split ? launch_fwd<DP, F16, false, 2>(st, a) : launch_fwd<DP, F16, false, 1>(st, a);
}

int mi_launch_attention(hipStream_t st, mi_attn_args a, int dtype)
{
    const bool f16 = dtype == MI_DTYPE_F16;
    if (a.hd <= 32) return f16 ? launch_fwd<32, true>(st, a) : launch_fwd<32, false>(st, a);
    if (a.hd <= 64) return f16 ? launch_fwd<64, true>(st, a) : launch_fwd<64, false>(st, a);
    return f16 ? launch_fwd<128, true>(st, a) : launch_fwd<128, false>(st, a);
}

// Shares of a group's query heads in the dK / dV kernel: the fewest that give AT_DKV_BLOCKS blocks (three per CU), all heads at most.  Fewer
// blocks leave CUs idle, more write and read again 2 x tokens x key heads x head_dim fp32 words each (whole backward pass, us, the shares
// in brackets; bf16; also measured at 32 heads on 4, at head size 32 and with a bias, with the same outcome):
//                                              at least 256   512        768        1,024      2,048
//   8,191 causal, 16 heads on 4 of 128         1,591 (1)      1,066 (2)  1,079 (4)  1,080 (4)  1,079 (4)
//   9 prompts up to 2,048, the same heads        252 (2)        208 (4)    208 (4)    208 (4)    208 (4)
//   60 x 300, the same heads                     309 (1)        310 (1)    310 (1)    395 (2)    455 (4)
//   60 x 300, 16 heads on 2 of 64                157 (1)        153 (2)    153 (2)    164 (4)    189 (8)
//   300 x 40, 16 heads on 2 of 32                 53 (1)         54 (1)     53 (1)     63 (2)     65 (4)
//   8,191 causal, 32 heads on 4 of 64          1,306 (1)      1,055 (2)  1,041 (4)  1,038 (4)  1,010 (8)
#define AT_DKV_BLOCKS 768
static int at_dkv_splits(const mi_attn_args& a)
{
    const int64_t blocks = (int64_t)(a.heads / a.group) * (a.tokens / 128 + a.nseq);
    if (a.tokens == 0) return 1;                                       // nothing to share out, nor to join
    for (int s = 1; s < a.group; ++s)
        if (a.group % s == 0 && blocks * s >= AT_DKV_BLOCKS) return s;
    return a.group;
}

size_t mi_attn_backward_bytes(const mi_attn_args& a)
{
    const size_t delta = mi_round_up((int64_t)a.heads * a.tokens * 8, 256);
    const int splits = at_dkv_splits(a);
    const size_t join = splits > 1 ? (size_t)mi_round_up((int64_t)splits * 2 * a.tokens * (a.heads / a.group) * a.hd * 4, 256) : 0;
    const int64_t tiles = a.offsets ? a.tokens / 64 + a.nseq + 1 : (int64_t)a.nseq * ((a.uniform_len + 63) / 64);   // at most
    return delta + join + (a.table ? (size_t)(a.heads * tiles) * MI_ATTN_MAX_BUCKETS * 4 : 0);
}

// With a bias the LDS of a dQ block grows by 40 bytes for each distance of `reach` (the bias and the waves' sums over r): two blocks a CU up to
// reach 466 at head size 32, 262 at 64 (210 with two waves to a row), one beyond, and at 128 (48 buckets, 100 x 512 rows of 12 heads of 64: reach
// 244 385 us, reach 288 675 us; 12 of 32: reach 374 331 us, reach 707 697 us).
template <int DP, bool F16, bool BIAS, int KS>
static int launch_dq(hipStream_t st, mi_attn_args& a)
{
    const dim3 grid = at_schedule(&a, a.heads, 128 / KS);
    if (grid.y == 0) return MI_OK;
    const size_t smem = AT_DQ_BUFFERS(DP, BIAS) * 2 * AtTile<DP>::BYTES + (BIAS ? (4 * 32 * 64 + 5 * (2 * (size_t)(a.reach + AT_PAD) + 1)) * 4 : 0);
    MI_TRY((at_lds<&attn_dq_kernel<DP, F16, BIAS, KS>>(smem)));
    attn_dq_kernel<DP, F16, BIAS, KS><<<grid, 256, smem, st>>>(a);
    MI_HIP(hipGetLastError());
    return MI_OK;
}

template <int DP, bool F16>
static int launch_bwd(hipStream_t st, mi_attn_args& a)
{
    const bool split = at_few(a, a.heads);
    if (a.table) MI_TRY((split ? launch_dq<DP, F16, true, 2>(st, a) : launch_dq<DP, F16, true, 1>(st, a)));
    else MI_TRY((split ? launch_dq<DP, F16, false, 2>(st, a) : launch_dq<DP, F16, false, 1>(st, a)));
    a.dq_tiles = a.tiles;
    const int units = a.heads / a.group * a.splits;
    const bool split_kv = DP < 128 && at_few(a, units);
    const dim3 grid = at_schedule(&a, units, split_kv ? 64 : 128, a.table ? 1 : 0);   // (and at_dtable's blocks)
    if (grid.y == 0) return MI_OK;
    const size_t bias = a.table ? (size_t)(2 * (a.reach + AT_PAD) + 1) * 4 : 0;
    if constexpr (DP == 128) {
        const size_t smem = 2 * (2 * AtTile<DP>::BYTES + 512) + 4 * 8 * 64 * 16 + bias;
        if (a.table) {
            MI_TRY((at_lds<&attn_dkv_pair_kernel<F16, true>>(smem)));
            attn_dkv_pair_kernel<F16, true><<<grid, 512, smem, st>>>(a);
        } else {
            MI_TRY((at_lds<&attn_dkv_pair_kernel<F16, false>>(smem)));
            attn_dkv_pair_kernel<F16, false><<<grid, 512, smem, st>>>(a);
        }
    } else {
        const size_t smem = AT_BUFFERS(DP) * (2 * AtTile<DP>::BYTES + 512) + bias;   // at most 59,652 bytes
        if (a.table) {
            if (split_kv) attn_dkv_kernel<DP, F16, true, 2><<<grid, 256, smem, st>>>(a);
            else attn_dkv_kernel<DP, F16, true, 1><<<grid, 256, smem, st>>>(a);
        } else {
            if (split_kv) attn_dkv_kernel<DP, F16, false, 2><<<grid, 256, smem, st>>>(a);
            else attn_dkv_kernel<DP, F16, false, 1><<<grid, 256, smem, st>>>(a);
        }
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
    a.lse2 = a.delta + (int64_t)a.heads * a.tokens;
    a.splits = at_dkv_splits(a);
    a.splits_inv = inv32(a.splits);
    a.share_heads = a.group / a.splits;
    a.parts_kv = (float*)((char*)workspace + mi_round_up((int64_t)a.heads * a.tokens * 8, 256));
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
    for (int32_t& x : a->border) x = INT32_MAX;
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

// What a call's sizes have to be, for its workspace as for the call.
static int check_heads(const char* who, const mi_attention_config* c)
{
    MI_REQUIRE(c->heads > 0 && c->heads <= 65535 && c->kv_heads > 0 && c->heads % c->kv_heads == 0, "%s: heads %d must be a positive multiple of kv_heads %d", who, c->heads, c->kv_heads);
    MI_REQUIRE(c->head_dim > 0 && c->head_dim % 8 == 0 && c->head_dim <= 128, "%s: head_dim %d must be a multiple of 8 up to 128", who, c->head_dim);
    return MI_OK;
}
static int check_rows(const char* who, int64_t tokens, int64_t nseq, bool packed)
{
    MI_REQUIRE(tokens >= 0 && tokens < ((int64_t)1 << 31) - 4096, "%s: %lld tokens out of range", who, (long long)tokens);
    MI_REQUIRE(nseq >= 0 && nseq < ((int64_t)1 << 24), "%s: %lld sequences out of range", who, (long long)nseq);
    MI_REQUIRE(packed || (nseq == 0 ? tokens == 0 : tokens % nseq == 0), "%s: %lld tokens are not %lld sequences of one length", who, (long long)tokens, (long long)nseq);
    return MI_OK;
}
static int check_launch(const char* who, const mi_attention_config* c, int64_t tokens, int64_t nseq)
{
    // one launch: fewer than 2^21 tiles of a head (of at least 64 rows each), 2^31 blocks
    MI_REQUIRE(tokens / 64 + nseq + 9 < ((int64_t)1 << 21) && (tokens / 64 + nseq + 9) * (int64_t)c->heads < ((int64_t)1 << 31) - 1, "%s: %lld tokens in %lld sequences x %d heads are too many for one call", who, (long long)tokens, (long long)nseq, c->heads);
    return MI_OK;
}

// Everything both directions check; fills the fields they share.
static int fill_args(const char* who, mi_ctx* ctx, const mi_attention_config* c, int64_t tokens, int64_t nseq, const int32_t* offsets,
                     const int32_t* key_mask, const mi_attention_rows* q, const mi_attention_rows* k, const mi_attention_rows* v,
                     const float* table, mi_attn_args* a)
{
    MI_REQUIRE(ctx && c, "%s: NULL argument", who);
    MI_REQUIRE(c->dtype == MI_DTYPE_BF16 || c->dtype == MI_DTYPE_F16, "%s: dtype %d is not MI_DTYPE_BF16 or MI_DTYPE_F16", who, c->dtype);
    MI_TRY(check_heads(who, c));
    MI_REQUIRE(c->scale >= 1e-20f && c->scale <= 1e20f, "%s: scale must be between 1e-20 and 1e20", who);
    MI_TRY(check_rows(who, tokens, nseq, offsets != nullptr));
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
    a->group_inv = inv32(a->group);
    a->hd = c->head_dim;
    a->causal = c->causal != 0;
    a->zero_tail = c->zero_tail != 0;
    a->scale = c->scale;
    a->scale_log2 = c->scale * AT_LOG2E;
    a->scale_inv = 1.0f / c->scale;
    return check_launch(who, c, tokens, nseq);
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
    const char* who = "mi_attention_backward_workspace";
    MI_TRY(check_heads(who, cfg));
    MI_TRY(check_rows(who, tokens, nseq, packed != 0));
    mi_attn_args a;
    static const int32_t some = 0;
    static const float one = 0.0f;
    if (cfg->num_buckets != 0) {
        MI_TRY(mi_attn_buckets(who, &a, cfg->num_buckets, cfg->max_distance, cfg->bidirectional));
        a.table = &one;
    }
    MI_TRY(check_launch(who, cfg, tokens, nseq));
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
