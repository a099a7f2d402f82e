// block_gemm.hip -- the product of the FC layers as an operator: y = act(x W^T + bias) with W chosen by the row's group, operands in bf16 or in
// e4m3 with a scale for every 128 values of a row of x and every 128 x 128 block of W.
//
//   y[j, c] = act( sum_t sa[t, src(j)] sb[g, c / 128, t] sum_{u < 128} a[src(j), 128 t + u] w[g, c, 128 t + u]  +  bias[g, c] )
//
// The inner sums run on the matrix pipe in fp32; fp32 scales multiply a block's sum on the vector pipe (one fma a value), e8m0 scales are operands
// of the 8-bit matrix instruction itself.  One matrix instruction of 16 x 16 x 128 covers a block along K; the bf16 form takes two of 16 x 16 x 32 for the
// same 128 bytes of a row, so one layout in LDS serves both: rows of 128 bytes, eight 16-byte chunks, chunk c of row r in slot c ^ ((r >> 1) & 7)
// -- of the sixteen rows that one access serves, two share a line of 256 bytes and the pairs lie in eight different slots.
//
// The weights are the instruction's FIRST operand: a lane then holds four neighbouring columns of one row of y (one activation scale a lane, vector
// stores).  Lane l: row l & 15 of either operand, chunks l >> 4 and (l >> 4) + 4.
#include "block_ops.h"
#include <atomic>
#include <cmath>
#include <type_traits>

namespace dce {

namespace {

__device__ __forceinline__ int clamp_to(int v, int hi) { return v < 0 ? 0 : v > hi ? hi : v; }

struct Place { int g, first, end, tn; };      // a tile: its group, its first row and the group's end, its column tile

// The tile of this workgroup.  Row tiles are counted group by group (offsets are held inside [0, m] whatever they say) and only here: the host knows no
// more than a bound.  Workgroups go round the eight XCDs, so workgroup 8 i + x takes the i-th tile of the x-th eighth of those that there are: neighbours
// share an L2.  They go in bands of eight column tiles, columns first: the 32 CUs of an XCD work on 4 x 8 tiles, and of the 64 panels that these take a
// step 12 come from beyond the L2 (without bands, 8192^3: 33; 434 us, with them 410).  64 groups a step, tiles counted by a scan over the lanes; every wave
// does it for itself.
__device__ __forceinline__ bool find_tile(const ProductArgs& p, int bm, Place& at)
{
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = p.m, tiles = 0, sum = 0;
    auto scan = [&](int base) {
        lo = hi = 0;
        if (base + lane < p.groups) { lo = clamp_to(p.offsets[base + lane], p.m); hi = clamp_to(p.offsets[base + lane + 1], p.m); }
        sum = tiles = hi > lo ? (hi - lo + bm - 1) / bm : 0;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(sum, d); if (lane >= d) sum += o; }
        return __builtin_amdgcn_readlane(sum, 63);
    };
    int total = 0;
    if (!p.offsets) total = (p.m + bm - 1) / bm;
    else for (int base = 0; base < p.groups; base += 64) total += scan(base);
    if ((unsigned)total > (unsigned)p.tiles_m) total = p.tiles_m;             // (offsets that fall: tiles of the same rows, of which the launch has no more than these)
    const unsigned all = (unsigned)total * (unsigned)p.tiles_n, per = (all + 7) >> 3, slot = blockIdx.x >> 3, id = (blockIdx.x & 7) * per + slot;
    if (slot >= per || id >= all) return false;
    const unsigned band = id / ((unsigned)total * 8), wide = p.tiles_n - band * 8 < 8 ? p.tiles_n - band * 8 : 8, in = id - band * total * 8;
    const int t = (int)(in / wide);
    at.tn = (int)(band * 8 + in % wide);
    if (!p.offsets) { at.g = 0; at.first = t * bm; at.end = p.m; return true; }
    int before = 0;
    for (int base = 0; base < p.groups; base += 64) {
        const int here = p.groups <= 64 ? total : scan(base);
        if (t < before + here) {
            const int w = __builtin_ctzll(__ballot(before + sum > t));
            at.g = base + w;
            at.first = __builtin_amdgcn_readlane(lo, w) + (t - (before + __builtin_amdgcn_readlane(sum, w) - __builtin_amdgcn_readlane(tiles, w))) * bm;
            at.end = __builtin_amdgcn_readlane(hi, w);
            return at.first >= __builtin_amdgcn_readlane(lo, w) && at.first < at.end;       // (... and their count may pass 32 bits)
        }
        before += here;
    }
    return false;
}

// the row of a that row j of y is made from; -1: a row of zeros
__device__ __forceinline__ long long source_row(const ProductArgs& p, int j, int end)
{
    if (j >= end) return -1;
    const long long s = p.index ? (long long)p.index[j] : (long long)j;
    return s >= 0 && s < p.a_rows ? s : -1;
}

// chunk c of row r of a tile in LDS
__device__ __forceinline__ int slot_of(int r, int c) { return r * KROW + ((c ^ ((r >> 1) & 7)) * 16); }
__device__ __forceinline__ i32x4 chunk(const char* lds, int r, int c) { return *reinterpret_cast<const i32x4*>(lds + slot_of(r, c)); }

// 16 e4m3 values -> fp16, without error
__device__ __forceinline__ void to_f16(i32x4 v, f16x8& lo, f16x8& hi)
{
    f16x2 h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[i], 1.f, false);
        h[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[i], 1.f, true);
    }
    lo = __builtin_shufflevector(__builtin_shufflevector(h[0], h[1], 0, 1, 2, 3), __builtin_shufflevector(h[2], h[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
    hi = __builtin_shufflevector(__builtin_shufflevector(h[4], h[5], 0, 1, 2, 3), __builtin_shufflevector(h[6], h[7], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}
// ... times the power of two of an e8m0 byte -> bf16, without error (bf16 has fp32's range)
__device__ __forceinline__ void to_bf16x16(i32x4 v, unsigned byte, bf16x8& lo, bf16x8& hi)
{
    const float s = __uint_as_float(byte << 23);                              // (the instruction takes the exponent alone)
    bf16x2 h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], s, false);
        h[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], s, true);
    }
    lo = __builtin_shufflevector(__builtin_shufflevector(h[0], h[1], 0, 1, 2, 3), __builtin_shufflevector(h[2], h[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
    hi = __builtin_shufflevector(__builtin_shufflevector(h[4], h[5], 0, 1, 2, 3), __builtin_shufflevector(h[6], h[7], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// One row's 128 bytes of a step as a lane holds its quarter of them for the matrix instruction.  EXACT: e4m3 in 16 bits (see mfma_row); `scale`: the
// row's, or the weights', e8m0 byte
template <int IN, bool EXACT> struct Frag {
    i32x4 c0, c1;
    __device__ __forceinline__ void set(i32x4 a, i32x4 b, unsigned) { c0 = a; c1 = b; }
};
template <> struct Frag<IN_F8_F32, true> {
    f16x8 h[4];
    __device__ __forceinline__ void set(i32x4 a, i32x4 b, unsigned) { to_f16(a, h[0], h[1]); to_f16(b, h[2], h[3]); }
};
template <> struct Frag<IN_F8_E8, true> {
    bf16x8 h[4];
    __device__ __forceinline__ void set(i32x4 a, i32x4 b, unsigned scale) { to_bf16x16(a, scale, h[0], h[1]); to_bf16x16(b, scale, h[2], h[3]); }
};

// The scales of a step for a lane's row of x and a block of columns.  fp32: their product.  e8m0: the two bytes for the 8-bit matrix instruction, whose
// byte 255 is NaN; where the fragments took them (EXACT) `bad` remembers that there was one.
template <int IN, bool EXACT> struct Scale {
    float s; int ew, ex;
    __device__ __forceinline__ void set(unsigned w, unsigned x, unsigned& bad)
    {
        if (IN == IN_F8_F32) s = __uint_as_float(w) * __uint_as_float(x);
        else if (EXACT) bad |= w == 255 || x == 255;
        else { ew = (int)w; ex = (int)x; }
    }
};
template <int IN, bool EXACT, int NT>
__device__ __forceinline__ void spoil(f32x4 (&acc)[NT], unsigned bad)
{
    if constexpr (IN == IN_F8_E8 && EXACT)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] = bad ? __builtin_nanf("") : acc[j][i];
}

// acc += the product of a block of 16 x 16 over one step of K.
//
// The 8-bit matrix instruction lines the eight products of a group up with the largest of them and keeps 13 bits below its leading one (measured: of
// 65536 + 8 everything, of 65536 + 4 nothing is left of the second, -4 neither; between groups sums are fp32): on random operands 1.5e-5 of the result, with
// products of one sign 7e-5, at worst 7 * 2^-13 of the sum of magnitudes.  The rounding to bf16 is 1.7e-3 of a result and that to e4m3 more, so results in
// those types take it (and e4m3 scales look again next to their borders).  fp32 results would be a hundred times worse
// than their type: their operands go through the 16-bit instructions, at half the rate, whose sums of 32 products are good to 1e-8 -- with e8m0 scales
// as bf16 with the scale in it, with fp32 scales as fp16 (every e4m3 number is one).
//
// One row of blocks at a time: instructions that add to the same sums are as far apart as the row is long (a dependent one waits for its predecessor).
// Where the matrix instruction can apply the scales (or there are none) it adds to `acc`; otherwise the block's sums go to `part` and fold_row brings
// them home -- behind the next row's matrix instructions, which hide it.
template <int IN, bool EXACT> constexpr bool FOLDS = IN == IN_F8_F32;

template <int IN, bool EXACT, int NT>
__device__ __forceinline__ void mfma_row(f32x4 (&acc)[NT], f32x4 (&part)[NT], const Frag<IN, EXACT> (&w)[NT], const Frag<IN, EXACT>& x, const Scale<IN, EXACT>& sc)
{
    if constexpr (IN == IN_BF16) {
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w[j].c0), __builtin_bit_cast(bf16x8, x.c0), acc[j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w[j].c1), __builtin_bit_cast(bf16x8, x.c1), acc[j], 0, 0, 0);
    } else if constexpr (EXACT) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if constexpr (IN == IN_F8_E8) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j].h[k], x.h[k], acc[j], 0, 0, 0);
                else part[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[j].h[k], x.h[k], k ? part[j] : f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            }
    } else {
        const i32x8 xv = __builtin_shufflevector(x.c0, x.c1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const i32x8 wv = __builtin_shufflevector(w[j].c0, w[j].c1, 0, 1, 2, 3, 4, 5, 6, 7);
            if constexpr (IN == IN_F8_E8) acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, acc[j], 0, 0, 0, sc.ew, 0, sc.ex);
            else part[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 127, 0, 127);
        }
    }
}
template <int IN, bool EXACT, int NT>
__device__ __forceinline__ void fold_row(f32x4 (&acc)[NT], const f32x4 (&part)[NT], const Scale<IN, EXACT>& sc)
{
    if constexpr (FOLDS<IN, EXACT>)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] = fmaf(part[j][i], sc.s, acc[j][i]);
}
template <int IN, bool EXACT, int NT>
__device__ __forceinline__ void mac_row(f32x4 (&acc)[NT], const Frag<IN, EXACT> (&w)[NT], const Frag<IN, EXACT>& x, const Scale<IN, EXACT>& sc)
{
    f32x4 part[NT];
    mfma_row<IN, EXACT, NT>(acc, part, w, x, sc);
    fold_row<IN, EXACT, NT>(acc, part, sc);
}

__device__ __forceinline__ unsigned short to_bf16(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }

// four neighbouring columns c .. of row j
template <int OUT>
__device__ __forceinline__ void store4(const ProductArgs& p, int j, int c, f32x4 v, bool wide)
{
    constexpr int SZ = OUT == OUT_F32 ? 4 : OUT == OUT_BF16 ? 2 : 1;
    char* at = p.y + (long long)j * p.y_row + (long long)c * SZ;
    if constexpr (OUT == OUT_F32) {
        if (wide && c + 4 <= p.n) { *reinterpret_cast<f32x4*>(at) = v; return; }
#pragma unroll
        for (int i = 0; i < 4; ++i) if (c + i < p.n) reinterpret_cast<float*>(at)[i] = v[i];
    } else if constexpr (OUT == OUT_BF16) {
        unsigned short h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = to_bf16(v[i]);
        if (wide && c + 4 <= p.n) { *reinterpret_cast<uint2*>(at) = make_uint2(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16); return; }
#pragma unroll
        for (int i = 0; i < 4; ++i) if (c + i < p.n) reinterpret_cast<unsigned short*>(at)[i] = h[i];
    } else {
        const int w = to_e4m3x4(v[0], v[1], v[2], v[3]);
        if (wide && c + 4 <= p.n) { *reinterpret_cast<int*>(at) = w; return; }
#pragma unroll
        for (int i = 0; i < 4; ++i) if (c + i < p.n) at[i] = (char)(w >> (8 * i));
    }
}
__device__ __forceinline__ bool wide_stores(const ProductArgs& p, int bytes)
{
    return ((p.y_row | (long long)reinterpret_cast<uintptr_t>(p.y)) & (bytes - 1)) == 0;
}

}  // namespace

// ---- the kernel for operands whose rows start at multiples of 16 bytes: BM x BN a workgroup, MT x NT blocks of 16 x 16 a wave, the steps of K dealt
//      out in turn to KG groups of four waves, each with panels of its own, that add up their sums at the end (group 0's first).  A step's panels and
//      scales come by LDS-DMA into a ring of NBUF buffers, fragments from there into registers a step ahead of their instructions; one barrier for KG
//      steps.  The requests are what bounds it (a CU takes one of 1 KB in 16 cycles), then the barrier: two groups share that.
// 64 lanes x 16 bytes from `from` + the lanes' offsets to LDS at `lds` (+ lane * 16)
__device__ __forceinline__ void dma16s(const char* from, unsigned at, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0" :: "s"(from), "v"(at), "s"(lds) : "memory");
}
__device__ __forceinline__ void dma4s(const char* from, unsigned at, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, %0" :: "s"(from), "v"(at), "s"(lds) : "memory");
}
__device__ __forceinline__ void dma1s(const char* from, unsigned at, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, %0" :: "s"(from), "v"(at), "s"(lds) : "memory");
}
__device__ __forceinline__ unsigned lds_addr(const void* p) { return (unsigned)(unsigned long long)(const __attribute__((address_space(3))) char*)p; }

template <int N> __device__ __forceinline__ void wait_all_but() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }

template <int WM_, int WN_, int MT_, int NT_, int NBUF_, int KG_> struct Ring {
    static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_, NBUF = NBUF_, KG = KG_;   // waves along the rows / the columns; blocks of 16 a wave
    static constexpr int BM = WM * MT * 16, BN = WN * NT * 16, WAVES = WM * WN, THREADS = 64 * WAVES * KG;
    static constexpr int PANELS = (BM + BN) * KROW, PIECES = PANELS / 1024 / WAVES;   // a piece: eight rows, one instruction
    static constexpr int SA = (BM + 63) / 64, SLOT = (SA + 1) * 256, BUF = PANELS + SLOT;  // waves that bring the rows' scales; a word a row, then the columns'
    static constexpr int BIAS = KG * NBUF * BUF, LDS = BIAS + BN * 4;
    static_assert(PANELS % (1024 * WAVES) == 0 && BM % 8 == 0 && BN == BLK && LDS <= 160 * 1024 && SA < WAVES && WAVES == 4, "tile");
};

// The tile's bias -> LDS, asked for first and there with the first panels (the epilogue would wait for it once more)
template <class T>
__device__ __forceinline__ void bring_bias(const ProductArgs& p, const char* smem, int g, int n0, int wave, int lane)
{
    if (!p.bias || wave * 64 >= T::BN) return;
    const int c = n0 + wave * 64 + lane;
    dma4s(reinterpret_cast<const char*>(p.bias + g * p.bias_group), (unsigned)(c < p.n ? c : p.n - 1) * 4, lds_addr(smem) + T::BIAS + wave * 256);
}

// ---- the scale of e4m3 results.  Its exponent hangs on which side of 448 * 2^e a block's largest value lies, and the 8-bit matrix instruction's sums may be
// on the other side: each product loses less than 2^-13 of the largest of its group of eight, towards zero, so that a sum of products of one sign comes
// out up to 7 * 2^-13 of itself too small (and good to fp32 otherwise).  So where a largest value lies within 2^-10 below such a border or 2^-12 above
// it (one block in 570), every value there is summed once more in fp32, and the block lies above the border if one of them does.  The values that are
// stored stay the first sums, which both scales hold.  Operands that cancel can be off by more (7 * 2^-13 of the sum of magnitudes), and the scale with them.
//
// One or two values of a row (and of a wave's columns): each by itself, K dealt out to the waves' lanes.  More: 16 x 16 at a time through the 16-bit matrix
// instructions.  That reads 32 rows of K where a value needs two: with K 4736 it takes 7 us where one value takes 1.3.  What it costs (results in e4m3, with
// no value ever in question, and as it is; bf16): 1024 rows of 2048 x 4736 20.3, 22.6 and 19.0 us; 4096 39.3, 42.6 and 38.0; 32768 263, 276 and 257.  Where every
// value of 4096 rows lies on a border, 730.
constexpr int FEW = 2, AT_ONCE = 64, MANY = 1 << 30;
template <class T> struct Doubts {                                            // in LDS
    unsigned blocks[8];                                                       // a bit for every 16 x 16 values of the tile with rows of many in question
    int found;                                                                // single ones; MANY: there are such blocks
    int list[FEW * T::BM * T::WN];                                            // row << 8 | column of the tile
    int above[T::BM * (T::BN / BLK)];                                         // by column block * BM + row: one of them lies above the border
    union {
        float rows[T::WAVES][16][T::NT * 16 + 4];                             // a wave's values of sixteen rows, to look for them
        f32x4 parts[T::WAVES][64];                                            // the waves' sums of 16 x 16 values, or of AT_ONCE single ones
    };
};
constexpr int UNDER = 14336, OVER = 3584;                                     // 2^-10 and 2^-12 of 0xe00000, the border with its leading bit (448 = 1.75 * 2^8)
__device__ __forceinline__ bool in_doubt(float most)
{
    const int m = (int)(__float_as_uint(most) & 0x7fffffu) - 0x600000;
    return m > -UNDER && m < OVER;
}
__device__ __forceinline__ int border_of(float most) { return (int)((__float_as_uint(most) & 0x7f800000u) | 0x600000u); }      // (in bits)

// one value: what one wave of WAVES sums of it
template <int IN, int WAVES>
__device__ __forceinline__ float sum_one(const ProductArgs& p, int g, long long src, int c, int wave, int lane)
{
    const char* const a = p.a + src * p.a_row;
    const char* const b = p.b + g * p.b_group + (long long)c * p.b_row;
    const long long sb0 = g * p.sb_group + (long long)(c / BLK) * p.sb_row;
    float sum = 0.f;
#pragma unroll 1
    for (int at = (wave * 64 + lane) * 16; at < p.kbytes; at += WAVES * 1024) {
        const bool whole = at + 16 <= p.kbytes;
        const i32x4 x = whole ? load16(a + at) : load16_tail(a, at, p.kbytes), w = whole ? load16(b + at) : load16_tail(b, at, p.kbytes);
        const int t = at / BLK;
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            part = fmaf(__builtin_amdgcn_cvt_f32_fp8(x[i], 0), __builtin_amdgcn_cvt_f32_fp8(w[i], 0), part);
            part = fmaf(__builtin_amdgcn_cvt_f32_fp8(x[i], 1), __builtin_amdgcn_cvt_f32_fp8(w[i], 1), part);
            part = fmaf(__builtin_amdgcn_cvt_f32_fp8(x[i], 2), __builtin_amdgcn_cvt_f32_fp8(w[i], 2), part);
            part = fmaf(__builtin_amdgcn_cvt_f32_fp8(x[i], 3), __builtin_amdgcn_cvt_f32_fp8(w[i], 3), part);
        }
        if constexpr (IN == IN_F8_F32) sum = fmaf(part, static_cast<const float*>(p.sa)[t * p.sa_block + src] * static_cast<const float*>(p.sb)[sb0 + t], sum);
        else sum += ldexpf(part, (int)static_cast<const unsigned char*>(p.sa)[t * p.sa_block + src] + (int)static_cast<const unsigned char*>(p.sb)[sb0 + t] - 254);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    return sum;
}
// 16 x 16 values: one wave's steps (of WAVES) of their sums, as the few-rows kernel makes them: row lane & 15 of either operand
template <int IN, int WAVES, int U>
__device__ __forceinline__ f32x4 sum_many(const ProductArgs& p, int g, int row, int end, int col, int wave, int lane)
{
    const int r = lane & 15, q = lane >> 4, c = col + r, whole = p.kbytes / KROW;
    const long long s0 = source_row(p, row + r, end), src = s0 < 0 ? 0 : s0, sb0 = g * p.sb_group + (long long)(col / BLK) * p.sb_row;
    const char* const x_row = p.a + src * p.a_row + q * 16;
    const char* const w_row = p.b + g * p.b_group + (long long)(c < p.n ? c : p.n - 1) * p.b_row + q * 16;
    f32x4 acc[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
    unsigned bad = 0;
    auto scale_at = [&](int s, unsigned& sw, unsigned& sx) {
        if constexpr (IN == IN_F8_F32) { sw = static_cast<const unsigned*>(p.sb)[sb0 + s]; sx = static_cast<const unsigned*>(p.sa)[s * p.sa_block + src]; }
        else { sw = static_cast<const unsigned char*>(p.sb)[sb0 + s]; sx = static_cast<const unsigned char*>(p.sa)[s * p.sa_block + src]; }
    };
    auto add = [&](i32x4 w0, i32x4 w1, i32x4 x0, i32x4 x1, unsigned sw, unsigned sx) {
        Frag<IN, true> wf[1], xf;
        Scale<IN, true> sc;
        wf[0].set(w0, w1, sw);
        xf.set(x0, x1, sx);
        sc.set(sw, sx, bad);
        mac_row<IN, true, 1>(acc, wf, xf, sc);
    };
#pragma unroll 1
    for (int s = wave; s < whole; s += WAVES * U) {
        i32x4 w[U][2], x[U][2];
        unsigned sw[U], sx[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = s + u * WAVES;
            if (t >= whole) continue;
            w[u][0] = load16(w_row + t * KROW); w[u][1] = load16(w_row + t * KROW + 64);
            x[u][0] = load16(x_row + t * KROW); x[u][1] = load16(x_row + t * KROW + 64);
            scale_at(t, sw[u], sx[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) if (s + u * WAVES < whole) add(w[u][0], w[u][1], x[u][0], x[u][1], sw[u], sx[u]);
    }
    if (p.kbytes % KROW && whole % WAVES == wave) {
        const int at = whole * KROW + q * 16;
        unsigned sw, sx;
        scale_at(whole, sw, sx);
        add(load16_tail(w_row - q * 16, at, p.kbytes), load16_tail(w_row - q * 16, at + 64, p.kbytes), load16_tail(x_row - q * 16, at, p.kbytes), load16_tail(x_row - q * 16, at + 64, p.kbytes), sw, sx);
    }
    return acc[0];
}
// f(block) for the blocks with many.  Every wave of the workgroup sees the same ones.
template <class T, class F>
__device__ __forceinline__ void blocks_of(const Doubts<T>& d, F f)
{
    const int bits = (int)d.blocks[threadIdx.x & 7];
#pragma unroll 1
    for (int w = 0; w < 8; ++w)
        for (unsigned left = (unsigned)__builtin_amdgcn_readlane(bits, w); left; left &= left - 1) f(w * 32 + __builtin_ctz(left));
}
// the barriers of store_tile, for waves of the workgroup that have no sums
template <class T>
__device__ __forceinline__ void stand_by(const char* smem)
{
    __syncthreads();
    __syncthreads();
    const Doubts<T>& d = *reinterpret_cast<const Doubts<T>*>(smem + T::BIAS - sizeof(Doubts<T>));
    const int found = __builtin_amdgcn_readfirstlane(d.found);
    for (int i = found & ~MANY; i > 0; i -= AT_ONCE) { __syncthreads(); __syncthreads(); }
    if (found & MANY) blocks_of<T>(d, [](int) { __syncthreads(); __syncthreads(); });
}

// What a tile kernel does with its sums: bias, ReLU, the scale of a row's 128 columns, and stores of whole 16-byte pieces of rows: a wave turns
// sixteen rows at a time round in its own corner of LDS (a lane holds four columns of a row, a store takes neighbouring lanes along a row).  Rows of y that
// do not start at multiples of four values are stored value by value.
template <int IN, int OUT, class T>
__device__ __forceinline__ void store_tile(const ProductArgs& p, f32x4 (&acc)[T::MT][T::NT], char* smem, int g, int first, int end, int n0, int wave, int lane)
{
    constexpr int SZ = OUT == OUT_F32 ? 4 : OUT == OUT_BF16 ? 2 : 1, ROW = T::NT * 16 * SZ, PITCH = ROW + 16, PER = BLK / (T::NT * 16);
    const int r = lane & 15, q = lane >> 4, wm = (wave / T::WN) * T::MT * 16, wn = (wave % T::WN) * T::NT * 16;
    float* const most = reinterpret_cast<float*>(smem);                       // [wave column][row]
    char* const turn = smem + (OUT == OUT_E4M3 ? T::WN * T::BM * 4 : 0) + wave * 16 * PITCH;
    using D = Doubts<T>;
    static_assert(T::WN * T::BM * 4 + T::WAVES * 16 * PITCH + sizeof(D) <= T::BIAS && T::BM * T::BN <= 256 * 256 && T::BN <= 256 && sizeof(D) % 16 == 0 && T::BIAS % 16 == 0, "LDS");
    D& doubts = *reinterpret_cast<D*>(smem + T::BIAS - sizeof(D));
    if constexpr (OUT == OUT_E4M3) {
        for (int i = wave * 64 + lane; i < T::BM * (T::BN / BLK); i += T::WAVES * 64) doubts.above[i] = 0;
        if (wave == 0 && lane < 8) doubts.blocks[lane] = 0;
        if (wave == 0 && lane == 8) doubts.found = 0;
    }
    auto finish = [&](float sum, float b) { const float y = sum + b; return p.relu && y < 0.f ? 0.f : y; };      // (NaN stays)
    auto bias_of = [&](int c) { return p.bias ? *reinterpret_cast<const f32x4*>(smem + T::BIAS + (c + q * 4) * 4) : f32x4{0.f, 0.f, 0.f, 0.f}; };
    unsigned live = 0;                                                        // the rows of this lane that have a source, a bit for each
#pragma unroll
    for (int i = 0; i < T::MT; ++i) live |= source_row(p, first + wm + i * 16 + r, end) >= 0 ? 1u << i : 0;
#pragma unroll
    for (int u = 0; u < T::NT; ++u) {
        const f32x4 bias = bias_of(wn + u * 16);
#pragma unroll
        for (int i = 0; i < T::MT; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[i][u][v] = finish(live >> i & 1 ? acc[i][u][v] : 0.f, bias[v]);
    }
    if constexpr (OUT == OUT_E4M3) {
        const int cb = (n0 + wn) / BLK, block = wn / BLK * T::BM;             // (of the result; of the tile)
        auto column = [&](int u, int v) { return n0 + wn + u * 16 + q * 4 + v; };
        float top[T::MT];
#pragma unroll
        for (int i = 0; i < T::MT; ++i) {
            float t = 0.f;
#pragma unroll
            for (int u = 0; u < T::NT; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) t = column(u, v) < p.n ? fmaxf(t, finite_abs(acc[i][u][v])) : t;
            t = fmaxf(t, __shfl_xor(t, 16));
            t = fmaxf(t, __shfl_xor(t, 32));
            if (q == 0) most[(wave % T::WN) * T::BM + wm + i * 16 + r] = t;
        }
        __syncthreads();
        unsigned many = 0, look = 0;                                          // (a bit for each of this lane's rows; for each sixteen rows)
#pragma unroll
        for (int i = 0; i < T::MT; ++i) {
            top[i] = 0.f;
#pragma unroll
            for (int u = 0; u < PER; ++u) top[i] = fmaxf(top[i], most[((wave % T::WN) / PER * PER + u) * T::BM + wm + i * 16 + r]);
            if (__ballot(live >> i & 1 && in_doubt(top[i]))) look |= 1u << i;
        }
        // (What follows runs seldom, so its instructions come from far away: unrolled, 1 KB of them for every
        // sixteen rows, 32768 rows of 2048 x 4736 took 292 us where they take 276 now.)
#pragma unroll 1
        for (; look; look &= look - 1) {
            const int i = __builtin_ctz(look);
            float limits = 0.f;                                               // lane r: the row's largest
#pragma unroll
            for (int k = 0; k < T::MT; ++k)
                if (k == i) {
                    limits = live >> k & 1 ? top[k] : 0.f;
#pragma unroll
                    for (int u = 0; u < T::NT; ++u) *reinterpret_cast<f32x4*>(&doubts.rows[wave][r][u * 16 + q * 4]) = acc[k][u];
                }
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (unsigned rows = (unsigned)__ballot(q == 0 && in_doubt(limits)); rows; rows &= rows - 1) {
                const int row = __builtin_ctz(rows), limit = border_of(__uint_as_float((unsigned)__builtin_amdgcn_readlane(__float_as_int(limits), row))) - UNDER;
                const int y = lane < T::NT * 16 ? __float_as_int(doubts.rows[wave][row][lane]) & 0x7fffffff : 0;
                const bool in = y > limit && y < 0x7f800000 && n0 + wn + lane < p.n;                           // (larger ones may lie above the border)
                const unsigned long long all = __ballot(in);
                if (__popcll(all) <= FEW) {
                    if (in) doubts.list[atomicAdd(&doubts.found, 1)] = (wm + i * 16 + row) << 8 | (wn + lane);
                } else {
                    many |= r == row ? 1u << i : 0;
                    const int b = (wm / 16 + i) * (T::BN / 16) + wn / 16 + lane;
                    if (lane < T::NT && (all >> lane * 16 & 0xffff)) atomicOr(&doubts.blocks[b >> 5], 1u << (b & 31));
                    if (lane == 0) atomicOr(&doubts.found, MANY);
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        const int state = __builtin_amdgcn_readfirstlane(doubts.found), found = state & ~MANY;
#pragma unroll 1
        for (int i0 = 0; i0 < found; i0 += AT_ONCE) {
            float* const parts = reinterpret_cast<float*>(doubts.parts);
#pragma unroll 1
            for (int i = i0; i < found && i < i0 + AT_ONCE; ++i) {
                const int e = __builtin_amdgcn_readfirstlane(doubts.list[i]);
                const float sum = sum_one<IN, T::WAVES>(p, g, source_row(p, first + (e >> 8), end), n0 + (e & 255), wave, lane);
                if (lane == 0) parts[(i - i0) * T::WAVES + wave] = sum;
            }
            __syncthreads();
            if (wave == 0 && i0 + lane < found) {                             // (the order of the list does not matter: a value says the same from any place)
                const int e = doubts.list[i0 + lane], lr = e >> 8, c = e & 255;
                float y = 0.f, largest = 0.f;
#pragma unroll
                for (int w = 0; w < T::WAVES; ++w) y += parts[lane * T::WAVES + w];
                y = finish(y, p.bias ? *reinterpret_cast<const float*>(smem + T::BIAS + c * 4) : 0.f);
#pragma unroll
                for (int u = 0; u < PER; ++u) largest = fmaxf(largest, most[(c / BLK * PER + u) * T::BM + lr]);
                if ((int)(__float_as_uint(y) & 0x7fffffffu) > border_of(largest)) doubts.above[c / BLK * T::BM + lr] = 1;
            }
            __syncthreads();
        }
        if (state & MANY) blocks_of<T>(doubts, [&](int b) {
            const int row = b / (T::BN / 16) * 16, col = b % (T::BN / 16) * 16;
            doubts.parts[wave][lane] = sum_many<IN, T::WAVES, T::MT * T::NT < 32 ? 2 : 1>(p, g, first + row, end, n0 + col, wave, lane);
            __syncthreads();
            if (row >= wm && row < wm + T::MT * 16 && col >= wn && col < wn + T::NT * 16) {
                f32x4 y = doubts.parts[0][lane];
#pragma unroll
                for (int w = 1; w < T::WAVES; ++w) y += doubts.parts[w][lane];
                const f32x4 bias = bias_of(col);
                int border = 0x7fffffff;                                      // (rows that are summed one by one, or not at all)
#pragma unroll
                for (int i = 0; i < T::MT; ++i) if (row == wm + i * 16 && many >> i & 1) border = border_of(top[i]);
                bool over = false;
#pragma unroll
                for (int v = 0; v < 4; ++v) over |= n0 + col + q * 4 + v < p.n && (int)(__float_as_uint(finish(y[v], bias[v])) & 0x7fffffffu) > border;
                if (over) doubts.above[block + row + r] = 1;
            }
            __syncthreads();
        });
#pragma unroll
        for (int i = 0; i < T::MT; ++i) {
            const int lr = wm + i * 16 + r, j = first + lr;
            if (state && live >> i & 1 && in_doubt(top[i])) top[i] = __uint_as_float((unsigned)(border_of(top[i]) + doubts.above[block + lr]));
            const int e = block_exponent(top[i]);
            const float inv = two_to(-e);
#pragma unroll
            for (int u = 0; u < T::NT; ++u) acc[i][u] *= inv;
            if (q == 0 && j < end && (wave % T::WN) % PER == 0 && cb * BLK < p.n) {
                if (IN == IN_F8_E8) static_cast<unsigned char*>(p.ys)[cb * p.ys_block + j] = (unsigned char)(e + 127);
                else static_cast<float*>(p.ys)[cb * p.ys_block + j] = two_to(e);
            }
        }
    }
    const bool whole = wide_stores(p, 16) && n0 + wn + T::NT * 16 <= p.n;
    const bool wide = wide_stores(p, 4 * SZ);
    char* const y0 = p.y + (long long)(n0 + wn) * SZ;
#pragma unroll
    for (int i = 0; i < T::MT; ++i) {
        const int j0 = first + wm + i * 16;
        if (whole || !wide) {
#pragma unroll
            for (int u = 0; u < T::NT; ++u) {
                char* at = turn + r * PITCH + (u * 16 + q * 4) * SZ;
                if constexpr (OUT == OUT_F32) *reinterpret_cast<f32x4*>(at) = acc[i][u];
                else if constexpr (OUT == OUT_BF16)
                    *reinterpret_cast<uint2*>(at) = make_uint2(to_bf16(acc[i][u][0]) | (unsigned)to_bf16(acc[i][u][1]) << 16, to_bf16(acc[i][u][2]) | (unsigned)to_bf16(acc[i][u][3]) << 16);
                else *reinterpret_cast<int*>(at) = to_e4m3x4(acc[i][u][0], acc[i][u][1], acc[i][u][2], acc[i][u][3]);
            }
            __builtin_amdgcn_wave_barrier();
            if (whole) {
                constexpr int CH = ROW / 16;                                  // 16-byte pieces of a row
#pragma unroll
                for (int t = 0; t < (CH * 16 + 63) / 64; ++t) {
                    const int row = (t * 64 + lane) / CH, c = (t * 64 + lane) % CH;
                    if (row >= 16) break;
                    const i32x4 v = *reinterpret_cast<const i32x4*>(turn + row * PITCH + c * 16);
                    if (j0 + row < end) *reinterpret_cast<i32x4*>(y0 + (long long)(j0 + row) * p.y_row + c * 16) = v;
                }
            } else {                                                          // (neighbouring lanes: neighbouring values of a row)
                using E = std::conditional_t<OUT == OUT_F32, float, std::conditional_t<OUT == OUT_BF16, unsigned short, char>>;
#pragma unroll 4
                for (int t = 0; t < T::NT * 4; ++t) {
                    const int row = (t * 64 + lane) / (T::NT * 16), c = (t * 64 + lane) % (T::NT * 16);
                    E v;
                    __builtin_memcpy(&v, turn + row * PITCH + c * SZ, SZ);    // (written as words: to the compiler another type's memory)
                    if (j0 + row < end && n0 + wn + c < p.n) *reinterpret_cast<E*>(y0 + (long long)(j0 + row) * p.y_row + c * SZ) = v;
                }
            }
            __builtin_amdgcn_wave_barrier();
        } else if (j0 + r < end) {
#pragma unroll
            for (int u = 0; u < T::NT; ++u) {
                const int c = n0 + wn + u * 16 + q * 4;
                if (c < p.n) store4<OUT>(p, j0 + r, c, acc[i][u], wide);
            }
        }
    }
}

// The sums of the groups that share K, group 0's first; the other group is done then
template <int OUT, class T>
__device__ __forceinline__ bool gather_groups(f32x4 (&acc)[T::MT][T::NT], char* smem, int kg, int wave, int lane)
{
    if constexpr (T::KG == 2) {
        constexpr int B = T::MT * T::NT;
        static_assert(T::WAVES * B * 1024 <= T::BIAS, "LDS");
        f32x4* const sums = reinterpret_cast<f32x4*>(smem) + wave * B * 64 + lane;
        if (kg == 1) {
#pragma unroll
            for (int i = 0; i < B; ++i) sums[i * 64] = acc[i / T::NT][i % T::NT];
        }
        __syncthreads();
        if (kg == 0) {
#pragma unroll
            for (int i = 0; i < B; ++i) acc[i / T::NT][i % T::NT] += sums[i * 64];
        }
        __syncthreads();
        if (kg == 1) {
            if (OUT == OUT_E4M3) stand_by<T>(smem);
            return false;
        }
    }
    return true;
}

template <int IN, int OUT, class T>
__global__ __launch_bounds__(T::THREADS, 2) void product_ring_kernel(ProductArgs p)
{
    constexpr bool EXACT = OUT == OUT_F32;
    constexpr int BM = T::BM, MT = T::MT, NT = T::NT, NBUF = T::NBUF, KG = T::KG, PS = IN != IN_BF16;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    Place place;
    if (!find_tile(p, BM, place)) return;
    const int g = place.g, first = place.first, end = place.end, n0 = place.tn * T::BN;
    const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all % T::WAVES, kg = all / T::WAVES, r = lane & 15, q = lane >> 4;
    const int wm = (wave / T::WN) * MT * 16, wn = (wave % T::WN) * NT * 16;
    const int total = (p.kbytes + KROW - 1) / KROW, rounds = (total + KG - 1) / KG;   // this group's steps: kg, kg + KG, ..; a round: one of every group
    const int steps = kg < total ? (total - kg + KG - 1) / KG : 0;
    const int tail = p.kbytes % KROW;                                         // bytes of the last step, where K ends inside it
    const bool mine = tail && (total - 1) % KG == kg;                         // ... and it is this group's

    unsigned from[T::PIECES];                                                 // from the step's column of a, of the group's b
#pragma unroll
    for (int i = 0; i < T::PIECES; ++i) {
        const int lr = (i * T::WAVES + wave) * 8 + (lane >> 3), col = ((lane & 7) ^ ((lr >> 1) & 7)) * 16;
        unsigned row;
        if ((i * T::WAVES + wave) * 8 < BM) { const long long s = source_row(p, first + lr, end); row = (unsigned)(s < 0 ? 0 : s) * (unsigned)p.a_row; }   // (no source: any row, taken out at the end)
        else { const int c = n0 + lr - BM; row = (unsigned)(c < p.n ? c : p.n - 1) * (unsigned)p.b_row; }
        asm volatile("" : "+v"(row));                                         // (a product and a sum of 32 bits: not the instruction whose result fills two registers)
        from[i] = row + col;
    }
    // scales: waves 0 .. SA - 1 bring those of 64 rows each, the last wave that of the columns
    constexpr int SZ = IN == IN_F8_F32 ? 4 : 1;
    const bool rows_too = PS && wave < T::SA, cols_too = PS && wave == T::WAVES - 1;
    const char *ka = p.a + kg * KROW, *kb = p.b + g * p.b_group + kg * KROW, *ks = nullptr;
    long long s_step = 0;
    unsigned s_at = 0;
    if (rows_too) {
        const long long s = wave * 64 + lane < BM ? source_row(p, first + wave * 64 + lane, end) : -1;
        s_at = (unsigned)(s < 0 ? 0 : s) * SZ;
        ks = static_cast<const char*>(p.sa) + kg * p.sa_block * SZ;
        s_step = KG * p.sa_block * SZ;
    } else if (cols_too) {
        ks = static_cast<const char*>(p.sb) + (g * p.sb_group + (long long)place.tn * p.sb_row + kg) * SZ;
        s_step = KG * SZ;
    }
    char* const ring = smem + kg * NBUF * T::BUF;
    const unsigned lds0 = lds_addr(ring);
    int to = 0;                                                               // the buffer of the next step asked for
    auto tail_col = [&](int i) { const int lr = (i * T::WAVES + wave) * 8 + (lane >> 3); return ((lane & 7) ^ ((lr >> 1) & 7)) * 16; };
    // pieces lo .. hi - 1 of this group's step s (behind the last one: its scales)
    auto bring = [&](int s, int lo, int hi) {
        const unsigned at = lds0 + to * T::BUF;
        if (lo == 0 && mine && s == steps - 1) {                              // chunks behind the end: any that are there, made zeros below
#pragma unroll
            for (int i = 0; i < T::PIECES; ++i) if (tail_col(i) >= tail) from[i] -= tail_col(i);
        }
#pragma unroll
        for (int i = 0; i < T::PIECES; ++i) if (i >= lo && i < hi) dma16s((i * T::WAVES + wave) * 8 < BM ? ka : kb, from[i], at + (i * T::WAVES + wave) * 1024);
        if (hi < T::PIECES) return;
        ka += KG * KROW;
        kb += KG * KROW;
        if constexpr (PS)
            if (rows_too || cols_too) {
                const unsigned slot = at + T::PANELS + (cols_too ? T::SA : wave) * 256;
                if constexpr (SZ == 4) dma4s(ks, s_at, slot);
                else dma1s(ks, s_at, slot);
                ks += s_step;
            }
        to = to == NBUF - 1 ? 0 : to + 1;
    };
    // all of this wave's requests but those of the last `ahead` steps have landed
    auto landed = [&](auto ahead) {
        constexpr int N = decltype(ahead)::value;
        if (rows_too || cols_too) wait_all_but<N * (T::PIECES + 1)>();
        else wait_all_but<N * T::PIECES>();
    };

    f32x4 acc[MT][NT];
    unsigned bad[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        bad[i] = 0;
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bring_bias<T>(p, smem, g, n0, all, lane);
#pragma unroll
    for (int s = 0; s < NBUF; ++s) if (s < steps) bring(s, 0, T::PIECES);
    int buf = 0;
    struct Step { i32x4 w0[NT], w1[NT], x0[MT], x1[MT]; unsigned sw, sx[MT]; } even, odd;
    // step s is there, for every wave, and the fragments of step s - 1 have been read (so its buffer is free)
    auto arrive = [&](int s, auto ahead) {
        if (s + decltype(ahead)::value < steps) landed(ahead);
        else wait_all_but<0>();                                               // (fewer are under way at the end)
        if (mine && s == steps - 1) {
#pragma unroll
            for (int i = 0; i < T::PIECES; ++i)
                if (tail_col(i) >= tail) *reinterpret_cast<i32x4*>(ring + buf * T::BUF + (i * T::WAVES + wave) * 1024 + lane * 16) = i32x4{0, 0, 0, 0};
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    auto read = [&](Step& f) {
        const char* const xa = ring + buf * T::BUF;
        const char* const wa = xa + BM * KROW;
        const unsigned* const scales = reinterpret_cast<const unsigned*>(xa + T::PANELS);
#pragma unroll
        for (int j = 0; j < NT; ++j) { f.w0[j] = chunk(wa, wn + j * 16 + r, q); f.w1[j] = chunk(wa, wn + j * 16 + r, q + 4); }
#pragma unroll
        for (int i = 0; i < MT; ++i) { f.x0[i] = chunk(xa, wm + i * 16 + r, q); f.x1[i] = chunk(xa, wm + i * 16 + r, q + 4); }
        if (PS) {
            f.sw = scales[T::SA * 64];
#pragma unroll
            for (int i = 0; i < MT; ++i) f.sx[i] = scales[wm + i * 16 + r];
        }
        buf = buf == NBUF - 1 ? 0 : buf + 1;
    };
    auto step = [&](int s, const Step& f, Step& next) {
        if (s + 1 < rounds) {                                                 // (every group comes to every barrier)
            arrive(s + 1, std::integral_constant<int, NBUF - 2>{});
            if (s + 1 < steps) read(next);
        }
        if (s >= steps) return;
        constexpr bool LATE = MT * NT < 16;                                   // (a second row of block sums would spill)
        Frag<IN, EXACT> w[NT];
        f32x4 part[2][NT];
        Scale<IN, EXACT> sc[2];
#pragma unroll
        for (int j = 0; j < NT; ++j) w[j].set(f.w0[j], f.w1[j], f.sw);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            Frag<IN, EXACT> x;
            x.set(f.x0[i], f.x1[i], PS ? f.sx[i] : 0);
            if (PS) sc[i & 1].set(f.sw, f.sx[i], bad[i]);
            mfma_row<IN, EXACT, NT>(acc[i], part[i & 1], w, x, sc[i & 1]);
            if (s + NBUF < steps) {                                           // requests between the instructions, some behind each row: the pipe is busy while they are issued
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if constexpr (FOLDS<IN, EXACT>) asm volatile("" :: "v"(part[i & 1][j]));
                    else asm volatile("" :: "v"(acc[i][j]));
                }
                __builtin_amdgcn_sched_barrier(0);
                bring(s + NBUF, i * T::PIECES / MT, (i + 1) * T::PIECES / MT);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (LATE && i > 0) fold_row<IN, EXACT, NT>(acc[i - 1], part[(i - 1) & 1], sc[(i - 1) & 1]);
            if (!LATE) fold_row<IN, EXACT, NT>(acc[i], part[i & 1], sc[i & 1]);
        }
        if (LATE) fold_row<IN, EXACT, NT>(acc[MT - 1], part[(MT - 1) & 1], sc[(MT - 1) & 1]);
    };
    arrive(0, std::integral_constant<int, NBUF - 1>{});
    if (steps > 0) read(even);
    for (int s = 0; s < rounds; s += 2) {
        step(s, even, odd);
        if (s + 1 < rounds) step(s + 1, odd, even);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) spoil<IN, EXACT, NT>(acc[i], bad[i]);
    __syncthreads();                                                          // the panels have been read: LDS is the epilogue's
    if (!gather_groups<OUT, T>(acc, smem, kg, wave, lane)) return;
    store_tile<IN, OUT, T>(p, acc, smem, g, first, end, n0, wave, lane);
}

// ---- the kernel for operands at any address: panels come through registers as whole words, two steps ahead, and are shifted to their bytes on the way to
//      LDS (a lane's last word is its neighbour's first).  Bound: the shifts and a wave's latencies, so the small tile's steps are dealt out to two groups
//      of waves as the ring's are.  733 rows of 1001 x 1419 to fp32: 16-byte loads from any address and a last step byte by byte 22.6 us, whole words
//      14.5, two groups 12.9.
template <int WM_, int WN_, int MT_, int NT_, int KG_> struct Any {
    static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_, KG = KG_, BM = WM * MT * 16, BN = WN * NT * 16, WAVES = WM * WN, THREADS = 64 * WAVES * KG;
    static constexpr int AT_ONCE = WAVES * 8, CH = (BM + BN) / AT_ONCE, BIAS = KG * 2 * (BM + BN) * KROW, LDS = BIAS + BN * 4;   // rows that a group brings together; 16-byte chunks a thread and step
    static_assert(BN == BLK && BM % AT_ONCE == 0 && BN % AT_ONCE == 0, "tile");
};

template <int IN, int OUT, class T>
__global__ __launch_bounds__(T::THREADS, 2) void product_any_kernel(ProductArgs p)
{
    constexpr int BM = T::BM, BN = T::BN, CH = T::CH, MT = T::MT, NT = T::NT;
    constexpr bool EXACT = OUT == OUT_F32;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    Place at;
    if (!find_tile(p, BM, at)) return;
    const int g = at.g, first = at.first, end = at.end, tn = at.tn;
    const int n0 = tn * BN, lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all % T::WAVES, kg = all / T::WAVES, r = lane & 15, q = lane >> 4;
    const int wm = (wave / T::WN) * MT * 16, wn = (wave % T::WN) * NT * 16;
    const int total = p.a_rows ? (p.kbytes + KROW - 1) / KROW : 0, rounds = (total + T::KG - 1) / T::KG;    // this group's steps: kg, kg + KG, ..; a round: one of every group
    const int steps = kg < total ? (total - kg + T::KG - 1) / T::KG : 0, t8 = wave * 8 + (lane >> 3);

    const char* row[CH];                                                      // (rows without a source and columns behind the last: any, not stored or taken out at the end)
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int lr = t8 + T::AT_ONCE * i;
        if (lr < BM) { const long long s = source_row(p, first + lr, end); row[i] = p.a + (s < 0 ? 0 : s) * p.a_row; }
        else { const int c = n0 + lr - BM; row[i] = p.b + g * p.b_group + (long long)(c < p.n ? c : p.n - 1) * p.b_row; }
    }
    const int c8 = threadIdx.x & 7;
    long long mine[MT];                                                       // the rows whose scales this lane applies
#pragma unroll
    for (int i = 0; i < MT; ++i) { const long long s = source_row(p, first + wm + i * 16 + r, end); mine[i] = s < 0 ? 0 : s; }
    const long long sb0 = g * p.sb_group + (long long)tn * p.sb_row;
    struct Step { i32x4 v[CH]; int next[CH]; unsigned sw, sx[MT]; } even, odd;
    auto fetch = [&](int round, Step& f) {
        const int s = round * T::KG + kg;
        const int from = s * KROW + c8 * 16;
        if ((s + 1) * KROW <= p.kbytes) {
#pragma unroll
            for (int i = 0; i < CH; ++i) __builtin_memcpy(&f.v[i], __builtin_assume_aligned(word_of(row[i]) + from, 4), 16);
        } else {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int last = last_word(row[i], p.kbytes);
#pragma unroll
                for (int j = 0; j < 4; ++j) f.v[i][j] = word_at(word_of(row[i]), from + 4 * j < last ? from + 4 * j : last);
            }
        }
        if (c8 == 7) {
#pragma unroll
            for (int i = 0; i < CH; ++i) { const int last = last_word(row[i], p.kbytes); f.next[i] = word_at(word_of(row[i]), from + 16 < last ? from + 16 : last); }
        }
        if constexpr (IN == IN_F8_F32) {
            f.sw = static_cast<const unsigned*>(p.sb)[sb0 + s];
#pragma unroll
            for (int i = 0; i < MT; ++i) f.sx[i] = static_cast<const unsigned*>(p.sa)[s * p.sa_block + mine[i]];
        }
        if constexpr (IN == IN_F8_E8) {
            f.sw = static_cast<const unsigned char*>(p.sb)[sb0 + s];
#pragma unroll
            for (int i = 0; i < MT; ++i) f.sx[i] = static_cast<const unsigned char*>(p.sa)[s * p.sa_block + mine[i]];
        }
    };

    f32x4 acc[MT][NT];
    unsigned bad[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        bad[i] = 0;
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    auto step = [&](int round, Step& f) {
        const int s = round * T::KG + kg;
        char* const lds = smem + (kg * 2 + (round & 1)) * (BM + BN) * KROW;   // (last read two rounds ago: a barrier lies between)
        if (round >= steps) { __syncthreads(); return; }                      // (every group comes to every barrier)
        const int left = p.kbytes - s * KROW - c8 * 16;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int over = __builtin_amdgcn_update_dpp(0, f.v[i][0], 0x101, 0xf, 0xf, false);          // the next lane's first word
            i32x4 v = shift_words(f.v[i], c8 == 7 ? f.next[i] : over, (unsigned)reinterpret_cast<uintptr_t>(row[i]) & 3);
            if ((s + 1) * KROW > p.kbytes) v = cut_bytes(v, left);
            *reinterpret_cast<i32x4*>(lds + slot_of(t8 + T::AT_ONCE * i, c8)) = v;
        }
        unsigned sw = f.sw, sx[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) sx[i] = f.sx[i];
        if (round + 2 < steps) fetch(round + 2, f);
        __syncthreads();
        Frag<IN, EXACT> w[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) { const int wr = BM + wn + j * 16 + r; w[j].set(chunk(lds, wr, q), chunk(lds, wr, q + 4), sw); }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            Frag<IN, EXACT> x;
            x.set(chunk(lds, wm + i * 16 + r, q), chunk(lds, wm + i * 16 + r, q + 4), sx[i]);
            Scale<IN, EXACT> sc;
            if (IN != IN_BF16) sc.set(sw, sx[i], bad[i]);
            mac_row<IN, EXACT, NT>(acc[i], w, x, sc);
        }
    };
    even.sw = odd.sw = 0;
#pragma unroll
    for (int i = 0; i < MT; ++i) even.sx[i] = odd.sx[i] = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) even.next[i] = odd.next[i] = 0;
    bring_bias<T>(p, smem, g, n0, all, lane);
    if (steps > 0) fetch(0, even);
    if (steps > 1) fetch(1, odd);
    for (int s = 0; s < rounds; s += 2) {
        step(s, even);
        if (s + 1 < rounds) step(s + 1, odd);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) spoil<IN, EXACT, NT>(acc[i], bad[i]);
    wait_all_but<0>();
    __syncthreads();                                                          // the panels have been read: LDS is the epilogue's
    if (!gather_groups<OUT, T>(acc, smem, kg, wave, lane)) return;
    store_tile<IN, OUT, T>(p, acc, smem, g, first, end, n0, wave, lane);
}

// ---- the kernel for chip-filling products (operands within 4 GB): eight waves in two groups that are a phase apart.
//
// Waves w and w + 4 share a SIMD.  While one group's phase is its matrix instructions, the other group's is reads of fragments from LDS, requests and
// waits: the matrix pipe passes from one group to the other, and no wave waits for LDS with the pipe idle.  A step of group 0 is L0 M0 .. (of H = MT / XG
// pairs; L: XG rows of blocks read, M: multiplied; L0 reads all of the weights' fragments too), from phase 2H s on; group 1 runs the same one phase
// later; a barrier ends every phase.
//
// Panels (64 KB a step of 256 x 256) have to be asked for more than a step ahead.  Two buffers: each part of a panel once its buffer has been read for the
// last time, in L phases behind the reads -- of step s + 2 the weights and the first rows in the last L of step s, the other rows (then read themselves) in
// L0 of step s + 1; five phases or more lie between a request and its use.  Three buffers (smaller tiles, whose L phases are longer than their M phases):
// between matrix instructions, step s + 2 at phase 2H s + 1, by group 1 at 2H s.  Scales come the same way, a word a row.
//
// What bounds it, at 8192 x 2048 over long K: 1.10 us a step of 256 x 256 (zeros: the clock at its highest), with or without its requests, 0.87 of them
// matrix instructions and the rest the phases' barriers; 1.39 with random operands, where the power limit sets the clock (a library product of one scale
// for all: 0.86 and 1.18).  Requests between matrix instructions took 1.45 and 1.7 there.  Counters, 32768 rows of 2048 x 4736: 546 thousand cycles with
// zeros and with random operands, 238 and 264 .. 284 us; the matrix pipe is busy in 56 % of them, a wave waits in 38 % of its own; 4 % of the LDS cycles are
// conflicts, 78 % of the requests find their line in the L2.  8192^3: e4m3 415 us, 2650 TFLOP/s; bf16 781, 1408.
template <int WM_, int WN_, int MT_, int NT_, int NBUF_> struct Phased {
    static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_, NBUF = NBUF_;
    static constexpr int BM = WM * MT * 16, BN = WN * NT * 16, WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int BUF = (BM + BN) * KROW, PA = BM / 64, PB = BN / 64;   // pieces of eight rows a wave brings: of its group's rows, of the weights
    static constexpr int SLOT = (BM + 64) * 4;                                // a step's scales: the rows', the column blocks'
    static constexpr int BIAS = NBUF * BUF + 4 * SLOT, LDS = BIAS + BN * 4;
    template <int IN> static constexpr bool TAIL = !(MT == 8 && IN == IN_F8_F32);   // (no register left where block sums are folded)
    static_assert(WM == 2 && WN == 4 && BN / BLK <= 64 && (NBUF == 2 || NBUF == 3), "two groups of four waves");
};

template <int IN, int OUT, class T>
__global__ __launch_bounds__(T::THREADS, 2) void product_phased_kernel(ProductArgs p)
{
    constexpr bool EXACT = OUT == OUT_F32;
    constexpr int BM = T::BM, MT = T::MT, NT = T::NT, XG = MT % 4 == 0 ? 4 : 3, H = MT / XG;
    constexpr int PA = T::PA, PB = T::PB, PS = IN != IN_BF16, NBUF = T::NBUF;
    static_assert(MT % XG == 0 && (NBUF == 3 || H == 2), "phases");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    Place place;
    if (!find_tile(p, BM, place)) return;
    const int g = place.g, first = place.first, end = place.end, n0 = place.tn * T::BN;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, q = lane >> 4;
    const int grp = wave >> 2, w4 = wave & 3, wm = grp * MT * 16, wn = w4 * NT * 16;
    const int steps = (p.kbytes + KROW - 1) / KROW, tail = T::template TAIL<IN> ? p.kbytes % KROW : 0;      // (tail: bytes of the last step, where K ends inside it)

    const int col = ((lane & 7) ^ ((w4 & 1) * 4 + (lane >> 4))) * 16;         // this lane's chunk of a row (a wave's pieces of eight rows are all even ones or all odd ones)
    const bool cut = tail && col >= tail;                                     // ... lies behind the end in the last step: the first is read in its place and made zeros
    unsigned from[PA + PB];                                                   // from the step's column of a, of the group's b
#pragma unroll
    for (int i = 0; i < PA + PB; ++i) {
        const int lr = (i < PA ? grp * (BM / 16) + i * 4 + w4 : (i - PA) * 8 + wave) * 8 + (lane >> 3);
        unsigned row;
        if (i < PA) { const long long s = source_row(p, first + lr, end); row = (unsigned)(s < 0 ? 0 : s) * (unsigned)p.a_row; }
        else { const int c = n0 + lr; row = (unsigned)(c < p.n ? c : p.n - 1) * (unsigned)p.b_row; }
        asm volatile("" : "+v"(row));                                         // (a product and a sum of 32 bits: not the instruction whose result fills two registers)
        from[i] = row + col;
    }
    const unsigned lds0 = lds_addr(smem);
    const char* const b0 = p.b + g * p.b_group;
    // group 0 brings the scales of 64 rows a wave, group 1 those of the column blocks (every wave the same ones)
    constexpr int SZ = IN == IN_F8_F32 ? 4 : 1;
    const char* s_from = nullptr;
    long long s_step = 0;
    unsigned s_at = 0, s_to = 0;
    if (PS && grp == 0) {
        const int lr = w4 * 64 % BM + lane;
        const long long s = source_row(p, first + lr, end);
        s_from = static_cast<const char*>(p.sa);
        s_step = p.sa_block * SZ;
        s_at = (unsigned)(s < 0 ? 0 : s) * SZ;
        s_to = w4 * 64 % BM * 4;
    } else if (PS) {
        const int u = n0 / BLK + lane % (T::BN / BLK), last = (p.n - 1) / BLK;
        s_from = static_cast<const char*>(p.sb) + (g * p.sb_group + (long long)(n0 / BLK) * p.sb_row) * SZ;
        s_step = SZ;
        s_at = (unsigned)((u < last ? u : last) - n0 / BLK) * (unsigned)(p.sb_row * SZ);
        s_to = BM * 4;
    }
    // pieces lo .. hi - 1 of a step: the weights' (PB), the scales (PS), the group's rows (PA)
    auto bring = [&](int s, int buf, int lo, int hi) {
#pragma unroll
        for (int t = 0; t < PB + PS + PA; ++t) {
            if (t < lo || t >= hi) continue;
            if (tail && s == steps - 1 && (t < PB || t >= PB + PS)) from[t < PB ? PA + t : t - PB - PS] -= cut ? col : 0;
            if (t < PB) dma16s(b0 + (long long)s * KROW, from[PA + t], lds0 + buf * T::BUF + (BM / 8 + t * 8 + wave) * 1024);
            else if (t < PB + PS) {
                const unsigned to = lds0 + NBUF * T::BUF + (s & 3) * T::SLOT + s_to;
                if constexpr (SZ == 4) dma4s(s_from + s * s_step, s_at, to);
                else dma1s(s_from + s * s_step, s_at, to);
            } else dma16s(p.a + (long long)s * KROW, from[t - PB - PS], lds0 + buf * T::BUF + (grp * (BM / 16) + (t - PB - PS) * 4 + w4) * 1024);
        }
    };
    auto clear_tail = [&](int buf) {                                          // once this wave's pieces of the last step are there, before the barrier that says so
        if (!cut) return;
#pragma unroll
        for (int t = 0; t < PA + PB; ++t) {
            const int piece = t < PA ? grp * (BM / 16) + t * 4 + w4 : BM / 8 + (t - PA) * 8 + wave;
            *reinterpret_cast<i32x4*>(smem + buf * T::BUF + piece * 1024 + lane * 16) = i32x4{0, 0, 0, 0};
        }
    };
    constexpr int ALL = PB + PS + PA, FIRST = NBUF == 2 ? PB + PS + XG / 2 : ALL;   // (two buffers: rows that the first reads of a step take, XG / 2 pieces a wave, are free before the rest)
    auto phase_end = [&] {                                                    // (matrix instructions touch no memory: the scheduling barriers keep them in their phase)
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };

    auto pin = [&](const f32x4 (&row)[NT]) {                                  // the instructions that made these sums stay in front of what follows (they touch no memory:
#pragma unroll
        for (int j = 0; j < NT; ++j) asm volatile("" :: "v"(row[j]));         // the compiler would put them off, behind the waits)
    };

    f32x4 acc[MT][NT];
    unsigned bad[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        bad[i] = 0;
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bring_bias<T>(p, smem, g, n0, wave, lane);
    bring(0, 0, 0, ALL);
    if (steps > 1) { bring(1, 1, 0, FIRST); wait_all_but<FIRST>(); }
    else { wait_all_but<0>(); clear_tail(0); }
    phase_end();
    if (grp == 1) {
        if (NBUF == 3 && steps > 2) bring(2, 2, 0, ALL);
        phase_end();
    }
    int buf = 0;                                                              // of step s
    for (int s = 0; s < steps; ++s) {
        const int buf1 = buf == NBUF - 1 ? 0 : buf + 1, buf2 = buf1 == NBUF - 1 ? 0 : buf1 + 1;      // of the steps behind it
        const char* const xa = smem + buf * T::BUF;
        const char* const wa = xa + BM * KROW;
        const unsigned* const scales = reinterpret_cast<const unsigned*>(smem + NBUF * T::BUF + (s & 3) * T::SLOT);
        const bool more1 = s + 1 < steps, more2 = s + 2 < steps;
        // what the next reads but one phase need is there: the last two sets of requests are not part of it
        auto landed = [&](int h) {
            if (h < H - 1 ? !more1 : !more2) wait_all_but<0>();
            else if (h == H - 1 && XG % 2) wait_all_but<FIRST>();             // (a piece holds rows of both reads)
            else wait_all_but<ALL>();
            if (h == H - 1 && s + 2 == steps) clear_tail(buf1);
        };
        Frag<IN, EXACT> w[NT];
        unsigned sw = 0;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            // ---- L
            if (h == 0) {
                if (PS) sw = scales[BM + wn / BLK];
#pragma unroll
                for (int j = 0; j < NT; ++j) w[j].set(chunk(wa, wn + j * 16 + r, q), chunk(wa, wn + j * 16 + r, q + 4), sw);
            }
            Frag<IN, EXACT> x[XG];
            unsigned sv[XG];
#pragma unroll
            for (int i = 0; i < XG; ++i) {
                const int row = wm + (h * XG + i) * 16 + r;
                if (PS) sv[i] = scales[row];
                x[i].set(chunk(xa, row, q), chunk(xa, row, q + 4), PS ? sv[i] : 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (NBUF == 3) {}
            else if (h == H - 1) { if (more2) bring(s + 2, buf, 0, FIRST); }
            else if (more1) bring(s + 1, buf1, FIRST, ALL);
            if (grp == 1) landed(h);
            phase_end();
            // ---- M
            __builtin_amdgcn_s_setprio(1);
            f32x4 part[2][NT];
            Scale<IN, EXACT> sc[2];
#pragma unroll
            for (int i = 0; i < XG; ++i) {
                if (PS) sc[i & 1].set(sw, sv[i], bad[h * XG + i]);
                mfma_row<IN, EXACT, NT>(acc[h * XG + i], part[i & 1], w, x[i], sc[i & 1]);
                if (NBUF == 3 && s + 2 + grp < steps && i < XG - 1) {         // requests between the instructions, some behind each row: the pipe is busy while they are issued
                    if constexpr (FOLDS<IN, EXACT>) pin(part[i & 1]);
                    else pin(acc[h * XG + i]);
                    __builtin_amdgcn_sched_barrier(0);
                    bring(s + 2 + grp, grp ? buf : buf2, i * ALL / (XG - 1), (i + 1) * ALL / (XG - 1));
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (i > 0) fold_row<IN, EXACT, NT>(acc[h * XG + i - 1], part[(i - 1) & 1], sc[(i - 1) & 1]);
            }
            fold_row<IN, EXACT, NT>(acc[h * XG + XG - 1], part[(XG - 1) & 1], sc[(XG - 1) & 1]);
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int i = 0; i < XG; ++i) pin(acc[h * XG + i]);
            if (grp == 0) landed(h);
            phase_end();
        }
        buf = buf1;
    }
    if (grp == 0) phase_end();
#pragma unroll
    for (int i = 0; i < MT; ++i) spoil<IN, EXACT, NT>(acc[i], bad[i]);
    store_tile<IN, OUT, T>(p, acc, smem, g, first, end, n0, wave, lane);
}

// ---- the kernel for few rows a group: 16 MT rows x 16 columns a workgroup, K dealt out to its sixteen waves step by step, the waves' sums added in LDS in
//      their order.  What it does is read the weights once: operands go straight into registers, U steps of them asked for before the first is used.
//      Any alignment.
template <int IN, int OUT, int MT, int U>
__global__ __launch_bounds__(1024) void product_rows_kernel(ProductArgs p)
{
    constexpr bool EXACT = OUT == OUT_F32;
    constexpr int WAVES = 16;
    __shared__ __attribute__((aligned(16))) f32x4 part[WAVES][MT][64];
    Place place;
    if (!find_tile(p, MT * 16, place)) return;
    const int g = place.g, first = place.first, end = place.end, n0 = place.tn * 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int steps = (p.kbytes + KROW - 1) / KROW;
    const int c = n0 + r;
    const char* const w_row = p.b + g * p.b_group + (long long)(c < p.n ? c : p.n - 1) * p.b_row;
    const char* x_row[MT];
    long long src[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long long s = source_row(p, first + i * 16 + r, end);
        src[i] = s < 0 ? 0 : s;                                               // rows without a source: any row, taken out at the end
        x_row[i] = p.a + src[i] * p.a_row;
    }
    const long long sb0 = g * p.sb_group + (long long)(n0 / BLK) * p.sb_row;
    f32x4 bias;                                                               // (asked for here, used at the end)
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = p.bias && n0 + q * 4 + i < p.n ? p.bias[g * p.bias_group + n0 + q * 4 + i] : 0.f;
    f32x4 acc[MT][1];
    unsigned bad[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) { acc[i][0] = f32x4{0.f, 0.f, 0.f, 0.f}; bad[i] = 0; }
    for (int s0 = wave; s0 < steps; s0 += WAVES * U) {
        i32x4 w[U][2], x[U][MT][2];
        unsigned sw[U], sx[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * WAVES;
            if (s < steps) {
                const int at = s * KROW + q * 16;
                if ((s + 1) * KROW <= p.kbytes) {
                    w[u][0] = load16(w_row + at); w[u][1] = load16(w_row + at + 64);
#pragma unroll
                    for (int i = 0; i < MT; ++i) { x[u][i][0] = load16(x_row[i] + at); x[u][i][1] = load16(x_row[i] + at + 64); }
                } else {
                    w[u][0] = load16_tail(w_row, at, p.kbytes); w[u][1] = load16_tail(w_row, at + 64, p.kbytes);
#pragma unroll
                    for (int i = 0; i < MT; ++i) { x[u][i][0] = load16_tail(x_row[i], at, p.kbytes); x[u][i][1] = load16_tail(x_row[i], at + 64, p.kbytes); }
                }
                if (IN == IN_F8_F32) {
                    sw[u] = static_cast<const unsigned*>(p.sb)[sb0 + s];
#pragma unroll
                    for (int i = 0; i < MT; ++i) sx[u][i] = static_cast<const unsigned*>(p.sa)[s * p.sa_block + src[i]];
                } else if (IN == IN_F8_E8) {
                    sw[u] = static_cast<const unsigned char*>(p.sb)[sb0 + s];
#pragma unroll
                    for (int i = 0; i < MT; ++i) sx[u][i] = static_cast<const unsigned char*>(p.sa)[s * p.sa_block + src[i]];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u * WAVES < steps) {
                Frag<IN, EXACT> wf[1], xf;
                wf[0].set(w[u][0], w[u][1], IN != IN_BF16 ? sw[u] : 0);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    xf.set(x[u][i][0], x[u][i][1], IN != IN_BF16 ? sx[u][i] : 0);
                    Scale<IN, EXACT> sc;
                    if (IN != IN_BF16) sc.set(sw[u], sx[u][i], bad[i]);
                    mac_row<IN, EXACT, 1>(acc[i], wf, xf, sc);
                }
            }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) { spoil<IN, EXACT, 1>(acc[i], bad[i]); part[wave][i][lane] = acc[i][0]; }
    __syncthreads();
    if (threadIdx.x >= MT * 64) return;
    const int j = first + wave * 16 + r, col = n0 + q * 4;                    // (waves 0 .. MT - 1: a row tile each)
    f32x4 y = part[0][wave][lane];
#pragma unroll
    for (int u = 1; u < WAVES; ++u) y += part[u][wave][lane];
    if (j >= end) return;
    if (p.index && source_row(p, j, end) < 0) y = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) { y[i] += bias[i]; if (p.relu) y[i] = y[i] < 0.f ? 0.f : y[i]; }          // (NaN stays)
    if (col < p.n) store4<OUT>(p, j, col, y, wide_stores(p, OUT == OUT_F32 ? 16 : 8));
}

namespace {

// a kernel's LDS beyond the default, once for each device
hipError_t allow_lds(const void* kernel, int bytes, std::atomic<unsigned long long>& devices)
{
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (devices.load(std::memory_order_relaxed) & bit) return hipSuccess;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) devices.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

long long row_tiles(const ProductArgs& p, int bm)                             // at most: a group of rows ends inside a tile
{
    return p.offsets ? (long long)p.m / bm + (p.groups < p.m ? p.groups : p.m) : ((long long)p.m + bm - 1) / bm;
}

bool fits(long long workgroups, int threads) { return workgroups * threads < 1ll << 32; }      // (a launch has fewer than 2^32 threads)

template <int IN, int OUT, class T>
hipError_t launch_any(ProductArgs p, hipStream_t st)
{
    p.tiles_n = (p.n + T::BN - 1) / T::BN;
    p.tiles_m = (int)row_tiles(p, T::BM);
    const long long grid = (row_tiles(p, T::BM) * p.tiles_n + 7) / 8 * 8;
    if (!fits(grid, T::THREADS)) return hipErrorInvalidConfiguration;
    static std::atomic<unsigned long long> devices{0};
    const hipError_t e = allow_lds(reinterpret_cast<const void*>(product_any_kernel<IN, OUT, T>), T::LDS, devices);
    if (e != hipSuccess) return e;
    product_any_kernel<IN, OUT, T><<<(unsigned)grid, T::THREADS, T::LDS, st>>>(p);
    return hipGetLastError();
}

template <int IN, int OUT, class T>
hipError_t launch_ring(ProductArgs p, hipStream_t st)
{
    p.tiles_n = (p.n + T::BN - 1) / T::BN;
    p.tiles_m = (int)row_tiles(p, T::BM);
    const long long tiles = row_tiles(p, T::BM) * p.tiles_n, grid = (tiles + 7) / 8 * 8;
    if (!fits(grid, T::THREADS)) return hipErrorInvalidConfiguration;
    static std::atomic<unsigned long long> devices{0};
    const hipError_t e = allow_lds(reinterpret_cast<const void*>(product_ring_kernel<IN, OUT, T>), T::LDS, devices);
    if (e != hipSuccess) return e;
    product_ring_kernel<IN, OUT, T><<<(unsigned)grid, T::THREADS, T::LDS, st>>>(p);
    return hipGetLastError();
}

template <int IN, int OUT, class T>
hipError_t launch_phased(ProductArgs p, hipStream_t st)
{
    p.tiles_n = (p.n + T::BN - 1) / T::BN;
    p.tiles_m = (int)row_tiles(p, T::BM);
    const long long tiles = row_tiles(p, T::BM) * p.tiles_n, grid = (tiles + 7) / 8 * 8;
    if (!fits(grid, T::THREADS)) return hipErrorInvalidConfiguration;
    static std::atomic<unsigned long long> devices{0};
    const hipError_t e = allow_lds(reinterpret_cast<const void*>(product_phased_kernel<IN, OUT, T>), T::LDS, devices);
    if (e != hipSuccess) return e;
    product_phased_kernel<IN, OUT, T><<<(unsigned)grid, T::THREADS, T::LDS, st>>>(p);
    return hipGetLastError();
}

template <int IN, int OUT, int MT, int U>
hipError_t launch_rows(ProductArgs p, hipStream_t st)
{
    p.tiles_n = (p.n + 15) / 16;
    p.tiles_m = (int)row_tiles(p, MT * 16);
    const long long grid = (row_tiles(p, MT * 16) * p.tiles_n + 7) / 8 * 8;
    if (!fits(grid, 1024)) return hipErrorInvalidConfiguration;
    product_rows_kernel<IN, OUT, MT, U><<<(unsigned)grid, 1024, 0, st>>>(p);
    return hipGetLastError();
}

// Which kernel: the one with the least estimated time, 2 us + rounds of 256 tiles x (a tile's beginning and end + its steps).  The microseconds below are
// fitted to runs on 1 .. 32768 rows of 2048 x 4736 and 512 x 2048 and to grouped ones (a graph of 20 calls each; us):
//
//   rows   e4m3 to bf16:   16 / 32 at a time   32 x 128   64 x 128   128 x 128   128 x 256   192 x 256   256 x 256
//        1                       5.8 /  6.4       14.1       16.5
//       32                       7.5 /  9.4       14.4       16.8
//      128                      23.3 / 17.7       15.2       17.0
//     1024                                        29.6       19.3        24.8        30.6        47.6        54.4
//     2048                                        55.1       35.1        26.6        31.1        48.1        55.0
//     4096                                                               53.1        39.2        50.4        56.5
//     5000                                                               72.5        63.6        51.5        56.6
//     8192                                                               98.5        76.0        99.8        65.3
//    32768                                       833        527         387         297         299         257
//
// Operands at any address (1001 x 1419; 2048 x 4729), 32 x 128 tiles | 128 x 128:  733 rows 10.6 | 16.8, 3000 31.3 | 18.3, 20000 189 | 92; 4096 212 | 98.
//
// Folded block sums (fp32 scales) take 1.02 .. 1.2 times as long (32768 rows 311), 16-bit operands from e4m3 (fp32 results) 1.35 times in the rings and
// 1.4 .. 2 in the large tiles (2048 rows 48.7, 32768 527 with e8m0 scales and 569 with fp32 ones), bf16 operands over the same K twice, since a step of
// K is 64 of theirs (4096 rows 74.8 in 128 x 256 tiles, 32768 484 in 256 x 256).  A K that ends inside a step costs up to 5 %.
template <int IN, int OUT>
hipError_t launch_out(const ProductArgs& p, hipStream_t st)
{
    constexpr bool EXACT = OUT == OUT_F32;
    constexpr int F = IN != IN_BF16 && EXACT ? 2 : FOLDS<IN, EXACT> ? 1 : 0;                 // scales for the matrix instruction (or none) | block sums folded | e4m3 as fp16
    if (p.kbytes == 0 || p.a_rows == 0) return launch_any<IN, OUT, Any<1, 4, 2, 2, 2>>(p, st);
    const bool aligned = ((reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b) | (uintptr_t)p.a_row | (uintptr_t)p.b_row | (uintptr_t)p.b_group | (uintptr_t)p.kbytes) & 15) == 0;
    const bool near = p.sb_row < (1ll << 29) && p.a_rows * p.a_row < (1ll << 32) && p.n * p.b_row < (1ll << 32);      // the ring's and the phased kernel's 32-bit offsets
    const bool dma = aligned && near;
    const double steps = (p.kbytes + KROW - 1) / KROW;
    enum { ROWS16, ROWS32, ANY, ANY128, R32, R64, P128N, P128, P192, P256 };
    int best = -1;
    double least = 0;
    auto offer = [&](int kernel, bool can, int bm, int bn, double edge, double step) {
        if (!can || !fits((row_tiles(p, bm) * ((p.n + bn - 1) / bn) + 7) / 8 * 8, bn == 16 ? 1024 : 512)) return;
        const double rows = p.groups > 1 ? (double)p.m / bm + 0.5 * (p.groups < p.m ? p.groups : p.m) : (double)((p.m + bm - 1) / bm);   // (a group's last tile is half full)
        const double us = 2 + ceil(rows * ((p.n + bn - 1) / bn) / 256) * (edge + steps * step);
        if (best < 0 || us < least) { best = kernel; least = us; }
    };
    offer(ROWS16, OUT != OUT_E4M3, 16, 16, 1.5, aligned ? 0.13 : 0.2);
    offer(ROWS32, OUT != OUT_E4M3, 32, 16, 1.5, aligned ? 0.17 : 0.25);
    offer(ANY, !dma, 32, 128, 2, F ? 0.6 : 0.5);                              // (several at once on a CU)
    offer(ANY128, !dma, 128, 128, 3, F ? 1.65 : 1.2);
    offer(R32, dma, 32, 128, 2, F == 0 ? 0.34 : F == 1 ? 0.36 : 0.50);
    offer(R64, dma, 64, 128, 2, F == 0 ? 0.42 : F == 1 ? 0.45 : 0.69);
    offer(P128N, dma, 128, 128, 3, F == 0 ? 0.68 : F == 1 ? 0.69 : 1.06);
    offer(P128, dma, 128, 256, 4, F == 0 ? 1.03 : F == 1 ? 1.13 : 1.75);
    offer(P192, dma && F < 2, 192, 256, 4, F == 0 ? 1.30 : 1.44);             // (16-bit operands do not fit its registers)
    offer(P256, dma && (F == 0 || (F == 1 && p.kbytes % KROW == 0)), 256, 256, 5, F == 0 ? 1.60 : 1.90);
    if (best < 0) return hipErrorInvalidConfiguration;
    if constexpr (OUT != OUT_E4M3) {
        if (best == ROWS16) return launch_rows<IN, OUT, 1, 3>(p, st);
        if (best == ROWS32) return launch_rows<IN, OUT, 2, 2>(p, st);
    }
    if constexpr (F < 2) {
        if (best == P192) return launch_phased<IN, OUT, Phased<2, 4, 6, 4, 2>>(p, st);
        if (best == P256) return launch_phased<IN, OUT, Phased<2, 4, 8, 4, 2>>(p, st);
    }
    switch (best) {
    case R32: return launch_ring<IN, OUT, Ring<1, 4, 2, 2, 3, 2>>(p, st);
    case R64: return launch_ring<IN, OUT, Ring<2, 2, 2, 4, 3, 2>>(p, st);
    case P128N: return launch_phased<IN, OUT, Phased<2, 4, 4, 2, 3>>(p, st);
    case P128: return launch_phased<IN, OUT, Phased<2, 4, 4, 4, 3>>(p, st);
    case ANY128: return launch_any<IN, OUT, Any<2, 4, 4, 2, 1>>(p, st);
    default: return launch_any<IN, OUT, Any<1, 4, 2, 2, 2>>(p, st);
    }
}

template <int IN>
hipError_t launch_in(const ProductArgs& p, int out, hipStream_t st)
{
    if (out == OUT_F32) return launch_out<IN, OUT_F32>(p, st);
    if (out == OUT_BF16) return launch_out<IN, OUT_BF16>(p, st);
    if constexpr (IN != IN_BF16) return launch_out<IN, OUT_E4M3>(p, st);
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_product(const ProductArgs& p, int in, int out, hipStream_t st)
{
    if (in == IN_BF16) return launch_in<IN_BF16>(p, out, st);
    if (in == IN_F8_F32) return launch_in<IN_F8_F32>(p, out, st);
    return launch_in<IN_F8_E8>(p, out, st);
}

}  // namespace dce
