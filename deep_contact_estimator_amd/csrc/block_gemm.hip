// block_gemm.hip -- the product of the FC layers as an operator: y = act(x W^T + bias) with W chosen by the row's group, operands in bf16 or in
// e4m3 with a scale for every 128 values of a row of x and every 128 x 128 block of W.
//
//   y[j, c] = act( sum_t sa[t, src(j)] sb[g, c / 128, t] sum_{u < 128} a[src(j), 128 t + u] w[g, c, 128 t + u]  +  bias[g, c] )
//
// The inner sums run on the matrix pipe in fp32; fp32 scales multiply a block's sum on the vector pipe (one fma a value), e8m0 scales are operands
// of the 8-bit matrix instruction itself.  One matrix instruction of 16 x 16 x 128 covers a block along K; the bf16 form takes two of 16 x 16 x 32 for the
// same 128 bytes of a row, so one layout in LDS serves both: rows of 128 bytes, eight 16-byte chunks, chunk c of row r in slot c ^ (r & 7) -- the
// eight rows that one access serves lie in eight different slots.
//
// The weights are the instruction's FIRST operand: a lane then holds four neighbouring columns of one row of y (one activation scale a lane, vector
// stores).  Lane l: row l & 15 of either operand, chunks l >> 4 and (l >> 4) + 4.
#include "block_ops.h"

namespace dce {

namespace {

__device__ __forceinline__ int clamp_to(int v, int hi) { return v < 0 ? 0 : v > hi ? hi : v; }

// The group, first row and end of row tile t (tiles of bm rows, counted group by group).  Offsets are held inside [0, m] whatever they say.
// Every wave works it out for itself: 64 groups a step, tiles counted by a scan over the lanes.
__device__ __forceinline__ bool find_tile(const ProductArgs& p, int bm, int t, int& g, int& first, int& end)
{
    if (!p.offsets) { g = 0; first = t * bm; end = p.m; return first < p.m; }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < p.groups; base += 64) {
        int lo = 0, hi = 0;
        if (base + lane < p.groups) { lo = clamp_to(p.offsets[base + lane], p.m); hi = clamp_to(p.offsets[base + lane + 1], p.m); }
        const int tiles = hi > lo ? (hi - lo + bm - 1) / bm : 0;
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(sum, d); if (lane >= d) sum += o; }
        const int total = __builtin_amdgcn_readlane(sum, 63);
        if (t < before + total) {
            const int w = __builtin_ctzll(__ballot(before + sum > t));
            const int at = t - (before + __builtin_amdgcn_readlane(sum, w) - __builtin_amdgcn_readlane(tiles, w));
            g = base + w;
            first = __builtin_amdgcn_readlane(lo, w) + at * bm;
            end = __builtin_amdgcn_readlane(hi, w);
            return true;
        }
        before += total;
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
__device__ __forceinline__ i32x4 chunk(const char* lds, int r, int c) { return *reinterpret_cast<const i32x4*>(lds + r * KROW + ((c ^ (r & 7)) * 16)); }

// 32 e4m3 values -> fp16, without error
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

// One row's 32 values of a step as a lane holds them for the matrix instruction.  EXACT: e4m3 as fp16 (see mac)
template <int IN, bool EXACT> struct Frag {
    i32x4 c0, c1;
    __device__ __forceinline__ void set(i32x4 a, i32x4 b) { c0 = a; c1 = b; }
};
template <int IN> struct Frag<IN, true> {
    f16x8 h[4];
    __device__ __forceinline__ void set(i32x4 a, i32x4 b) { to_f16(a, h[0], h[1]); to_f16(b, h[2], h[3]); }
};
template <> struct Frag<IN_BF16, true> : Frag<IN_BF16, false> {};

// The scales of a step for a lane's row of x and a block of columns.  fp32: their product.  e8m0: the two bytes for the matrix instruction, or (EXACT) the
// sum of the exponents; a byte of 255 is NaN there too.
template <int IN, bool EXACT> struct Scale {
    float s, start; int ew, ex;
    __device__ __forceinline__ void set_f32(float w, float x) { s = w * x; }
    __device__ __forceinline__ void set_e8(int w, int x)
    {
        if (EXACT) { ew = w + x - 254; start = w == 255 || x == 255 ? __builtin_nanf("") : 0.f; }
        else { ew = w; ex = x; }
    }
};

// acc += the product of a block of 16 x 16 over one step of K.
//
// The 8-bit matrix instruction lines the eight products of a group up with the largest of them and keeps 13 bits below its leading one (measured: of
// 65536 + 8 everything, of 65536 + 4 nothing is left of the second; between groups sums are fp32): on random operands 1.5e-5 of the result, a hundredth
// of the rounding to bf16 (1.7e-3) and less still of that to e4m3, so results in those types take it.  fp32 results would be a hundred times worse
// than their type: they take the operands as fp16 (every e4m3 number is one) through the fp16 instruction, at half the rate, whose sums of 32 products
// are good to 1e-8.
template <int IN, bool EXACT>
__device__ __forceinline__ void mac(f32x4& acc, const Frag<IN, EXACT>& w, const Frag<IN, EXACT>& x, const Scale<IN, EXACT>& sc)
{
    if constexpr (IN == IN_BF16) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w.c0), __builtin_bit_cast(bf16x8, x.c0), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w.c1), __builtin_bit_cast(bf16x8, x.c1), acc, 0, 0, 0);
    } else if constexpr (EXACT) {
        const float z = IN == IN_F8_E8 ? sc.start : 0.f;
        f32x4 part = {z, z, z, z};
#pragma unroll
        for (int i = 0; i < 4; ++i) part = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.h[i], x.h[i], part, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = IN == IN_F8_E8 ? acc[i] + ldexpf(part[i], sc.ew) : fmaf(part[i], sc.s, acc[i]);
    } else {
        const i32x8 wv = __builtin_shufflevector(w.c0, w.c1, 0, 1, 2, 3, 4, 5, 6, 7), xv = __builtin_shufflevector(x.c0, x.c1, 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (IN == IN_F8_E8) acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, acc, 0, 0, 0, sc.ew, 0, sc.ex);
        else {
            const f32x4 part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 127, 0, 127);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(part[i], sc.s, acc[i]);
        }
    }
}

__device__ __forceinline__ unsigned short to_bf16(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }

__device__ __forceinline__ f32x4 finish(const ProductArgs& p, f32x4 v, const float* bias, int c)
{
    if (bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (c + i < p.n) v[i] += bias[c + i];
    }
    if (p.relu) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];          // (NaN stays)
    }
    return v;
}

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

// ---- the kernel for every case: 64 rows x 128 columns a workgroup, sixteen rows a wave; operands through registers into LDS, from any alignment
template <int IN, int OUT>
__global__ __launch_bounds__(256) void product_any_kernel(ProductArgs p)
{
    constexpr int BM = 64, BN = 128, CH = (BM + BN) * 8 / 256;               // 16-byte chunks a thread brings each step
    constexpr bool EXACT = OUT == OUT_F32;
    __shared__ __attribute__((aligned(16))) char lds[(BM + BN) * KROW];
    int g, first, end;
    const int tn = (int)(blockIdx.x % (unsigned)p.tiles_n);
    if (!find_tile(p, BM, (int)(blockIdx.x / (unsigned)p.tiles_n), g, first, end)) return;
    const int n0 = tn * BN, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int steps = (p.kbytes + KROW - 1) / KROW;

    const char* row[CH];                                                      // null: a row of zeros
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int lr = (int)(threadIdx.x >> 3) + 32 * i;
        row[i] = nullptr;
        if (lr < BM) { const long long s = source_row(p, first + lr, end); if (s >= 0) row[i] = p.a + s * p.a_row; }
        else if (n0 + lr - BM < p.n) row[i] = p.b + g * p.b_group + (long long)(n0 + lr - BM) * p.b_row;
    }
    const int c8 = threadIdx.x & 7;
    auto fetch = [&](int s, i32x4 (&v)[CH]) {
#pragma unroll
        for (int i = 0; i < CH; ++i) v[i] = row[i] ? load16_tail(row[i], s * KROW + c8 * 16, p.kbytes) : i32x4{0, 0, 0, 0};
    };
    const long long mine = source_row(p, first + wave * 16 + r, end);         // the row whose scales this lane applies
    const long long sb0 = g * p.sb_group + (long long)tn * p.sb_row;

    f32x4 acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    i32x4 next[CH];
    if (steps) fetch(0, next);
    for (int s = 0; s < steps; ++s) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int lr = (int)(threadIdx.x >> 3) + 32 * i;
            *reinterpret_cast<i32x4*>(lds + lr * KROW + ((c8 ^ (lr & 7)) * 16)) = next[i];
        }
        __syncthreads();
        Scale<IN, EXACT> sc;
        if constexpr (IN == IN_F8_F32) sc.set_f32(static_cast<const float*>(p.sb)[sb0 + s], mine >= 0 ? static_cast<const float*>(p.sa)[s * p.sa_block + mine] : 1.f);
        if constexpr (IN == IN_F8_E8) sc.set_e8(static_cast<const unsigned char*>(p.sb)[sb0 + s], mine >= 0 ? static_cast<const unsigned char*>(p.sa)[s * p.sa_block + mine] : 127);
        if (s + 1 < steps) fetch(s + 1, next);
        const int xr = wave * 16 + r;
        Frag<IN, EXACT> x, w;
        x.set(chunk(lds, xr, q), chunk(lds, xr, q + 4));
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
            const int wr = BM + nt * 16 + r;
            w.set(chunk(lds, wr, q), chunk(lds, wr, q + 4));
            mac<IN, EXACT>(acc[nt], w, x, sc);
        }
    }
    const int j = first + wave * 16 + r;
    const float* bias = p.bias ? p.bias + g * p.bias_group : nullptr;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) acc[nt] = finish(p, acc[nt], bias, n0 + nt * 16 + q * 4);
    float inv = 1.f;
    if constexpr (OUT == OUT_E4M3) {
        float most = 0.f;                                                     // (columns from n on hold bias-free zeros of zero rows)
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, finite_abs(acc[nt][i]));
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        const int e = block_exponent(most);
        inv = two_to(-e);
        if (q == 0 && j < end) {
            if (IN == IN_F8_E8) static_cast<unsigned char*>(p.ys)[tn * p.ys_block + j] = (unsigned char)(e + 127);
            else static_cast<float*>(p.ys)[tn * p.ys_block + j] = two_to(e);
        }
    }
    if (j >= end) return;
    const bool wide = wide_stores(p, OUT == OUT_F32 ? 16 : OUT == OUT_BF16 ? 8 : 4);
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
        const int c = n0 + nt * 16 + q * 4;
        if (c < p.n) store4<OUT>(p, j, c, acc[nt] * inv, wide);
    }
}

namespace {
template <int IN>
hipError_t launch_any(ProductArgs p, int out, hipStream_t st)
{
    p.tiles_n = (p.n + 127) / 128;
    const long long tiles_m = p.offsets ? (long long)p.m / 64 + (p.groups < p.m ? p.groups : p.m) : ((long long)p.m + 63) / 64;
    if (tiles_m * p.tiles_n > 0x7fffffffll) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)(tiles_m * p.tiles_n));
    if (out == OUT_F32) product_any_kernel<IN, OUT_F32><<<grid, 256, 0, st>>>(p);
    else if (out == OUT_BF16) product_any_kernel<IN, OUT_BF16><<<grid, 256, 0, st>>>(p);
    else if constexpr (IN != IN_BF16) product_any_kernel<IN, OUT_E4M3><<<grid, 256, 0, st>>>(p);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}
}  // namespace

hipError_t launch_product(const ProductArgs& p, int in, int out, hipStream_t st)
{
    if (in == IN_BF16) return launch_any<IN_BF16>(p, out, st);
    if (in == IN_F8_F32) return launch_any<IN_F8_F32>(p, out, st);
    return launch_any<IN_F8_E8>(p, out, st);
}

}  // namespace dce
