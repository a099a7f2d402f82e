// block_quant.hip -- x (fp32 | bf16) -> e4m3 with a power of two for every block of 1 x 128 values (activations) or 128 x 128 (weights).
//
//   e = min{ e : max|x| <= 448 * 2^e },  q = round(x * 2^-e) to e4m3, ties to even
//
// A power of two costs a floating-point format nothing: x * 2^-e is exact, so q carries the ONE rounding to 4 significant bits, and the matrix pipe
// can apply the exponents itself.  NaN and infinities become NaN and do not set the scale.
// Bound: memory, one read of x and one write of q: 32768 x 4736 bf16 83 us, 5.6 TB/s; one row 2.5 us, the launch; weights, 2048 x 4736
// fp32, 10.4 us, 4.7 TB/s (592 workgroups, each one block: a read, a barrier and a write).
#include "block_ops.h"

namespace dce {

template <int BF16>
__device__ __forceinline__ void load8(const char* row, int at, int k, float (&v)[8])
{
    if (at + 8 <= k) {
        if (BF16) {
            const i32x4 r = load16(row + 2ll * at);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float((unsigned)r[i] << 16); v[2 * i + 1] = __uint_as_float((unsigned)r[i] & 0xffff0000u); }
        } else {
            const i32x4 r0 = load16(row + 4ll * at), r1 = load16(row + 4ll * at + 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = __int_as_float(r0[i]); v[4 + i] = __int_as_float(r1[i]); }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (at + i >= k) v[i] = 0.f;
        else if (BF16) { unsigned short h; __builtin_memcpy(&h, row + 2ll * (at + i), 2); v[i] = __uint_as_float((unsigned)h << 16); }
        else __builtin_memcpy(&v[i], row + 4ll * (at + i), 4);
    }
}

__device__ __forceinline__ void store8(unsigned char* row, int at, int k, const float (&v)[8], float inv)
{
    int w[2];
    w[0] = to_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    w[1] = to_e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    if (at + 8 <= k) { __builtin_memcpy(row + at, w, 8); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i) if (at + i < k) row[at + i] = (unsigned char)(w[i >> 2] >> (8 * (i & 3)));
}

template <int E8>
__device__ __forceinline__ void store_scale(void* s, long long at, int e)
{
    if (E8) static_cast<unsigned char*>(s)[at] = (unsigned char)(e + 127);
    else static_cast<float*>(s)[at] = two_to(e);
}

// 1 x 128 blocks: sixteen lanes hold one block, eight values each
template <int BF16, int E8>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs p)
{
    const int lane16 = threadIdx.x & 15;
    for (long long u = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); u < p.units; u += (long long)gridDim.x * 16) {
        const long long row = u / p.kblocks;
        const int t = (int)(u - row * p.kblocks), at = t * BLK + lane16 * 8;
        float v[8], most = 0.f;
        load8<BF16>(p.x + row * p.x_row, at, p.k, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, finite_abs(v[i]));
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
        const int e = block_exponent(most);
        store8(p.q + row * p.q_row, at, p.k, v, two_to(-e));
        if (lane16 == 0) store_scale<E8>(p.s, t * p.s_block + row, e);
    }
}

// 128 x 128 blocks: one workgroup holds a block, 64 values a thread (16 threads a row, 16 rows a pass)
template <int BF16, int E8>
__global__ __launch_bounds__(256) void quantize_weights_kernel(QuantArgs p)
{
    __shared__ float part[4];
    const int t = blockIdx.x, rb = blockIdx.y, g = blockIdx.z;
    const int at = t * BLK + (threadIdx.x & 15) * 8;
    const long long r0 = (long long)rb * BLK + (threadIdx.x >> 4);
    const char* x = p.x + g * p.x_batch;
    unsigned char* q = p.q + g * p.q_batch;
    float v[8][8], most = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const long long r = r0 + 16 * j;
        if (r < p.rows) load8<BF16>(x + r * p.x_row, at, p.k, v[j]);
        else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, finite_abs(v[j][i]));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
    __syncthreads();
    const int e = block_exponent(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
    const float inv = two_to(-e);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const long long r = r0 + 16 * j;
        if (r < p.rows) store8(q + r * p.q_row, at, p.k, v[j], inv);
    }
    if (threadIdx.x == 0) store_scale<E8>(p.s, ((long long)g * gridDim.y + rb) * p.s_block + t, e);
}

hipError_t launch_quantize(const QuantArgs& p, int x_bf16, int batch, int block_rows, int e8m0, hipStream_t st)
{
    if (block_rows == 1) {
        const long long wgs = (p.units + 15) / 16;
        const dim3 grid((unsigned)(wgs < 256 * 64 ? wgs : 256 * 64));
        if (x_bf16) { if (e8m0) quantize_rows_kernel<1, 1><<<grid, 256, 0, st>>>(p); else quantize_rows_kernel<1, 0><<<grid, 256, 0, st>>>(p); }
        else        { if (e8m0) quantize_rows_kernel<0, 1><<<grid, 256, 0, st>>>(p); else quantize_rows_kernel<0, 0><<<grid, 256, 0, st>>>(p); }
    } else {
        const dim3 grid((unsigned)p.kblocks, (unsigned)((p.rows + BLK - 1) / BLK), (unsigned)batch);
        if (x_bf16) { if (e8m0) quantize_weights_kernel<1, 1><<<grid, 256, 0, st>>>(p); else quantize_weights_kernel<1, 0><<<grid, 256, 0, st>>>(p); }
        else        { if (e8m0) quantize_weights_kernel<0, 1><<<grid, 256, 0, st>>>(p); else quantize_weights_kernel<0, 0><<<grid, 256, 0, st>>>(p); }
    }
    return hipGetLastError();
}

}  // namespace dce
