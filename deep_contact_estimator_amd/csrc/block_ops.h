// block_ops.h -- the matrix products of the FC layers as operators of their own (include/dce.h: dce_quantize, dce_matmul, dce_group_rows, dce_decide):
// arguments of the kernels and the device helpers they share.  Internal to libdce.so.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace dce {

constexpr int BLK = 128;                      // columns (and, of weights, rows) that share a scale
constexpr int GROUPS_MAX = 1024;
constexpr int KROW = 128;                     // bytes of a row that one step along K takes: 128 e4m3 or 64 bf16 values

enum { IN_BF16 = 0, IN_F8_F32 = 1, IN_F8_E8 = 2 };     // operands: bf16 | e4m3 with fp32 scales | e4m3 with e8m0 scales
enum { OUT_F32 = 0, OUT_BF16 = 1, OUT_E4M3 = 2 };

// y[j,:] = act( a[src(j),:] W[g]^T + bias[g] ) for the rows j of group g; without offsets there is one group, without an index src(j) = j
struct ProductArgs {
    const char* a; long long a_row;           // bytes from row to row
    const char* b; long long b_row, b_group;  // (groups, n, k)
    const void* sa; long long sa_block;       // scale of row i and block t: sa[t * sa_block + i]
    const void* sb; long long sb_row, sb_group;        // scale of columns 128 u .. and block t: sb[g * sb_group + u * sb_row + t]
    const float* bias; long long bias_group;
    char* y; long long y_row;                 // bytes from row to row
    void* ys; long long ys_block;             // OUT_E4M3: scale of row j and columns 128 u ..: ys[u * ys_block + j]
    const int* offsets; const int* index;
    long long a_rows;                         // rows of a: an index outside reads as a row of zeros
    int m, n, kbytes, groups, relu;
    int tiles_n, tiles_m;                     // column tiles; row tiles, at most
};

struct QuantArgs {
    const char* x; long long x_row, x_batch;  // bytes
    unsigned char* q; long long q_row, q_batch;
    void* s; long long s_block;               // 1 x 128 blocks: s[t * s_block + row]; 128 x 128: s[(batch * row blocks + row block) * s_block + t]
    long long rows; int k, kblocks; long long units;
};

hipError_t launch_product(const ProductArgs& p, int in, int out, hipStream_t st);
hipError_t launch_quantize(const QuantArgs& p, int x_bf16, int batch, int block_rows, int e8m0, hipStream_t st);
long long group_rows_work(long long n, int groups);
hipError_t launch_group_rows(const void* ids, int id_bytes, int n, int groups, int* offsets, int* order, int* place, int* work, hipStream_t st);
hipError_t launch_decide(const float* logits, long long n, long long rows, const int* index, float* out, int* pred, unsigned char* contacts, hipStream_t st);

#ifdef __HIPCC__
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// 16 bytes from any address (global memory serves unaligned 16-byte loads)
__device__ __forceinline__ i32x4 load16(const char* p) { i32x4 v; __builtin_memcpy(&v, p, 16); return v; }
// Bytes of a row at any address from whole words: those that hold them, and no word that holds none of the row's.  `row` & 3 is the shift.
__device__ __forceinline__ const char* word_of(const char* row) { return row - (reinterpret_cast<uintptr_t>(row) & 3); }
__device__ __forceinline__ int last_word(const char* row, int end) { return (end - 1 + (int)(reinterpret_cast<uintptr_t>(row) & 3)) & ~3; }
__device__ __forceinline__ int word_at(const char* words, int at) { return *reinterpret_cast<const int*>(words + at); }
// words w[0 .. 4] -> sixteen bytes; what lies at `left` or behind it reads as zero
__device__ __forceinline__ i32x4 shift_words(i32x4 w, int next, unsigned by)
{
    return i32x4{(int)__builtin_amdgcn_alignbyte(w[1], w[0], by), (int)__builtin_amdgcn_alignbyte(w[2], w[1], by), (int)__builtin_amdgcn_alignbyte(w[3], w[2], by),
                 (int)__builtin_amdgcn_alignbyte(next, w[3], by)};
}
__device__ __forceinline__ i32x4 cut_bytes(i32x4 v, int left)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = left - 4 * i;
        v[i] = n >= 4 ? v[i] : n <= 0 ? 0 : v[i] & ((1 << 8 * n) - 1);
    }
    return v;
}
// bytes [at, at + 16) of a row that ends at byte `end` > 0: what lies behind it reads as zero
__device__ __forceinline__ i32x4 load16_tail(const char* row, int at, int end)
{
    const char* const words = word_of(row);
    const int last = last_word(row, end);
    i32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = word_at(words, at + 4 * i < last ? at + 4 * i : last);
    return cut_bytes(shift_words(w, word_at(words, at + 16 < last ? at + 16 : last), (unsigned)reinterpret_cast<uintptr_t>(row) & 3), end - at);
}

// The scale of a block whose largest finite magnitude is `most`: the smallest e with most <= 448 * 2^e.  most = f * 2^p with f in [0.5, 1) and
// 448 = 0.875 * 2^9, so e is p - 9, or p - 8 for f above 0.875.  Held inside [-126, 120]: 2^e and 2^-e are normal fp32 numbers.
__device__ __forceinline__ int block_exponent(float most)
{
    const unsigned u = __float_as_uint(most);
    const int p = (int)(u >> 23) - 126;                       // (a subnormal `most` is clamped either way)
    const int e = p - 9 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e > 120 ? 120 : e;
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
__device__ __forceinline__ float finite_abs(float v) { const float a = fabsf(v); return a < __builtin_inff() ? a : 0.f; }      // (NaN and infinities do not set a scale)

// four values (already times 2^-e: at most 448 in magnitude) -> e4m3, round to nearest even: the instruction's own rounding.  e4m3 has no infinity:
// one becomes NaN, as a NaN does.
__device__ __forceinline__ float or_nan(float v) { return fabsf(v) < __builtin_inff() ? v : __builtin_nanf(""); }
__device__ __forceinline__ int to_e4m3x4(float a, float b, float c, float d)
{
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(or_nan(a), or_nan(b), 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(or_nan(c), or_nan(d), r, true);
}
#endif

}  // namespace dce
