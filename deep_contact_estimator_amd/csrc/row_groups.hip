// row_groups.hip -- rows in the order of their group (a stable counting sort of group numbers), and what a row of logits says.
//
//   offsets[g]  the first place of group g;  offsets[groups] the number of rows that have a group
//   order[j]    the row at place j (rows of one group in their own order; -1 behind the last group)
//   place[i]    the place of row i, -1 for a row whose number is outside [0, groups)
//
// A chunk of rows belongs to one workgroup, an eighth of it to each of its waves.  A wave takes 64 rows at a time: the lanes with an equal number are
// found with one ballot for each bit of the number, a row's rank among them is a count of bits, and the running count of every group lives in LDS.
// No atomics on results: places do not depend on the order in which workgroups run.  Bound: latency (the ids are 4 bytes a row): 30 rows 2.8 us, 200000 of
// 64 groups 8.8 us, of 1024 groups 26 us (there every workgroup reads the counts of all chunks, 4 KB each).
#include "block_ops.h"

namespace dce {

namespace {

constexpr int GW = 8;                         // waves a workgroup
constexpr int CHUNKS_MAX = 256;

// Rows of a chunk: a workgroup reads every chunk's counts, so no more chunks than a card has workgroups at once, and none whose counts outnumber half its
// rows.  us at 4000 x 64 groups | 200000 x 64 | 200000 x 1024 (a graph of 20 calls): chunks of 512 rows 5.8 | 8.8 | 34.0, of 2048 8.2 | 10.6 | 26.2.
int chunk_rows(int n, int groups)
{
    const int per = (n + CHUNKS_MAX - 1) / CHUNKS_MAX, c = per > 2 * groups ? per : 2 * groups;
    return (c + GW * 64 - 1) / (GW * 64) * (GW * 64);
}

template <typename ID>
__device__ __forceinline__ int key_of(const ID* ids, int i, int groups)
{
    const ID v = ids[i];
    return v >= 0 && v < (ID)groups ? (int)v : -1;
}

// the lanes whose key equals this lane's (lanes without a key: none that counts)
__device__ __forceinline__ unsigned long long same_key(int key, int bits)
{
    unsigned long long m = __ballot(key >= 0);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((key >> b) & 1);
        m &= ((key >> b) & 1) ? set : ~set;
    }
    return m;
}

}  // namespace

// counts of every chunk: work[chunk][group]
template <typename ID>
__global__ __launch_bounds__(GW * 64) void group_count_kernel(const ID* __restrict__ ids, int n, int groups, int chunk, int* __restrict__ work)
{
    __shared__ int hist[GROUPS_MAX];
    for (int g = threadIdx.x; g < groups; g += GW * 64) hist[g] = 0;
    __syncthreads();
    const long long lo = (long long)blockIdx.x * chunk;
    const int hi = lo + chunk < n ? (int)(lo + chunk) : n;
    for (int i = (int)lo + threadIdx.x; i < hi; i += GW * 64) { const int k = key_of(ids, i, groups); if (k >= 0) atomicAdd(&hist[k], 1); }
    __syncthreads();
    for (int g = threadIdx.x; g < groups; g += GW * 64) work[(long long)blockIdx.x * groups + g] = hist[g];
}

template <typename ID>
__global__ __launch_bounds__(GW * 64) void group_place_kernel(const ID* __restrict__ ids, int n, int groups, int bits, int chunk, const int* __restrict__ work,
                                                              int* __restrict__ offsets, int* __restrict__ order, int* __restrict__ place)
{
    __shared__ int run[GW][GROUPS_MAX];       // a wave's next place in every group
    __shared__ int base[GROUPS_MAX], before[GROUPS_MAX];   // rows of every group, then its first place; its rows in front of this chunk
    __shared__ int total;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, chunks = gridDim.x, me = blockIdx.x;
    const long long lo = (long long)me * chunk;
    const int hi = lo + chunk < n ? (int)(lo + chunk) : n;
    const int part = chunk / GW;
    const long long wl = lo + (long long)wave * part;
    const int wlo = wl < hi ? (int)wl : hi, whi = wl + part < hi ? (int)(wl + part) : hi;

    for (int g = lane; g < groups; g += 64) run[wave][g] = 0;
    for (int g = threadIdx.x; g < groups; g += GW * 64) base[g] = before[g] = 0;
    __syncthreads();
    for (int i = wlo + lane; i < whi; i += 64) { const int k = key_of(ids, i, groups); if (k >= 0) atomicAdd(&run[wave][k], 1); }
    // rows of every group in all chunks, and in the chunks before this one (sums of whole numbers: any order)
    if (chunks > 1) {
        const int wide = 1 << bits < GW * 64 ? 1 << bits : GW * 64, per = GW * 64 / wide;   // threads along the groups, along the chunks
        for (int g = threadIdx.x % wide; g < groups; g += wide) {
            int all = 0, first = 0;
#pragma unroll 8
            for (int c = threadIdx.x / wide; c < chunks; c += per) { const int v = work[(long long)c * groups + g]; all += v; first += c < me ? v : 0; }
            atomicAdd(&base[g], all);
            atomicAdd(&before[g], first);
        }
    }
    __syncthreads();
    for (int g = threadIdx.x; g < groups; g += GW * 64) {
        int at = before[g];
        for (int w = 0; w < GW; ++w) { const int v = run[w][g]; run[w][g] = at; at += v; }
        if (chunks == 1) base[g] = at;
    }
    __syncthreads();
    if (wave == 0) {                          // the groups' first places: a scan over 64 groups a step
        int carry = 0;
        for (int g0 = 0; g0 < groups; g0 += 64) {
            const int own = g0 + lane < groups ? base[g0 + lane] : 0;
            int sum = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(sum, d); if (lane >= d) sum += o; }
            if (g0 + lane < groups) {
                base[g0 + lane] = carry + sum - own;
                if (me == 0) offsets[g0 + lane] = carry + sum - own;
            }
            carry += __builtin_amdgcn_readlane(sum, 63);
        }
        if (lane == 0) { total = carry; if (me == 0) offsets[groups] = carry; }
    }
    __syncthreads();
    const unsigned long long below = (1ull << lane) - 1;
    for (int i0 = wlo; i0 < whi; i0 += 64) {
        const int i = i0 + lane;
        const int k = i < whi ? key_of(ids, i, groups) : -1;
        const unsigned long long same = same_key(k, bits);
        int at = -1;
        if (k >= 0) at = base[k] + run[wave][k] + __popcll(same & below);
        __builtin_amdgcn_wave_barrier();
        if (k >= 0 && (same & below) == 0) run[wave][k] += __popcll(same);      // the first of the equal ones counts them all
        __builtin_amdgcn_wave_barrier();
        if (i < whi) { place[i] = at; if (at >= 0) order[at] = i; }
    }
    for (int j = (int)lo + threadIdx.x; j < hi; j += GW * 64) if (j >= total) order[j] = -1;
}

long long group_rows_work(long long n, int groups)
{
    const int c = chunk_rows((int)n, groups);
    const long long chunks = (n + c - 1) / c;
    return chunks > 1 ? chunks * groups : 0;
}

namespace {
template <typename ID>
void launch_groups(const ID* ids, int n, int groups, int* offsets, int* order, int* place, int* work, hipStream_t st)
{
    const int chunk = chunk_rows(n, groups);
    const int chunks = n ? (int)(((long long)n + chunk - 1) / chunk) : 1;
    int bits = 0;
    while ((1 << bits) < groups) ++bits;
    if (chunks > 1) group_count_kernel<ID><<<chunks, GW * 64, 0, st>>>(ids, n, groups, chunk, work);
    group_place_kernel<ID><<<chunks, GW * 64, 0, st>>>(ids, n, groups, bits, chunk, work, offsets, order, place);
}
}  // namespace

hipError_t launch_group_rows(const void* ids, int id_bytes, int n, int groups, int* offsets, int* order, int* place, int* work, hipStream_t st)
{
    if (id_bytes == 8) launch_groups(static_cast<const long long*>(ids), n, groups, offsets, order, place, work, st);
    else launch_groups(static_cast<const int*>(ids), n, groups, offsets, order, place, work, st);
    return hipGetLastError();
}

// ---- logits -> class and contact bits, the row of logits picked by `index` (first of equal ones; a NaN is the largest, the first NaN wins; an index
//      outside the rows: NaN logits, class 0).  Sixteen lanes a row.  4096 rows 2.8 us; 200000 in another order (28 MB) 15.3.
__global__ __launch_bounds__(256) void decide_kernel(const float* __restrict__ logits, long long n, long long rows, const int* __restrict__ index,
                                                     float* __restrict__ out, int* __restrict__ pred, unsigned char* __restrict__ contacts)
{
    const int c = threadIdx.x & 15;
    for (long long i = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); i < n; i += (long long)gridDim.x * 16) {
        const long long s = index ? (long long)index[i] : i;
        const float v = s >= 0 && s < rows ? logits[s * 16 + c] : __builtin_nanf("");
        if (out) out[i * 16 + c] = v;
        float best = v; int at = c;
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            const float o = __shfl_xor(best, d); const int oc = __shfl_xor(at, d);
            const bool on = o != o, bn = best != best;
            const bool take = on ? (!bn || oc < at) : (!bn && (o > best || (o == best && oc < at)));
            if (take) { best = o; at = oc; }
        }
        if (c == 0) {
            if (pred) pred[i] = at;
            if (contacts) for (int b = 0; b < 4; ++b) contacts[i * 4 + b] = (unsigned char)((at >> (3 - b)) & 1);
        }
    }
}

hipError_t launch_decide(const float* logits, long long n, long long rows, const int* index, float* out, int* pred, unsigned char* contacts, hipStream_t st)
{
    const long long wgs = (n + 15) / 16, most = 1 << 20;                      // (a launch has fewer than 2^32 threads; up to 16 million rows each workgroup takes its sixteen)
    decide_kernel<<<(unsigned)(wgs < most ? wgs : most), 256, 0, st>>>(logits, n, rows, index, out, pred, contacts);
    return hipGetLastError();
}

}  // namespace dce
