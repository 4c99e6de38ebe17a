// Tokens sorted by expert and the experts' rows summed back to tokens, each with its gradient, and their C ABI (include/fp6mi.h).  No counterpart in the reference.
//
// A place p = t * k + j is the j-th expert of token t.  Sorting puts the places in order of their experts, ties in their own order, those without an expert (a number outside 0..E-1) last:
//   place[p] = number of places q with (expert(q), q) < (expert(p), p),    order[place[p]] = p,    offsets[e] = number of places of an expert below e
// so place is a permutation, and a place has an expert where place[p] < offsets[E].  Everything here moves rows of H values and is bound by HBM; sums are float32, in the order of j.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "fp6mi_internal.h"

namespace {

#include "fp6mi_grid.inc"

typedef _Float16 half_t;
typedef __bf16   bf16_t;
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kWave = 64, kMostChosen = 64, kMostExperts = 1024;

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Vec { T v[VEC]; };

// Stores past the caches: outputs of many rows are read again when they have long been displaced (the copies of a sort of 4099 tokens x 2 of 8 KB: 28.4 us through the caches, 15.8 past them).
template <typename T, int VEC> __device__ __forceinline__ void store_past(Vec<T, VEC> *to, const Vec<T, VEC> &v)
{
    if constexpr (sizeof(T) * VEC == 16)
        __builtin_nontemporal_store(__builtin_bit_cast(v4u, v), reinterpret_cast<v4u *>(to));
    else if constexpr (sizeof(T) * VEC == 8)
        __builtin_nontemporal_store(__builtin_bit_cast(uint64_t, v), reinterpret_cast<uint64_t *>(to));
    else
        *to = v;
}

__device__ __forceinline__ int wave_sum(int v)
{
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// The expert of a place, E for none.
template <typename I> __device__ __forceinline__ int expert_of(const I *index, size_t p, int E)
{
    const I e = index[p];
    return e >= 0 && e < (I)E ? (int)e : E;
}

// ---------------------------------------------------------------------------------------------------------------
// Sorting
// ---------------------------------------------------------------------------------------------------------------
// offsets[0..E] from counts[0..E-1] in LDS, by the first wavefront; starts[e] likewise (may be counts itself).
__device__ __forceinline__ void scan_counts(const int *counts, int *starts, int *offsets, int E, int lane)
{
    int carry = 0;
    for (int b = 0; b < E; b += kWave) {
        const int n = b + lane < E ? counts[b + lane] : 0;
        int       s = n;
#pragma unroll
        for (int m = 1; m < kWave; m <<= 1) {
            const int o = __shfl_up(s, m);
            if (lane >= m) s += o;
        }
        if (b + lane < E) {
            starts[b + lane] = carry + s - n;
            if (offsets) offsets[b + lane] = carry + s - n;
        }
        carry += __shfl(s, kWave - 1);
    }
    if (lane == 0) {
        starts[E] = carry;
        if (offsets) offsets[E] = carry;
    }
}

// Few places: a workgroup to a token, which finds its places by comparing with all of them, and a last one for the offsets; no workgroup waits for another and there is one launch.
template <typename I, typename V>
__global__ __launch_bounds__(256) void sort_few(const I *__restrict__ index, int *__restrict__ offsets, int *__restrict__ order, int *__restrict__ place, const V *__restrict__ x, V *__restrict__ rows,
                                                size_t ldx, size_t nvec, uint32_t tokens, int k, int E)
{
    __shared__ int shared[kMostExperts + 1 + 4 * 8];
    const int      tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t t = blockIdx.x, P = tokens * k;
    if (t == tokens) {
        for (int e = tid; e < E; e += 256) shared[e] = 0;
        __syncthreads();
        for (uint32_t p = tid; p < P; p += 256)
            if (const int e = expert_of(index, p, E); e < E) atomicAdd(&shared[e], 1); // (whole numbers: the order does not count)
        __syncthreads();
        if (wave == 0) scan_counts(shared, shared, offsets, E, lane);
        return;
    }
    __shared__ int to[kMostChosen];
    V              v[4]; // the row's first pieces, asked for before it is known where they go
#pragma unroll
    for (uint32_t u = 0; u < 4; u++)
        if (rows && tid + 256 * u < nvec) v[u] = x[t * ldx + tid + 256 * u];
    for (int j0 = 0; j0 < k; j0 += 8) {
        const int n = k - j0 < 8 ? k - j0 : 8;
        int       mine[8], below[4] = {}; // (counts of 16 bits, two to a word)
#pragma unroll
        for (int j = 0; j < 8; j++) mine[j] = j < n ? expert_of(index, (size_t)t * k + j0 + j, E) : -1;
        for (uint32_t p = tid; p < P; p += 256) {
            const int e = expert_of(index, p, E);
#pragma unroll
            for (int j = 0; j < 8; j++) below[j / 2] += (e < mine[j] || (e == mine[j] && p < t * k + j0 + j)) << 16 * (j & 1);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (2 * j >= n) break;
            const int s = wave_sum(below[j]);
            if (lane == 0) shared[wave * 8 + 2 * j] = s & 0xffff, shared[wave * 8 + 2 * j + 1] = (uint32_t)s >> 16;
        }
        __syncthreads();
        if (tid < n) {
            const int at = shared[tid] + shared[8 + tid] + shared[16 + tid] + shared[24 + tid];
            bool      none = false;
#pragma unroll
            for (int j = 0; j < 8; j++) none |= tid == j && mine[j] == E;
            to[j0 + tid] = none ? ~at : at;
            place[(size_t)t * k + j0 + tid] = at;
            order[at] = none ? -1 : (int)(t * k + j0 + tid);
        }
        __syncthreads();
    }
    if (!rows) return;
    for (size_t i0 = 0; i0 < nvec; i0 += 1024) {
        for (int j = 0; j < k; j++) {
            const int at = to[j];
            V        *row = rows + (size_t)(at < 0 ? ~at : at) * nvec + i0;
#pragma unroll
            for (uint32_t u = 0; u < 4; u++)
                if (i0 + tid + 256 * u < nvec) row[tid + 256 * u] = at < 0 ? V{} : v[u];
        }
#pragma unroll
        for (uint32_t u = 0; u < 4; u++)
            if (i0 + 1024 + tid + 256 * u < nvec) v[u] = x[t * ldx + i0 + 1024 + tid + 256 * u];
    }
}

// Many places, first launch: how many places of each expert every chunk of tokens holds, table[e][chunk] (rows of `stride` chunks).
template <typename I> __global__ __launch_bounds__(256) void count_chunks(const I *__restrict__ index, uint16_t *__restrict__ table, uint32_t P, uint32_t each, uint32_t stride, int E)
{
    __shared__ int counts[kMostExperts];
    const uint32_t b = blockIdx.x, lo = b * each, hi = lo + each < P ? lo + each : P;
    for (int e = threadIdx.x; e < E; e += 256) counts[e] = 0;
    __syncthreads();
    for (uint32_t p = lo + threadIdx.x; p < hi; p += 256)
        if (const int e = expert_of(index, p, E); e < E) atomicAdd(&counts[e], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += 256) table[(size_t)e * stride + b] = (uint16_t)counts[e];
}

// Second launch: a workgroup to a chunk.  It adds up the table for itself and ranks its places, 512 at a time.
template <typename I>
__global__ __launch_bounds__(512) void place_chunks(const I *__restrict__ index, const uint16_t *__restrict__ table, int *__restrict__ offsets, int *__restrict__ order, int *__restrict__ place,
                                                    uint32_t P, uint32_t each, uint32_t stride, int E)
{
    __shared__ int next[kMostExperts + 1], total[kMostExperts + 1]; // next: where the next place of an expert goes
    __shared__ int counts[8];
    const int      tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t b = blockIdx.x, chunks = gridDim.x, lo = b * each, hi = lo + each < P ? lo + each : P;
    int            e = lo + tid < hi ? expert_of(index, (size_t)lo + tid, E) : -1;
    for (int f = wave; f < E; f += 8) {
        int before = 0, all = 0;
        for (uint32_t c = lane; c < chunks; c += kWave) {
            const int v = table[(size_t)f * stride + c];
            all += v, before += c < b ? v : 0;
        }
        all = wave_sum(all), before = wave_sum(before);
        if (lane == 0) total[f] = all, next[f] = before;
    }
    __syncthreads();
    if (wave == 0) scan_counts(total, total, b == 0 ? offsets : nullptr, E, lane);
    __syncthreads();
    // (those without an expert: behind all others, and of those in the chunks before this one there are as many as have none of the counted ones)
    int counted = 0;
    for (int f = tid; f < E; f += 512) counted += next[f], next[f] += total[f];
    counted = wave_sum(counted);
    if (lane == 0) counts[wave] = counted;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 8; w++) counted += counts[w];
        next[E] = total[E] + (int)lo - counted;
    }
    // Ranks: the lanes of a wavefront that share an expert find each other bit by bit of its number; the wavefronts, one after another, let the first lane of each move the expert's next place on.
    for (uint32_t p0 = lo; p0 < hi; p0 += 512) {
        uint64_t same = __ballot(e >= 0);
        for (int bit = 1; bit <= E; bit <<= 1) {
            const uint64_t set = __ballot(e >= 0 && (e & bit));
            same &= e & bit ? set : ~set;
        }
        const int rank = __builtin_popcountll(same & ((1ull << lane) - 1)), leader = __builtin_ctzll(same | 1ull << 63);
        int       at = 0;
        for (int w = 0; w < 8; w++) {
            __syncthreads();
            if (wave == w && e >= 0 && rank == 0) at = atomicAdd(&next[e], __builtin_popcountll(same));
        }
        at = __shfl(at, leader) + rank;
        if (e >= 0) {
            place[(size_t)p0 + tid] = at;
            order[at] = e == E ? -1 : (int)(p0 + tid);
        }
        e = p0 + 512 + tid < hi ? expert_of(index, (size_t)p0 + 512 + tid, E) : -1;
    }
}

// Third launch: the rows.  A piece of a row is read once and written to its token's places; those without an expert get zeros.
template <typename V>
__global__ __launch_bounds__(256) void copy_tokens(V *__restrict__ rows, const V *__restrict__ x, const int *__restrict__ place, const int *__restrict__ valid_at, size_t ldx, uint32_t nvec,
                                                   uint32_t pieces, uint32_t tokens, int k)
{
    const uint32_t id = workgroup(), t = id / pieces, i = (id - t * pieces) * 512 + threadIdx.x;
    if (t >= tokens) return;
    const int      valid = *valid_at;
    V              v[2];
#pragma unroll
    for (uint32_t u = 0; u < 2; u++)
        if (i + 256 * u < nvec) v[u] = x[t * ldx + i + 256 * u];
    for (int j = 0; j < k; j++) {
        const int at = place[(size_t)t * k + j];
#pragma unroll
        for (uint32_t u = 0; u < 2; u++)
            if (i + 256 * u < nvec) __builtin_nontemporal_store(at < valid ? v[u] : V{}, &rows[(size_t)at * nvec + i + 256 * u]);
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Summing back: out[t] = sum_j w[t,j] * rows[place[t,j]], j of those that have an expert (w = 1 without weights: the gradient of sorting)
// ---------------------------------------------------------------------------------------------------------------
template <typename R, typename O, int VEC>
__global__ __launch_bounds__(256) void combine_rows(O *__restrict__ out, const R *__restrict__ rows, const int *__restrict__ place, const int *__restrict__ valid_at, const float *__restrict__ weights,
                                                    uint32_t nvec, uint32_t pieces, uint32_t tokens, int k)
{
    const uint32_t id = workgroup(), t = id / pieces, i = (id - t * pieces) * 256 + threadIdx.x;
    if (t >= tokens || i >= nvec) return;
    const int valid = *valid_at;
    float     sum[VEC] = {};
    for (int j0 = 0; j0 < k; j0 += 4) { // four rows on their way
        Vec<R, VEC> r[4];
        int         at[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            at[j] = j0 + j < k ? place[(size_t)t * k + j0 + j] : valid;
            if (at[j] < valid) r[j] = reinterpret_cast<const Vec<R, VEC> *>(rows)[(size_t)at[j] * nvec + i];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (at[j] >= valid) continue;
            const float w = weights ? weights[(size_t)t * k + j0 + j] : 1.f;
#pragma unroll
            for (int v = 0; v < VEC; v++) sum[v] += w * (float)r[j].v[v];
        }
    }
    Vec<O, VEC> o;
#pragma unroll
    for (int v = 0; v < VEC; v++) o.v[v] = (O)sum[v];
    store_past(reinterpret_cast<Vec<O, VEC> *>(out) + (size_t)t * nvec + i, o);
}

// Its gradient: grad_rows[place[t,j]] = w[t,j] * grad[t] (zeros where there is no expert), grad_weights[t,j] = <grad[t], rows[place[t,j]]>; either may be left out.  A workgroup to a token
// and four of its experts (64 tokens x 8 of 4096: 10.1 us for all eight one after another, 6.2; 8192 x 8 of 2048 102 and 100).
template <typename R, typename O, int VEC>
__global__ __launch_bounds__(256) void combine_gradient(R *__restrict__ grad_rows, float *__restrict__ grad_weights, const O *__restrict__ grad, const R *__restrict__ rows,
                                                        const int *__restrict__ place, const int *__restrict__ valid_at, const float *__restrict__ weights, uint32_t nvec, uint32_t tokens, int k, uint32_t parts)
{
    constexpr int  J = 4;
    __shared__ float part[4][J];
    const uint32_t id = workgroup(), t = id / parts, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (t >= tokens) return;
    const int      valid = *valid_at, j0 = (int)(id - t * parts) * J;
    const auto    *g_row = reinterpret_cast<const Vec<O, VEC> *>(grad) + (size_t)t * nvec;
    int            at[J];
    float          w[J], dot[J] = {};
#pragma unroll
    for (int j = 0; j < J; j++) {
        at[j] = j0 + j < k ? place[(size_t)t * k + j0 + j] : -1;
        w[j] = j0 + j < k ? (weights ? weights[(size_t)t * k + j0 + j] : 1.f) : 0.f;
    }
    for (uint32_t i = tid; i < nvec; i += 256) {
        const Vec<O, VEC> g = g_row[i];
        Vec<R, VEC>       r[J];
        if (grad_weights) {
#pragma unroll
            for (int j = 0; j < J; j++)
                if (at[j] >= 0 && at[j] < valid) r[j] = reinterpret_cast<const Vec<R, VEC> *>(rows)[(size_t)at[j] * nvec + i];
        }
#pragma unroll
        for (int j = 0; j < J; j++) {
            if (at[j] < 0) continue;
            Vec<R, VEC> d;
#pragma unroll
            for (int v = 0; v < VEC; v++) d.v[v] = at[j] < valid ? (R)(w[j] * (float)g.v[v]) : (R)0.f;
            if (grad_rows) store_past(reinterpret_cast<Vec<R, VEC> *>(grad_rows) + (size_t)at[j] * nvec + i, d);
            if (grad_weights && at[j] < valid) {
#pragma unroll
                for (int v = 0; v < VEC; v++) dot[j] += (float)g.v[v] * (float)r[j].v[v];
            }
        }
    }
    if (!grad_weights) return;
#pragma unroll
    for (int j = 0; j < J; j++) {
        const float s = wave_sum(dot[j]);
        if (lane == 0) part[wave][j] = s;
    }
    __syncthreads();
    if (tid < J && j0 + (int)tid < k) grad_weights[(size_t)t * k + j0 + tid] = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
}

// ---------------------------------------------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------------------------------------------
inline bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline size_t type_size(int dtype) { return dtype == 2 ? 4 : 2; }
inline bool known_type(int dtype) { return dtype >= 0 && dtype <= 2; }

// Up to how many places the sort takes one launch.
constexpr size_t kFewPlaces = 2048;

struct Chunks { uint32_t each, count, stride; }; // places of a chunk; how many chunks; the table's row length
Chunks chunks_of(size_t places)
{
    size_t count = (places + 511) / 512; // (as many as a workgroup ranks at a time; every workgroup reads the whole table)
    count = count > 256 ? 256 : count;
    const size_t each = (places + count - 1) / count < 65535 ? (places + count - 1) / count : 65535; // (counts have 16 bits)
    count = (places + each - 1) / each;
    return { (uint32_t)each, (uint32_t)count, (uint32_t)((count + 7) / 8 * 8) };
}

template <typename F> int by_index(int index64, const F &f) { return index64 ? f(std::integral_constant<bool, true>{}) : f(std::integral_constant<bool, false>{}); }

template <typename I, typename V>
int launch_sort(hipStream_t st, const void *index, int *offsets, int *order, int *place, const void *x, void *rows, size_t ldx, size_t nvec, size_t tokens, size_t k, size_t E, void *ws)
{
    const size_t P = tokens * k;
    if (P <= kFewPlaces) {
        hipLaunchKernelGGL((sort_few<I, V>), dim3((uint32_t)tokens + 1), dim3(256), 0, st, static_cast<const I *>(index), offsets, order, place, static_cast<const V *>(x), static_cast<V *>(rows), ldx,
                           nvec, (uint32_t)tokens, (int)k, (int)E);
        return (int)hipGetLastError();
    }
    const Chunks c = chunks_of(P);
    uint16_t    *table = static_cast<uint16_t *>(ws);
    hipLaunchKernelGGL(count_chunks<I>, dim3(c.count), dim3(256), 0, st, static_cast<const I *>(index), table, (uint32_t)P, c.each, c.stride, (int)E);
    if (const hipError_t e = hipGetLastError()) return (int)e;
    hipLaunchKernelGGL(place_chunks<I>, dim3(c.count), dim3(512), 0, st, static_cast<const I *>(index), table, offsets, order, place, (uint32_t)P, c.each, c.stride, (int)E);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess || !rows) return (int)e;
    const uint32_t pieces = (uint32_t)((nvec + 511) / 512);
    hipLaunchKernelGGL(copy_tokens<V>, grid_of(tokens * pieces), dim3(256), 0, st, static_cast<V *>(rows), static_cast<const V *>(x), place, offsets + E, ldx, (uint32_t)nvec, pieces, (uint32_t)tokens,
                       (int)k);
    return (int)hipGetLastError();
}

int check_places(size_t tokens, size_t k, size_t E)
{
    return k < 1 || k > kMostChosen || E < 1 || E > kMostExperts || tokens > ((size_t)1 << 30) / k ? FP6MI_ERR_SHAPE : FP6MI_OK;
}

// f(row type, output type, values of a vector that both sides' rows can be read and written by)
template <typename F> int by_types(int row_type, int out_type, size_t H, bool vectors, const F &f)
{
    auto with = [&](auto r, auto o) {
        constexpr int V = 16 / (int)sizeof(r);
        return vectors && H % V == 0 ? f(r, o, std::integral_constant<int, V>{}) : f(r, o, std::integral_constant<int, 1>{});
    };
    if (row_type == 0 && out_type == 0) return with(half_t{}, half_t{});
    if (row_type == 1 && out_type == 1) return with(bf16_t{}, bf16_t{});
    if (row_type == 2 && out_type == 2) return with(float{}, float{});
    if (row_type == 2 && out_type == 0) return with(float{}, half_t{});
    if (row_type == 2 && out_type == 1) return with(float{}, bf16_t{});
    return FP6MI_ERR_TYPE;
}

int check_combine(size_t tokens, size_t k, size_t H, int row_type, int out_type)
{
    if (!known_type(row_type) || !known_type(out_type) || (row_type != out_type && row_type != 2)) return FP6MI_ERR_TYPE;
    if (k < 1 || k > kMostChosen || H < 1 || H > (size_t)1 << 24 || tokens > ((size_t)1 << 30) / k) return FP6MI_ERR_SHAPE;
    return FP6MI_OK;
}

} // namespace

extern "C" {

size_t fp6mi_expert_sort_workspace_bytes(size_t tokens, size_t k, size_t experts)
{
    if (tokens == 0 || check_places(tokens, k, experts) != FP6MI_OK || tokens * k <= kFewPlaces) return 0;
    return experts * chunks_of(tokens * k).stride * sizeof(uint16_t);
}

int fp6mi_expert_sort(void *stream, const void *index, int index64, int *offsets, int *order, int *place, const void *x, size_t ldx, void *rows, size_t tokens, size_t k, size_t experts, size_t H,
                      int dtype, void *workspace)
{
    if (const int e = check_places(tokens, k, experts)) return e;
    if (!offsets || (tokens && (!index || !order || !place))) return FP6MI_ERR_NULL;
    if (!aligned(offsets, 4) || !aligned(order, 4) || !aligned(place, 4) || !aligned(index, index64 ? 8 : 4)) return FP6MI_ERR_ALIGN;
    const bool copies = rows != nullptr && tokens != 0;
    size_t     unit = 16;
    if (copies) {
        if (!x) return FP6MI_ERR_NULL;
        if (!known_type(dtype)) return FP6MI_ERR_TYPE;
        if (H < 1 || H > (size_t)1 << 24 || (ldx < H && tokens > 1) || ldx > (size_t)1 << 40) return FP6MI_ERR_SHAPE;
        unit = type_size(dtype);
        if (!aligned(x, unit) || !aligned(rows, unit)) return FP6MI_ERR_ALIGN;
        if (tokens * ((H * unit + 511) / 512) > 0x7fffffffu) return FP6MI_ERR_SHAPE;
        if (aligned(x, 16) && aligned(rows, 16) && H * unit % 16 == 0 && (ldx * unit % 16 == 0 || tokens == 1)) unit = 16;
    }
    if (fp6mi_expert_sort_workspace_bytes(tokens, k, experts) && !workspace) return FP6MI_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return FP6MI_ERR_ALIGN;
    hipStream_t  st = static_cast<hipStream_t>(stream);
    const size_t bytes = copies ? type_size(dtype) : 16, nvec = copies ? H * bytes / unit : 0, ld = copies ? ldx * bytes / unit : 0;
    void        *to = copies ? rows : nullptr;
    return by_index(index64, [&](auto wide) {
        typedef std::conditional_t<decltype(wide)::value, int64_t, int32_t> I;
        if (unit == 16) return launch_sort<I, v4u>(st, index, offsets, order, place, x, to, ld, nvec, tokens, k, experts, workspace);
        if (unit == 4) return launch_sort<I, uint32_t>(st, index, offsets, order, place, x, to, ld, nvec, tokens, k, experts, workspace);
        return launch_sort<I, uint16_t>(st, index, offsets, order, place, x, to, ld, nvec, tokens, k, experts, workspace);
    });
}

int fp6mi_expert_combine(void *stream, const void *rows, const int *place, const int *valid, const float *weights, void *out, size_t tokens, size_t k, size_t H, int row_type, int out_type)
{
    if (const int e = check_combine(tokens, k, H, row_type, out_type)) return e;
    if (tokens == 0) return FP6MI_OK;
    if (!rows || !place || !valid || !out) return FP6MI_ERR_NULL;
    if (!aligned(rows, type_size(row_type)) || !aligned(out, type_size(out_type)) || !aligned(place, 4) || !aligned(valid, 4) || !aligned(weights, 4)) return FP6MI_ERR_ALIGN;
    return by_types(row_type, out_type, H, aligned(rows, 16) && aligned(out, 16), [&](auto r, auto o, auto vec) {
        typedef decltype(r) R;
        typedef decltype(o) O;
        constexpr int  V = decltype(vec)::value;
        const uint32_t nvec = (uint32_t)(H / V), pieces = (nvec + 255) / 256;
        if (tokens * pieces > 0x7fffffffu) return FP6MI_ERR_SHAPE;
        hipLaunchKernelGGL((combine_rows<R, O, V>), grid_of(tokens * pieces), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<O *>(out), static_cast<const R *>(rows), place, valid,
                           weights, nvec, pieces, (uint32_t)tokens, (int)k);
        return (int)hipGetLastError();
    });
}

int fp6mi_expert_combine_backward(void *stream, const void *grad, const void *rows, const int *place, const int *valid, const float *weights, void *grad_rows, float *grad_weights, size_t tokens,
                                  size_t k, size_t H, int row_type, int out_type)
{
    if (const int e = check_combine(tokens, k, H, row_type, out_type)) return e;
    if (tokens == 0) return FP6MI_OK;
    if (!grad || !place || !valid || (grad_weights && !rows) || (!grad_rows && !grad_weights)) return FP6MI_ERR_NULL;
    if (!aligned(rows, type_size(row_type)) || !aligned(grad_rows, type_size(row_type)) || !aligned(grad, type_size(out_type)) || !aligned(place, 4) || !aligned(valid, 4) ||
        !aligned(weights, 4) || !aligned(grad_weights, 4))
        return FP6MI_ERR_ALIGN;
    return by_types(row_type, out_type, H, aligned(rows, 16) && aligned(grad_rows, 16) && aligned(grad, 16), [&](auto r, auto o, auto vec) {
        typedef decltype(r) R;
        typedef decltype(o) O;
        constexpr int  V = decltype(vec)::value;
        const uint32_t parts = (uint32_t)((k + 3) / 4);
        if (tokens * parts > 0x7fffffffu) return FP6MI_ERR_SHAPE;
        hipLaunchKernelGGL((combine_gradient<R, O, V>), grid_of(tokens * parts), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<R *>(grad_rows), grad_weights, static_cast<const O *>(grad),
                           static_cast<const R *>(rows), place, valid, weights, (uint32_t)(H / V), (uint32_t)tokens, (int)k, parts);
        return (int)hipGetLastError();
    });
}

} // extern "C"
