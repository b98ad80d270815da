// Attention over the 4-bit key/value cache: tiles of rows whose positions several CTAs took, joined from the CTAs'
// records (maxima, sums of weights, outputs that are not divided by them).
//
// A CTA here for each that has the first chunk of a shared tile: weights of all records first, then their outputs, every
// load independent of the others.  A thread has four channels of a row and every kParts-th record; the parts meet in
// shared memory.  The order of all sums is fixed.  Bound by three dependent rounds of loads and the launch: alone, with records in L2, 6.4 us
// for 296 records of 4 rows of 128, 37 a tile (0.6 MB; 8.7 from DRAM), 4.6 where 300 tiles are shared by one to ten, 13.9 for 148 of 256 rows
// (27 MB; 19 from DRAM).
#include "cache4.cuh"
#include "cache4_work.cuh"
#include "dense.cuh"
#include "launch.cuh"

namespace tllm {

namespace {

constexpr int kThreads = 512;
template <int ROWS> constexpr int kMostCtas = ROWS <= 16 ? 512 : 160;
// Rows of a CTA: tiles of 128 in 16s 79 tokens behind 2500 take 25.7 us, in 32s 27.1, in 8s 28; tiles of 256 in 32s 512 behind 16000 163, in 16s 164, in 8s 175.
template <int ROWS> constexpr int kJoinRows = ROWS <= 16 ? 4 : ROWS / 8;

template <typename T, int DIM, int ROWS>
__global__ void __launch_bounds__(kThreads)
cache4_join_kernel(const Cache4Call a, const Rows<T> out, const int ctas)
{
    constexpr int kBlock = kJoinRows<ROWS>;
    constexpr int kElems = kBlock * (DIM / 4), kParts = kElems < kThreads ? kThreads / kElems : 1, kStride = 2 * kRecord<DIM, ROWS>;
    __shared__ float weight[kBlock][kMostCtas<ROWS>], sums[kBlock];
    __shared__ float4 parts[kParts > 1 ? kThreads : 1];
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per = a.heads / a.c.kv_heads, r0 = blockIdx.y * kBlock;
    pdl_wait();
    const Shared4 tile = *entry_of(a.ws, blockIdx.x);
    const int n = tile.parts, rows = min(min(ROWS, tile.n * per - tile.tile * ROWS) - r0, kBlock);
    if (n == 0 || rows <= 0) return;
    const float* rec = record_of<DIM, ROWS>(a.ws, ctas, blockIdx.x, 0);
    const int first = tile.slot ? kRecord<DIM, ROWS> : 0;
    const auto at = [&](int i) { return rec + (size_t)i * kStride + (i == 0 ? first : 0); };
    // four channels of a row
    const auto store = [&](int r, int col, float4 y) {
        const int i = (tile.tile * ROWS + r0 + r) / per, head = tile.head * per + (tile.tile * ROWS + r0 + r) % per;
        store_row<T>(out.p + (size_t)(tile.row0 + i) * out.ld + (size_t)head * DIM + col, y, sums[r], tile.len - tile.n + i >= 0);
    };

    constexpr int kAhead = 8;                                               // outputs requested before the weights are known
    const int e0 = tid % (kParts > 1 ? kElems : kThreads), part = kParts > 1 ? tid / kElems : 0;
    const auto output = [&](int e, int i) { return *reinterpret_cast<const float4*>(at(i) + 2 * ROWS + (r0 + e / (DIM / 4)) * DIM + e % (DIM / 4) * 4); };
    float4 ahead[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; k++)
        if (e0 < rows * (DIM / 4) && part + k * kParts < n) ahead[k] = output(e0, part + k * kParts);
    for (int r = warp; r < rows; r += kThreads / 32) {
        float m = -INFINITY, l = 0.f;
        for (int i = lane; i < n; i += 32) m = fmaxf(m, at(i)[r0 + r]);
        m = warp_max(m);
        const float ref = m == -INFINITY ? 0.f : m;
        for (int i = lane; i < n; i += 32) {
            const float w = exp2_neg(at(i)[r0 + r] - ref);
            weight[r][i] = w;
            l = fmaf(at(i)[ROWS + r0 + r], w, l);
        }
        l = warp_sum(l);
        if (lane == 0) sums[r] = l;
    }
    __syncthreads();
    for (int e = e0; e < rows * (DIM / 4); e += kParts > 1 ? kElems : kThreads) {
        const int r = e / (DIM / 4), col = e % (DIM / 4) * 4;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        const auto add = [&](float4 v, int i) {
            const float w = weight[r][i];
            y = make_float4(fmaf(v.x, w, y.x), fmaf(v.y, w, y.y), fmaf(v.z, w, y.z), fmaf(v.w, w, y.w));
        };
        int i = part;
        if (e == e0) {
#pragma unroll
            for (int k = 0; k < kAhead; k++, i += kParts)
                if (i < n) add(ahead[k], i);
        }
#pragma unroll 8
        for (; i < n; i += kParts) add(output(e, i), i);
        if (kParts > 1) parts[tid] = y;
        else store(r, col, y);
    }
    if (kParts > 1) {
        __syncthreads();
        if (tid < rows * (DIM / 4)) {
            float4 y = parts[tid];
#pragma unroll
            for (int i = 1; i < kParts; i++) {
                const float4 v = parts[tid + i * kElems];
                y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
            }
            store(tid / (DIM / 4), tid % (DIM / 4) * 4, y);
        }
    }
}

template <typename T, int ROWS>
int launch(const Cache4Call& a, Rows<T> out, int ctas, cudaStream_t stream)
{
    if (ctas > kMostCtas<ROWS>) return fail(TLLM_ERR_SIZE, "cache4_join: %d parts", ctas);
    const auto kernel = a.c.dim == 64 ? cache4_join_kernel<T, 64, ROWS> : cache4_join_kernel<T, 128, ROWS>;
    return launch_pdl("cache4_join", kernel, dim3(ctas, ROWS / kJoinRows<ROWS>), dim3(kThreads), 0, stream, a, out, ctas);
}

}  // namespace

template <typename T>
int launch_cache4_join(const Cache4Call& a, Rows<T> out, int rows, int ctas, cudaStream_t stream)
{
    if (rows == 4) return launch<T, 4>(a, out, ctas, stream);
    if (rows == 8) return launch<T, 8>(a, out, ctas, stream);
    if (rows == 16) return launch<T, 16>(a, out, ctas, stream);
    if (rows == 128) return launch<T, 128>(a, out, ctas, stream);
    return launch<T, 256>(a, out, ctas, stream);
}

template int launch_cache4_join<half>(const Cache4Call&, Rows<half>, int, int, cudaStream_t);
template int launch_cache4_join<bf16>(const Cache4Call&, Rows<bf16>, int, int, cudaStream_t);

}  // namespace tllm
