// Attention over the 4-bit key/value cache: tiles of rows whose positions several CTAs took, joined in the order of
// the CTAs from their records (maxima, sums of weights, outputs that are not divided by them).
#include "cache4.cuh"
#include "cache4_work.cuh"
#include "dense.cuh"
#include "launch.cuh"

namespace tllm {

namespace {

constexpr int kThreads = 256, kBlockRows = 16;       // rows of a tile that a CTA joins

template <typename T, int DIM, int ROWS, int CHUNK>
__global__ void __launch_bounds__(kThreads)
cache4_join_kernel(const Cache4Call a, const Rows<T> out, const int ctas)
{
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, per = a.heads / a.c.kv_heads;
    pdl_wait();
    Work<ROWS, CHUNK> work(a.s, per, a.c.kv_heads, false, lane), items(a.s, per, a.c.kv_heads, true, lane);
    for (long long item = blockIdx.x; item < items.total; item += gridDim.x) {
        items.find(item, lane);
        // the chunks of this tile among all
        long long x0 = work.before(items.b, lane) + items.head * work.units(items.span);
        for (int i = 0; i < items.tile; i++) x0 += work.chunks_of(items.span, i);
        const int c0 = work.owner(x0, ctas), c1 = work.owner(x0 + items.chunks - 1, ctas);
        if (c0 == c1) continue;
        const int r0 = items.tile * ROWS, from = blockIdx.y * kBlockRows, to = min(min(ROWS, items.rows - r0), from + kBlockRows);
        const bool later = work.start(c0, ctas) < x0;                      // the first CTA had another tile before
        for (int e = from * (DIM / 4) + threadIdx.x; e < to * (DIM / 4); e += kThreads) {
            const int r = e / (DIM / 4), col = e % (DIM / 4) * 4;
            float m = -INFINITY, l = 0.f;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = c0; c <= c1; c++) {
                const float* rec = static_cast<const float*>(a.ws) + ((size_t)c * 2 + (c == c0 && later)) * kRecord<DIM, ROWS>;
                const float top = fmaxf(m, rec[r]), ref = top == -INFINITY ? 0.f : top, f = exp2_neg(m - ref), w = exp2_neg(rec[r] - ref);
                const float4 v = *reinterpret_cast<const float4*>(rec + 2 * ROWS + r * DIM + col);
                m = top;
                l = fmaf(rec[ROWS + r], w, l * f);
                y = make_float4(fmaf(v.x, w, y.x * f), fmaf(v.y, w, y.y * f), fmaf(v.z, w, y.z * f), fmaf(v.w, w, y.w * f));
            }
            const int i = (r0 + r) / per, head = items.head * per + (r0 + r) % per;
            store_row<T>(out.p + (size_t)(items.span.row0 + i) * out.ld + (size_t)head * DIM + col, y, l, items.span.position(i) >= 0);
        }
    }
}

template <typename T, int ROWS, int CHUNK>
int launch(const Cache4Call& a, Rows<T> out, int ctas, int items, cudaStream_t stream)
{
    const auto kernel = a.c.dim == 64 ? cache4_join_kernel<T, 64, ROWS, CHUNK> : cache4_join_kernel<T, 128, ROWS, CHUNK>;
    return launch_pdl("cache4_join", kernel, dim3(items, (ROWS + kBlockRows - 1) / kBlockRows), dim3(kThreads), 0, stream, a, out, ctas);
}

}  // namespace

template <typename T>
int launch_cache4_join(const Cache4Call& a, Rows<T> out, int rows, int ctas, int items, cudaStream_t stream)
{
    if (rows == 8) return launch<T, 8, kStepChunk>(a, out, ctas, items, stream);
    if (rows == 16) return launch<T, 16, kStepChunk>(a, out, ctas, items, stream);
    return launch<T, kPromptRows, kPromptChunk>(a, out, ctas, items, stream);
}

template int launch_cache4_join<half>(const Cache4Call&, Rows<half>, int, int, int, cudaStream_t);
template int launch_cache4_join<bf16>(const Cache4Call&, Rows<bf16>, int, int, int, cudaStream_t);

}  // namespace tllm
