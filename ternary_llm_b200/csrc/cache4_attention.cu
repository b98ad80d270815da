// Attention over the 4-bit key/value cache for sequences of different lengths.
#include <cfloat>

#include "cache4.cuh"
#include "cache4_work.cuh"
#include "launch.cuh"

namespace tllm {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;

// A warp has a query head of a row and walks over the positions that it sees, 32 at once: a lane has a position's
// score, then two outputs of every group of 64.  One pass, running maximum and sum in FP32.
template <typename T, int DIM>
__global__ void __launch_bounds__(kThreads)
cache4_attention_kernel(const Cache4Call a, const Rows<const T> q, const Rows<T> out)
{
    __shared__ float qs[kWarps][DIM];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x, h = blockIdx.y * kWarps + warp;
    if (h >= a.heads) return;
    if (row == 0 && h == 0)
        for (int b = lane; b < a.s.batch; b += 32) span_of(a.s, b, true);
    const int b = seq_of_row(a.s, row, lane);
    if (b >= a.s.batch) return;
    const Span sp = span_of(a.s, b, false);
    if (row < sp.row0) return;
    const int sees = sp.position(row - sp.row0) + 1, g = h / (a.heads / a.c.kv_heads);
    for (int e = lane; e < DIM; e += 32) qs[warp][e] = as_float(q.p[(size_t)row * q.ld + (size_t)h * DIM + e]) * a.scale * 1.4426950408889634f;
    __syncwarp();
    const size_t base = cache_row(a.c, b, g, 0);
    float m = -INFINITY, l = 0.f, o[DIM / 32] = {};
    for (int p0 = 0; p0 < sees; p0 += 32) {
        float s = -INFINITY;
        if (p0 + lane < sees) {
            const size_t at = base + p0 + lane;
            s = 0.f;
            for (int i = 0; i < DIM / 64; i++) {
                const float2 par = __half22float2(a.c.kp[at * (DIM / 64) + i]);
                for (int j = 0; j < 8; j++) {
                    const uint32_t w = reinterpret_cast<const uint32_t*>(a.c.kc + at * (DIM / 2))[i * 8 + j];
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        s = fmaf(fmaf((float)((w >> (4 * (e >> 1) + 16 * (e & 1))) & 15), par.x, par.y), qs[warp][i * 64 + j * 8 + e], s);
                }
            }
        }
        const float top = fmaxf(m, warp_max(s)), f = m == -INFINITY ? 0.f : exp2f(m - top), p = exp2f(s - (top == -INFINITY ? 0.f : top));
        m = top;
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < DIM / 32; i++) o[i] *= f;
        for (int j = 0; j < min(32, sees - p0); j++) {
            const float pj = __shfl_sync(0xffffffffu, p, j);
            const size_t at = base + p0 + j;
#pragma unroll
            for (int i = 0; i < DIM / 64; i++) {
                const uint32_t w = reinterpret_cast<const uint32_t*>(a.c.vc + at * (DIM / 2))[i * 8 + (lane >> 2)] >> (4 * (lane & 3));
                const float2 par = __half22float2(a.c.vp[at * (DIM / 64) + i]);
                o[2 * i] = fmaf(pj, fmaf((float)(w & 15), par.x, par.y), o[2 * i]);
                o[2 * i + 1] = fmaf(pj, fmaf((float)((w >> 16) & 15), par.x, par.y), o[2 * i + 1]);
            }
        }
    }
    l = warp_sum(l);
    T* y = out.p + (size_t)row * out.ld + (size_t)h * DIM;
#pragma unroll
    for (int i = 0; i < DIM / 32; i++) y[(i >> 1) * 64 + 2 * lane + (i & 1)] = as_type<T>(sees > 0 ? o[i] / l : 0.f);
}

}  // namespace

static bool takes_step(const Cache4& c, int tokens, int heads, int max_new) { return (max_new > 0 ? max_new : tokens) * (heads / c.kv_heads) <= 16; }

size_t cache4_workspace(const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    return takes_step(c, tokens, heads, max_new) ? step_plan(c, tokens, heads, max_new, max_len).bytes : 0;
}

template <typename T>
int launch_cache4_attention(const Cache4Call& a, Rows<const T> q, Rows<T> out, cudaStream_t stream)
{
    if (a.s.tokens == 0 || a.s.batch == 0) return TLLM_OK;
    if (takes_step(a.c, a.s.tokens, a.heads, a.max_new))
        return launch_cache4_step<T>(a, q, out, step_plan(a.c, a.s.tokens, a.heads, a.max_new, a.max_len), stream);
    return launch_pdl("cache4_attention", a.c.dim == 64 ? cache4_attention_kernel<T, 64> : cache4_attention_kernel<T, 128>,
                      dim3(a.s.tokens, (a.heads + kWarps - 1) / kWarps), dim3(kThreads), 0, stream, a, q, out);
}

template int launch_cache4_attention<half>(const Cache4Call&, Rows<const half>, Rows<half>, cudaStream_t);
template int launch_cache4_attention<bf16>(const Cache4Call&, Rows<const bf16>, Rows<bf16>, cudaStream_t);

}  // namespace tllm
