// Rows of the 4-bit key/value cache: append (rotation of queries and keys, rounding of keys and values to
// 4 bits) and read back.
//
// A warp has a row of a head.  Of 64 values x, limited to +-61440: l = half(min x), s = half((max x - l) / 15),
// c = rint((x - l) / s) within 0..15; the limit keeps s c + l inside FP16.  Both differences and quotients are
// single FP32 operations, so the codes follow from the rounded activations alone.
#include <cfloat>

#include "cache4.cuh"
#include "launch.cuh"

namespace tllm {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;

template <typename T>
struct AppendArgs {
    Cache4 c;
    Rotary r;
    Seqs s;
    int heads;
    Rows<const T> q, k, v;
    Rows<T> q_out;
};

// Entries 64 g + 2 lane and the next of a row, turned.
template <typename T, int DIM>
__device__ __forceinline__ void turned_row(const Rotary& r, const T* x, int position, int lane, float (&y)[DIM / 32])
{
#pragma unroll
    for (int i = 0; i < DIM / 32; i++) {
        const int e = (i >> 1) * 64 + 2 * lane + (i & 1);
        y[i] = as_float(x[e]);
        if (r.turns && e < r.rot) {
            const int pairs = r.rot / 2, pair = r.half_layout ? e % pairs : e >> 1;
            const bool second = r.half_layout ? e >= pairs : e & 1;
            const float other = as_float(x[r.half_layout ? (second ? e - pairs : e + pairs) : e ^ 1]);
            float c, s;
            turn(r, r.turns[pair], position, c, s);
            y[i] = as_float(as_type<T>(second ? y[i] * c + other * s : y[i] * c - other * s));
        }
    }
}

// Writes a row of DIM values; `bad`: its params become NaN.
template <int DIM>
__device__ __forceinline__ void write_row(uint8_t* codes, half2* params, size_t row, int lane, const float (&x)[DIM / 32], bool bad)
{
#pragma unroll
    for (int g = 0; g < DIM / 64; g++) {
        float v[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float a = x[2 * g + i];
            v[i] = a != a ? 0.f : fminf(fmaxf(a, -TLLM_CACHE4_LIMIT), TLLM_CACHE4_LIMIT);
        }
        const half l = __float2half_rn(-warp_max(fmaxf(-v[0], -v[1])));
        const float lf = __half2float(l);
        const half s = __float2half_rn((warp_max(fmaxf(v[0], v[1])) - lf) / 15.f);
        const float sf = __half2float(s);
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float c = sf > 0.f ? fminf(fmaxf(rintf((v[i] - lf) / sf), 0.f), 15.f) : 0.f;
            word |= (uint32_t)c << (4 * (lane & 3) + 16 * i);
        }
        word |= __shfl_xor_sync(0xffffffffu, word, 1);
        word |= __shfl_xor_sync(0xffffffffu, word, 2);
        if ((lane & 3) == 0) reinterpret_cast<uint32_t*>(codes + row * (DIM / 2))[g * 8 + (lane >> 2)] = word;
        if (lane == 0) params[row * (DIM / 64) + g] = bad ? __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff)) : __halves2half2(s, l);
    }
}

// Warps of a row: one for each query head, one for each key/value head.
template <typename T, int DIM>
__global__ void __launch_bounds__(kThreads)
cache4_append_kernel(const AppendArgs<T> a)
{
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, row = blockIdx.x, h = blockIdx.y * kWarps + (threadIdx.x >> 5);
    if (h >= a.heads + a.c.kv_heads) return;
    if (row == 0 && h == 0)
        for (int b = lane; b < a.s.batch; b += 32) span_of(a.s, b, true);
    const int b = seq_of_row(a.s, row, lane);
    if (b >= a.s.batch) return;
    const Span sp = span_of(a.s, b, false);
    const int position = sp.position(row - sp.row0);
    if (position < 0 || row < sp.row0) return;
    float y[DIM / 32];
    if (h < a.heads) {
        turned_row<T, DIM>(a.r, a.q.p + (size_t)row * a.q.ld + (size_t)h * DIM, position, lane, y);
        __syncwarp();                                       // q_out may be q
        T* o = a.q_out.p + (size_t)row * a.q_out.ld + (size_t)h * DIM;
#pragma unroll
        for (int i = 0; i < DIM / 32; i++) o[(i >> 1) * 64 + 2 * lane + (i & 1)] = as_type<T>(y[i]);
        return;
    }
    const int g = h - a.heads;
    const size_t at = cache_row(a.c, b, g, position);
    float v[DIM / 32];
    turned_row<T, DIM>(a.r, a.k.p + (size_t)row * a.k.ld + (size_t)g * DIM, position, lane, y);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < DIM / 32; i++) {
        v[i] = as_float(a.v.p[(size_t)row * a.v.ld + (size_t)g * DIM + (i >> 1) * 64 + 2 * lane + (i & 1)]);
        bad = bad || y[i] != y[i] || v[i] != v[i];
    }
    bad = __any_sync(0xffffffffu, bad);
    write_row<DIM>(a.c.kc, a.c.kp, at, lane, y, bad);
    write_row<DIM>(a.c.vc, a.c.vp, at, lane, v, false);
}

template <typename T, int DIM>
__global__ void __launch_bounds__(kThreads)
cache4_read_kernel(const Cache4 c, const Seqs s, const Rows<T> k, const Rows<T> v)
{
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, row = blockIdx.x, g = blockIdx.y * kWarps + (threadIdx.x >> 5);
    if (g >= c.kv_heads) return;
    if (row == 0 && g == 0)
        for (int b = lane; b < s.batch; b += 32) span_of(s, b, true);
    const int b = seq_of_row(s, row, lane);
    if (b >= s.batch) return;
    const Span sp = span_of(s, b, false);
    const int position = sp.position(row - sp.row0);
    if (row < sp.row0) return;
    const size_t at = cache_row(c, b, g, max(position, 0));
#pragma unroll
    for (int side = 0; side < 2; side++) {
        const Rows<T>& o = side ? v : k;
        if (!o.p) continue;
#pragma unroll
        for (int i = 0; i < DIM / 64; i++) {
            float2 x = make_float2(0.f, 0.f);
            if (position >= 0) {
                const uint32_t w = reinterpret_cast<const uint32_t*>((side ? c.vc : c.kc) + at * (DIM / 2))[i * 8 + (lane >> 2)] >> (4 * (lane & 3));
                const float2 p = __half22float2((side ? c.vp : c.kp)[at * (DIM / 64) + i]);
                x = make_float2(fmaf((float)(w & 15), p.x, p.y), fmaf((float)((w >> 16) & 15), p.x, p.y));
            }
            T* y = o.p + (size_t)row * o.ld + (size_t)g * DIM + i * 64 + 2 * lane;
            y[0] = as_type<T>(x.x);
            y[1] = as_type<T>(x.y);
        }
    }
}

}  // namespace

template <typename T>
int launch_cache4_append(const Cache4& c, const Rotary& r, const Seqs& s, Rows<const T> q, Rows<T> q_out, int heads, Rows<const T> k, Rows<const T> v,
                         cudaStream_t stream)
{
    if (s.tokens == 0 || s.batch == 0) return TLLM_OK;
    const dim3 grid(s.tokens, (heads + c.kv_heads + kWarps - 1) / kWarps);
    return launch_pdl("cache4_append", c.dim == 64 ? cache4_append_kernel<T, 64> : cache4_append_kernel<T, 128>, grid, dim3(kThreads), 0, stream,
                      AppendArgs<T>{c, r, s, heads, q, k, v, q_out});
}

template <typename T>
int launch_cache4_read(const Cache4& c, const Seqs& s, Rows<T> k, Rows<T> v, cudaStream_t stream)
{
    if (s.tokens == 0 || s.batch == 0) return TLLM_OK;
    return launch_pdl("cache4_read", c.dim == 64 ? cache4_read_kernel<T, 64> : cache4_read_kernel<T, 128>,
                      dim3(s.tokens, (c.kv_heads + kWarps - 1) / kWarps), dim3(kThreads), 0, stream, c, s, k, v);
}

#define TLLM_INSTANTIATE(T)                                                                                                                       \
    template int launch_cache4_append<T>(const Cache4&, const Rotary&, const Seqs&, Rows<const T>, Rows<T>, int, Rows<const T>, Rows<const T>, \
                                         cudaStream_t);                                                                                          \
    template int launch_cache4_read<T>(const Cache4&, const Seqs&, Rows<T>, Rows<T>, cudaStream_t);
TLLM_INSTANTIATE(half)
TLLM_INSTANTIATE(bf16)
#undef TLLM_INSTANTIATE
template int launch_cache4_read<float>(const Cache4&, const Seqs&, Rows<float>, Rows<float>, cudaStream_t);

}  // namespace tllm
