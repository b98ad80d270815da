// The 4-bit key/value cache: its layout, the sequences of a call, rotary angles; launchers of
// rotary.cu, cache4_rows.cu and cache4_attention.cu.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"
#include "tllm_b200_cache4.h"

namespace tllm {

using bf16 = __nv_bfloat16;

constexpr int kCacheGroup = TLLM_CACHE4_GROUP;

// Rotation of a head's first `rot` entries; turns null: none.
struct Rotary {
    const unsigned long long* turns;
    int rot, half_layout;
    float amplitude;
    int inverse;
};

// Rows of activations: p + row * ld + head * dim.
template <typename T>
struct Rows {
    T* p;
    long long ld;
};

struct Cache4 {
    uint8_t *kc, *vc;
    half2 *kp, *vp;                    // (s, l)
    int batch, kv_heads, rows, dim;
};

// The sequences of a call; what the device holds is cut to the limits of the tensors, see Span.
struct Seqs {
    const int *first, *lens;
    int batch, tokens, rows;           // rows: of the cache
    int* err;
};

#ifdef __CUDACC__
// Sequence b of a call: n activation rows from row0 on at positions len - n .. len - 1.
struct Span {
    int row0, n, len;
    bool falls;                        // first does: sequences may share rows
    __device__ __forceinline__ int position(int i) const { return len - n + i; }
};
__device__ __forceinline__ Span span_of(const Seqs& s, int b, bool report)
{
    const int lo = s.first[b], hi = s.first[b + 1], len = s.lens[b];
    Span r;
    r.row0 = min(max(lo, 0), s.tokens);
    r.n = max(min(max(hi, 0), s.tokens) - r.row0, 0);
    r.len = min(max(len, 0), s.rows);
    r.falls = hi < lo;
    if (report && (lo < 0 || hi > s.tokens || hi < lo || len < 0 || len > s.rows)) atomicExch(s.err, TLLM_ERR_SHAPE);
    return r;
}
// Cosine and sine of a pair at a position, times the amplitude.  The position times the turns a position, as 64-bit fractions of a turn,
// is exact modulo whole turns; from there on 64 bits until the one rounding (a row's angles are computed once for all of its heads).
__device__ __forceinline__ void turn(const Rotary& r, unsigned long long turns, int position, float& c, float& s)
{
    const long long phase = (long long)(turns * (unsigned long long)(long long)position);
    double sd, cd;
    sincospi((double)phase * 0x1p-63, &sd, &cd);
    c = (float)(cd * (double)r.amplitude);
    s = (float)(sd * (double)(r.inverse ? -r.amplitude : r.amplitude));
}

// The turned pair: products and sum are FP32 operations of their own, so that every kernel rounds alike and codes follow from the definition.
__device__ __forceinline__ float turned_first(float x1, float x2, float2 c) { return __fsub_rn(__fmul_rn(x1, c.x), __fmul_rn(x2, c.y)); }
__device__ __forceinline__ float turned_second(float x1, float x2, float2 c) { return __fadd_rn(__fmul_rn(x2, c.x), __fmul_rn(x1, c.y)); }

template <typename T> __device__ __forceinline__ float as_float(T x);
template <> __device__ __forceinline__ float as_float<half>(half x) { return __half2float(x); }
template <> __device__ __forceinline__ float as_float<bf16>(bf16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float as_float<float>(float x) { return x; }
template <typename T> __device__ __forceinline__ T as_type(float x);
template <> __device__ __forceinline__ half as_type<half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ bf16 as_type<bf16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ float as_type<float>(float x) { return x; }

// 16 bytes of activations as FP32 numbers.
template <typename T>
struct Vec {
    static constexpr int n = 16 / sizeof(T);
    float v[n];
    __device__ __forceinline__ void load(const T* p)
    {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
        for (int i = 0; i < n; i++) v[i] = as_float(e[i]);
    }
    __device__ __forceinline__ void store(T* p) const
    {
        uint4 x;
        T* e = reinterpret_cast<T*>(&x);
#pragma unroll
        for (int i = 0; i < n; i++) e[i] = as_type<T>(v[i]);
        *reinterpret_cast<uint4*>(p) = x;
    }
};

// The rotation of a head in units of 16 bytes.  Half layout with pairs in whole units: unit u < pairs / n is two, u and u + pairs / n, which
// turn together; other units are one each.  cs: cos and sin of the pairs at a position.
template <typename T>
struct Turn {
    static constexpr int n = Vec<T>::n;
    int pairs, together, per_head;     // units that hold two, units of a head
    bool half_layout;
    __host__ __device__ Turn(const Rotary& r, int dim) : pairs(r.rot / 2), half_layout(r.half_layout)
    {
        together = half_layout ? pairs / n : 0;
        per_head = dim / n - together;
    }
    static bool whole(const Rotary& r) { return !r.half_layout || r.rot / 2 % n == 0; }
    // requests unit u of a head
    __device__ __forceinline__ void load(const T* x, int u, uint4 (&w)[2]) const
    {
        const int at = u < together ? u : u + together;
        w[0] = reinterpret_cast<const uint4*>(x)[at];
        if (u < together) w[1] = reinterpret_cast<const uint4*>(x)[u + together];
    }
    __device__ __forceinline__ void turn_and_store(T* y, int u, const uint4 (&w)[2], const float2* cs) const
    {
        Vec<T> a, b;
        a.load(reinterpret_cast<const T*>(&w[0]));
        if (u < together) {
            b.load(reinterpret_cast<const T*>(&w[1]));
#pragma unroll
            for (int i = 0; i < n; i++) {
                const float2 c = cs[u * n + i];
                const float x1 = a.v[i], x2 = b.v[i];
                a.v[i] = turned_first(x1, x2, c);
                b.v[i] = turned_second(x1, x2, c);
            }
            a.store(y + u * n);
            b.store(y + (u + together) * n);
            return;
        }
        const int at = u + together;
        if (!half_layout) {
#pragma unroll
            for (int i = 0; i < n; i += 2)
                if (at * n + i < 2 * pairs) {
                    const float2 c = cs[(at * n + i) / 2];
                    const float x1 = a.v[i], x2 = a.v[i + 1];
                    a.v[i] = turned_first(x1, x2, c);
                    a.v[i + 1] = turned_second(x1, x2, c);
                }
        }
        a.store(y + at * n);
    }
};

// First element of a row of the cache, in groups of 64 values.
__device__ __forceinline__ size_t cache_row(const Cache4& c, int b, int g, int row) { return ((size_t)b * c.kv_heads + g) * c.rows + row; }
#endif

template <typename T>
int launch_rotary(const Rotary& r, const int* positions, int tokens, Rows<const T> q, Rows<T> q_out, int heads, Rows<const T> k, Rows<T> k_out,
                  int kv_heads, int dim, cudaStream_t stream);
template <typename T>
int launch_cache4_append(const Cache4& c, const Rotary& r, const Seqs& s, Rows<const T> q, Rows<T> q_out, int heads, Rows<const T> k, Rows<const T> v,
                         cudaStream_t stream);
template <typename T>
int launch_cache4_read(const Cache4& c, const Seqs& s, Rows<T> k, Rows<T> v, cudaStream_t stream);

struct Cache4Call {
    Cache4 c;
    Seqs s;
    int heads, max_new, max_len;
    float scale;
    void* ws;
};
size_t cache4_workspace(const Cache4& c, int tokens, int heads, int max_new, int max_len);
template <typename T>
int launch_cache4_attention(const Cache4Call& a, Rows<const T> q, Rows<T> out, cudaStream_t stream);

}  // namespace tllm
