// The work of a call over the 4-bit cache as one sequence of units, computed on the device from the
// sequences' lengths: tiles of rows of key/value heads, each a number of chunks of positions.
#pragma once
#include "cache4.cuh"

namespace tllm {

constexpr int kStepChunk = 32;                       // positions a warp of cache4_step.cu takes at once
constexpr int kPromptChunk = 128, kPromptRows = 256; // positions and rows a CTA of cache4_prompt.cu takes at once
// Floats of the part of a tile's rows that one CTA found: maxima, sums, outputs.
template <int DIM, int ROWS> constexpr int kRecord = ROWS * (DIM + 2);

struct StepPlan {
    int tiles;                                       // of 8 rows that go through the cache together
    bool whole;                                      // a tile's positions stay in one CTA
    int ctas, items;
    size_t bytes;
};
StepPlan step_plan(const Cache4& c, int tokens, int heads, int max_new, int max_len);
template <typename T>
int launch_cache4_step(const Cache4Call& a, Rows<const T> q, Rows<T> out, const StepPlan& p, cudaStream_t stream);

struct PromptPlan {
    bool whole;
    int ctas, items;
    size_t bytes;
};
PromptPlan prompt_plan(const Cache4& c, int tokens, int heads, int max_new, int max_len);
template <typename T>
int launch_cache4_prompt(const Cache4Call& a, Rows<const T> q, Rows<T> out, const PromptPlan& p, cudaStream_t stream);

// Joins what several of `ctas` CTAs found for one tile of rows; items: about how many tiles there are (cache4_join.cu).
template <typename T>
int launch_cache4_join(const Cache4Call& a, Rows<T> out, int rows, int ctas, int items, cudaStream_t stream);

#ifdef __CUDACC__
// Row r of sequence b and key/value head `head` is query head r % per of the head's, of new token r / per; a tile is R of
// them.  Units are chunks of positions, or whole tiles.  Members are found by whole warps, every lane with the same result.
template <int R, int CHUNK>
struct Work {
    static constexpr int kLeast = CHUNK == kStepChunk ? 16 : 2;            // chunks that a CTA takes at least where work is cut
    Seqs s;
    int per, kv_heads;
    bool whole;
    long long total;
    // the unit that find() or next() came to
    int b, head, tile, offset, rows, chunks, visible;
    Span span;

    __device__ __forceinline__ int seen(const Span& sp, int tl) const      // positions that some row of a tile sees
    {
        const int last = min((tl + 1) * R, sp.n * per) - 1;
        return max(sp.position(last / per) + 1, 0);
    }
    __device__ __forceinline__ int chunks_of(const Span& sp, int tl) const { return max((seen(sp, tl) + CHUNK - 1) / CHUNK, 1); }
    // units of a head of a sequence
    __device__ __forceinline__ long long units(const Span& sp) const
    {
        const int tiles = (int)(((long long)sp.n * per + R - 1) / R);
        if (whole) return tiles;
        long long sum = 0;
        for (int i = 0; i < tiles; i++) sum += chunks_of(sp, i);
        return sum;
    }
    __device__ __forceinline__ Work(const Seqs& s_, int per_, int kv_heads_, bool whole_, int lane) : s(s_), per(per_), kv_heads(kv_heads_), whole(whole_), total(0)
    {
        for (int i = lane; i < s.batch; i += 32) total += units(span_of(s, i, false)) * kv_heads;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    // first unit of part c of `parts`
    __device__ __forceinline__ int used(int parts) const
    {
        if (whole) return parts;
        const long long most = total / kLeast;
        return most < 1 ? 1 : most < parts ? (int)most : parts;
    }
    __device__ __forceinline__ long long start(int c, int parts) const
    {
        const int n = used(parts);
        return c >= n ? total : total * c / n;
    }
    __device__ __forceinline__ int owner(long long x, int parts) const { return (int)(((x + 1) * used(parts) - 1) / total); }

    __device__ __forceinline__ void set_tile(int tl)
    {
        tile = tl;
        visible = seen(span, tl);
        chunks = max((visible + CHUNK - 1) / CHUNK, 1);
    }
    // units of all sequences before b
    __device__ __forceinline__ long long before(int seq, int lane) const
    {
        long long sum = 0;
        for (int i = lane; i < seq; i += 32) sum += units(span_of(s, i, false)) * kv_heads;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return sum;
    }
    // unit x < total
    __device__ __forceinline__ void find(long long x, int lane)
    {
        for (int b0 = 0; b0 < s.batch; b0 += 32) {
            long long mine = b0 + lane < s.batch ? units(span_of(s, b0 + lane, false)) * kv_heads : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(0xffffffffu, mine, o);
                if (lane >= o) mine += v;
            }
            const uint32_t m = __ballot_sync(0xffffffffu, mine > x);
            const int at = m ? __ffs(m) - 1 : 31;
            const long long below = __shfl_sync(0xffffffffu, mine, at > 0 ? at - 1 : 0);
            if (m) {
                b = b0 + at;
                x -= at > 0 ? below : 0;
                break;
            }
            x -= __shfl_sync(0xffffffffu, mine, 31);
        }
        span = span_of(s, b, false);
        rows = span.n * per;
        const long long u = units(span);
        head = (int)(x / u);
        x -= head * u;
        int tl = 0;
        offset = 0;
        if (whole) tl = (int)x;
        else {
            for (int n; x >= (n = chunks_of(span, tl)); tl++) x -= n;
            offset = (int)x;
        }
        set_tile(tl);
    }
    // the tile behind this one
    __device__ __forceinline__ void next()
    {
        offset = 0;
        if ((tile + 1) * R < rows) {
            set_tile(tile + 1);
            return;
        }
        if (++head == kv_heads) {
            head = 0;
            do span = span_of(s, ++b, false);
            while (span.n == 0 && b + 1 < s.batch);
            rows = span.n * per;
        }
        set_tile(0);
    }
};

template <typename T> struct Pair2;
template <> struct Pair2<half> {
    static __device__ __forceinline__ uint32_t of(float x, float y)
    {
        const half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <> struct Pair2<bf16> {
    static __device__ __forceinline__ uint32_t of(float x, float y)
    {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
// Four outputs: y / sum, 0 for a row that sees nothing.
template <typename T>
__device__ __forceinline__ void store_row(T* p, float4 y, float sum, bool sees)
{
    const float f = sees ? 1.f / sum : 0.f;
    if (!sees) y = make_float4(0.f, 0.f, 0.f, 0.f);
    *reinterpret_cast<uint2*>(p) = make_uint2(Pair2<T>::of(y.x * f, y.y * f), Pair2<T>::of(y.z * f, y.w * f));
}
#endif

}  // namespace tllm
