// The work of a call over the 4-bit cache as one sequence of units, computed on the device from the
// sequences' lengths: tiles of rows of key/value heads, each a number of chunks of positions and what a tile costs
// beside them.
#pragma once
#include "cache4.cuh"

namespace tllm {

constexpr int kStepChunk = 32;                       // positions a warp of cache4_step.cu takes at once
constexpr int kStepWhole = 160000;                   // entries of a head's positions up to which one CTA takes a tile of them, see step_plan
constexpr int kPromptChunk = 128;                    // positions a CTA of cache4_prompt.cu takes at once
// Floats of the part of a tile's rows that one CTA found: maxima, sums, outputs.
template <int DIM, int ROWS> constexpr int kRecord = ROWS * (DIM + 2);

// A tile of rows that several CTAs share, written by the one that has its first chunk (parts = 0 by a CTA that has none): its
// record is its first or second one, those of the CTAs behind it are their first.
struct Shared4 {
    int parts, slot, head, tile, row0, n, len, unused;
};
// Workspace: an entry of each CTA, then two records of each.
inline size_t join_bytes(int dim, int rows, int ctas) { return (size_t)ctas * (sizeof(Shared4) + 2 * (size_t)rows * (dim + 2) * sizeof(float)); }
#ifdef __CUDACC__
__device__ __forceinline__ Shared4* entry_of(void* ws, int cta) { return static_cast<Shared4*>(ws) + cta; }
template <int DIM, int ROWS>
__device__ __forceinline__ float* record_of(void* ws, int ctas, int cta, int slot)
{
    return reinterpret_cast<float*>(static_cast<Shared4*>(ws) + ctas) + ((size_t)cta * 2 + slot) * kRecord<DIM, ROWS>;
}
#endif

// New rows of a sequence: the most that the caller names, or as many as sequences have on the average.
inline int new_rows(const Cache4& c, int tokens, int max_new)
{
    if (max_new <= 0) return (tokens + c.batch - 1) / c.batch;
    return max_new < tokens ? max_new : tokens;
}

// Whether the units of a call fit 31 bits, whatever lens and a rising first hold: tiles of `rows` rows, whole or over `len` positions in chunks.
inline bool work_fits(const Cache4& c, int tokens, int heads, int len, int rows, int chunk, bool whole)
{
    const double tiles = (double)tokens * (heads / c.kv_heads) / rows + c.batch, units = whole ? 1 : (double)len / chunk + 22;
    return tiles * units * c.kv_heads < 2e9;
}

struct StepPlan {
    int rows;                                        // that go through the cache together: 4, 8 or 16
    bool whole;                                      // a tile's positions stay in one CTA
    int ctas;
    size_t bytes;
};
StepPlan step_plan(const Cache4& c, int tokens, int heads, int max_new, int max_len);
template <typename T>
int launch_cache4_step(const Cache4Call& a, Rows<const T> q, Rows<T> out, const StepPlan& p, cudaStream_t stream);

struct PromptPlan {
    int rows;                                        // of a CTA: 128 or 256
    bool whole;
    int ctas;
    size_t bytes;
};
PromptPlan prompt_plan(const Cache4& c, int tokens, int heads, int max_new, int max_len);
template <typename T>
int launch_cache4_prompt(const Cache4Call& a, Rows<const T> q, Rows<T> out, const PromptPlan& p, cudaStream_t stream);

// Joins what several of `ctas` CTAs found for one tile of rows (cache4_join.cu).
template <typename T>
int launch_cache4_join(const Cache4Call& a, Rows<T> out, int rows, int ctas, cudaStream_t stream);

#ifdef __CUDACC__
// Row r of sequence b and key/value head `head` is query head r % per of the head's, of new token r / per; a tile is R of
// them.  Units are whole tiles, or chunks of positions behind kFixed units a tile (its rows' loading, joining and
// storing, in chunks), so that CTAs with many short tiles and CTAs with a part of a long one take equally long; a CTA takes
// `share` units in a row.  One warp finds a CTA's first unit (its lanes share sequences or tiles), all threads walk on from there.
// Units are counted in 32 bits (work_fits).
template <int R, int CHUNK>
struct Work {
    static constexpr int kFixed = CHUNK == kStepChunk ? 20 : 4;
    static constexpr int kLeast = CHUNK == kStepChunk ? 36 : 4;            // units that a CTA takes at least where work is cut
    struct Start {
        int x, to, share, b, head, tile, offset;
    };
    Seqs s;
    int per, kv_heads;
    bool whole;
    // the CTA's units, and the tile that begin() or next() came to
    int x, to, share, b, head, tile, offset, rows, chunks, visible;
    Span span;

    __device__ __forceinline__ Work(const Seqs& s_, int per_, int kv_heads_, bool whole_) : s(s_), per(per_), kv_heads(kv_heads_), whole(whole_) {}
    __device__ __forceinline__ int seen(const Span& sp, int tl) const      // positions that some row of a tile sees
    {
        const int last = min((tl + 1) * R, sp.n * per) - 1;
        return max(sp.position(last / per) + 1, 0);
    }
    __device__ __forceinline__ int chunks_of(const Span& sp, int tl) const { return max((seen(sp, tl) + CHUNK - 1) / CHUNK, 1); }
    __device__ __forceinline__ int units_of(const Span& sp, int tl) const { return whole ? 1 : kFixed + chunks_of(sp, tl); }
    // the first chunk at or behind unit u of a tile
    static __device__ __forceinline__ int chunk_at(int u) { return max(u - kFixed, 0); }
    __device__ __forceinline__ int tiles_of(const Span& sp) const { return (sp.n * per + R - 1) / R; }
    __device__ __forceinline__ Span lane_span(int i) const
    {
        Span none;
        none.row0 = none.n = none.len = 0;
        none.falls = false;
        return i < s.batch ? span_of(s, i, false) : none;
    }
    static __device__ __forceinline__ int scan(int v, int lane)
    {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        return v;
    }
    // units of a head of each lane's sequence
    __device__ __forceinline__ int units(const Span& sp, int lane) const
    {
        const int tiles = tiles_of(sp);
        if (whole) return tiles;
        int sum = 0;
        if (__all_sync(0xffffffffu, tiles <= 2)) {
            for (int i = 0; i < tiles; i++) sum += units_of(sp, i);
            return sum;
        }
        for (uint32_t left = __ballot_sync(0xffffffffu, tiles > 0); left; left &= left - 1) {
            const int from = __ffs(left) - 1, n = __shfl_sync(0xffffffffu, tiles, from);
            Span one;
            one.n = __shfl_sync(0xffffffffu, sp.n, from);
            one.len = __shfl_sync(0xffffffffu, sp.len, from);
            int part = 0;
            for (int i = lane; i < n; i += 32) part += units_of(one, i);
            part = __reduce_add_sync(0xffffffffu, part);
            if (lane == from) sum = part;
        }
        return sum;
    }
    // by one warp: where part c of `parts` begins, and reports what is wrong with the sequences
    __device__ __forceinline__ void find(int c, int parts, int lane, Start* out) const
    {
        int total = 0, mine = 0;                      // mine: units of a head of the lane's sequence, of the last 32
        Span sp;
        bool falls = false;                           // then nothing is done: the units of such a call may not fit
        for (int b0 = 0; b0 < s.batch; b0 += 32) {
            sp = lane_span(b0 + lane);
            falls = falls || sp.falls;
            if (c == 0 && b0 + lane < s.batch) span_of(s, b0 + lane, true);
            mine = units(sp, lane);
            total += __reduce_add_sync(0xffffffffu, mine * kv_heads);
        }
        if (__any_sync(0xffffffffu, falls)) total = 0;
        Start r;
        r.share = max((total + parts - 1) / parts, whole ? 1 : kLeast);
        r.x = min((long long)c * r.share, (long long)total);
        r.to = min(r.x + r.share, total);
        r.b = r.head = r.tile = r.offset = 0;
        if (r.x < r.to) {
            int at = r.x, u = 0, i = 0;               // u: units of a head of the sequence
            for (int b0 = 0; b0 < s.batch; b0 += 32) {
                if (s.batch > 32) {
                    sp = lane_span(b0 + lane);
                    mine = units(sp, lane);
                }
                const int up_to = scan(mine * kv_heads, lane);
                const uint32_t m = __ballot_sync(0xffffffffu, up_to > at);
                i = m ? __ffs(m) - 1 : 31;
                const int end = __shfl_sync(0xffffffffu, up_to, i);
                u = __shfl_sync(0xffffffffu, mine, i);
                at -= m ? end - u * kv_heads : end;
                r.b = b0 + i;
                if (m) break;
            }
            sp.n = __shfl_sync(0xffffffffu, sp.n, i);
            sp.len = __shfl_sync(0xffffffffu, sp.len, i);
            r.head = at / u;
            at -= r.head * u;
            const int tiles = tiles_of(sp);
            for (; tiles > 1; r.tile += 32) {
                const int of = r.tile + lane < tiles ? units_of(sp, r.tile + lane) : 0, up_to = scan(of, lane);
                const uint32_t m = __ballot_sync(0xffffffffu, up_to > at);
                i = m ? __ffs(m) - 1 : 31;
                const int end = __shfl_sync(0xffffffffu, up_to, i);
                at -= m ? end - __shfl_sync(0xffffffffu, of, i) : end;
                if (m) {
                    r.tile += i;
                    break;
                }
            }
            r.offset = at;
        }
        if (lane == 0) *out = r;
    }
    __device__ __forceinline__ void set_tile(int tl)
    {
        tile = tl;
        visible = seen(span, tl);
        chunks = max((visible + CHUNK - 1) / CHUNK, 1);
    }
    __device__ __forceinline__ void begin(const Start& f)
    {
        x = f.x;
        to = f.to;
        share = f.share;
        b = f.b;
        head = f.head;
        offset = f.offset;
        if (x < to) {
            span = span_of(s, b, false);
            rows = span.n * per;
            set_tile(f.tile);
        }
    }
    // the CTA that has unit u
    __device__ __forceinline__ int owner(int u) const { return u / share; }
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
// A whole sector at once, on a 32-byte boundary.
__device__ __forceinline__ void store32(void* p, const uint32_t* v)
{
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
#endif

}  // namespace tllm
