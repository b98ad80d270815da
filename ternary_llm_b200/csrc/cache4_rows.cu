// Rows of the 4-bit key/value cache: append (rotation of queries and keys, rounding of keys and values to
// 4 bits) and read back.
//
// Of 64 values x, limited to +-61440: l = half(min x), s = half((max x - l) / 15), c = rint((x - l) / s) within
// 0..15; the limit keeps s c + l inside FP16.  Both differences and quotients are single FP32 operations, so the codes
// follow from the rounded activations alone.  Eight lanes have a group, a lane eight neighbouring values: 16 bytes in,
// a word of codes out.  The keys and values of a head of a row stay with the same lanes, which mark a NaN in either.
// Bound by the chain of a CTA (sequence and position, angles, row): three FP16 prompts of 3982 rows in all, 32 heads of 64
// over 8, 46 MB, take 19 us with four rows a CTA and four CTAs an SM, 24.5 with two CTAs, 22 with eight rows, 48 with one
// row; 24 rows of 128 take 4.8.
#include "cache4.cuh"
#include "launch.cuh"

namespace tllm {

namespace {

constexpr int kThreads = 256;

template <typename T>
struct AppendArgs {
    Cache4 c;
    Rotary r;
    Seqs s;
    int heads;
    Rows<const T> q, k, v;
    Rows<T> q_out;
};

// Where rows row0 .. of a CTA belong: sequence (-1: none) and position.
template <int ROWS>
struct Places {
    int seq[ROWS], position[ROWS];
};
template <int ROWS>
__device__ __forceinline__ void find_places(const Seqs& s, int row0, Places<ROWS>& p)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = row0 + warp;
    if (warp < ROWS) {
        // the first sequence whose end lies behind the row; 32 at once, all their numbers in one round of loads
        int seq = -1, position = 0;
        for (int b0 = 0; b0 < s.batch && row < s.tokens; b0 += 32) {
            const int b = b0 + lane;
            Span sp;
            sp.row0 = sp.n = sp.len = 0;
            int end = 0;
            if (b < s.batch) {
                end = s.first[b + 1];
                sp = span_of(s, b, false);
            }
            const uint32_t m = __ballot_sync(0xffffffffu, b < s.batch && row < end);
            if (!m) continue;
            const int from = __ffs(m) - 1, start = __shfl_sync(0xffffffffu, sp.row0, from), n = __shfl_sync(0xffffffffu, sp.n, from);
            position = __shfl_sync(0xffffffffu, sp.len, from) - n + row - start;
            if (row >= start && row - start < n) seq = b0 + from;
            break;
        }
        if (lane == 0) {
            p.seq[warp] = seq;
            p.position[warp] = position;
        }
    }
    if (row0 == 0 && blockIdx.y == 0 && warp == kThreads / 32 - 1)
        for (int b = lane; b < s.batch; b += 32) span_of(s, b, true);
}

// Sign-exact comparisons of eight lanes.
__device__ __forceinline__ float max8(float v)
{
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The codes and (s, l) of the group that eight lanes hold.  The quotient is the correctly rounded one in three operations:
// a product with the reciprocal and one correction by the exact remainder (Markstein 1990) is within 2^-45 of the true one,
// relative to it, and a quotient by the 11 bits of s lies no nearer than 2^-36 to the middle of two FP32 values.  Four
// codes are put together as one FP32 number.
__device__ __forceinline__ void write_group(uint8_t* codes, half2* params, size_t row, int words, int lane_of_row, const float (&x)[8], bool bad, bool write)
{
    float v[8], low = INFINITY, high = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = fminf(fmaxf(x[i], -TLLM_CACHE4_LIMIT), TLLM_CACHE4_LIMIT);
        low = fminf(low, v[i]);
        high = fmaxf(high, v[i]);
    }
    const half l = __float2half_rn(-max8(-low));
    const float lf = __half2float(l);
    const half s = __float2half_rn((max8(high) - lf) / 15.f);
    const float sf = __half2float(s), r = sf > 0.f ? __frcp_rn(sf) : 0.f;
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float t = v[i] - lf, q = t * r;
        c[i] = fminf(fmaxf(rintf(fmaf(fmaf(-q, sf, t), r, q)), 0.f), 15.f);
    }
    if (!write) return;
    const float even = fmaf(4096.f, c[6], fmaf(256.f, c[4], fmaf(16.f, c[2], c[0]))), odd = fmaf(4096.f, c[7], fmaf(256.f, c[5], fmaf(16.f, c[3], c[1])));
    reinterpret_cast<uint32_t*>(codes)[row * words + lane_of_row] = (uint32_t)even | (uint32_t)odd << 16;
    if ((lane_of_row & 7) == 0)
        params[row * (words / 8) + lane_of_row / 8] = bad ? __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff)) : __halves2half2(s, l);
}

// blockIdx.y = 0: keys and values, 1: queries.
template <typename T, int DIM, int ROWS>
__global__ void __launch_bounds__(kThreads, 4)
cache4_append_kernel(const AppendArgs<T> a)
{
    __shared__ Places<ROWS> at;
    __shared__ float2 cs[ROWS][DIM / 2];
    pdl_launch_dependents();
    const int tid = threadIdx.x, row0 = blockIdx.x * ROWS;
    const int pairs = a.r.turns ? a.r.rot / 2 : 0, rows = min(ROWS, a.s.tokens - row0);
    const bool whole = !a.r.half_layout || pairs % 8 == 0;
    const Turn<T> t(a.r, DIM);
    constexpr int kLanes = DIM / 8;                        // of a row of a head
    const int lane = tid % kLanes, e0 = lane * 8;
    int h = tid / t.per_head, u = tid % t.per_head;
    uint4 w[ROWS][2];
    const auto load = [&] {
#pragma unroll
        for (int r = 0; r < ROWS; r++)
            if (r < rows) t.load(a.q.p + (size_t)(row0 + r) * a.q.ld + (size_t)h * DIM, u, w[r]);
    };
    uint4 kv[3];                                           // key, value, what turns with the key
    const auto load_kv = [&](int i) {
        const int g = i % a.c.kv_heads, r = i / a.c.kv_heads;
        if (r >= rows) return;
        const T* x = a.k.p + (size_t)(row0 + r) * a.k.ld + (size_t)g * DIM;
        kv[0] = *reinterpret_cast<const uint4*>(x + e0);
        kv[1] = *reinterpret_cast<const uint4*>(a.v.p + (size_t)(row0 + r) * a.v.ld + (size_t)g * DIM + e0);
        if (a.r.half_layout && whole && e0 < 2 * pairs) kv[2] = *reinterpret_cast<const uint4*>(x + (e0 >= pairs ? e0 - pairs : e0 + pairs));
    };
    pdl_wait();
    // the rows are on their way while their places and angles are found
    const bool queries = blockIdx.y == 1;
    const unsigned long long first_turn = tid < ROWS * pairs ? a.r.turns[tid % pairs] : 0;
    if (!queries) load_kv(tid / kLanes);
    else if (whole && h < a.heads) load();
    find_places<ROWS>(a.s, row0, at);
    __syncthreads();
    for (int i = tid; i < ROWS * pairs; i += kThreads) {
        const int r = i / pairs, p = i % pairs;
        turn(a.r, i == tid ? first_turn : a.r.turns[p], at.position[r], cs[r][p].x, cs[r][p].y);
    }
    __syncthreads();
    if (queries) {
        if (whole) {
            const int step_h = kThreads / t.per_head, step_u = kThreads % t.per_head;
            for (bool again = false; h < a.heads; again = true) {
                if (again) load();
#pragma unroll
                for (int r = 0; r < ROWS; r++)
                    if (r < rows && at.seq[r] >= 0 && at.position[r] >= 0)
                        t.turn_and_store(a.q_out.p + (size_t)(row0 + r) * a.q_out.ld + (size_t)h * DIM, u, w[r], cs[r]);
                h += step_h;
                u += step_u;
                if (u >= t.per_head) {
                    u -= t.per_head;
                    h++;
                }
            }
            return;
        }
        const int per_head = DIM - pairs;
        for (int i = tid; i < ROWS * a.heads * per_head; i += kThreads) {
            const int e = i % per_head, h = i / per_head % a.heads, r = i / per_head / a.heads;
            if (at.seq[r] < 0 || at.position[r] < 0) continue;
            const T* x = a.q.p + (size_t)(row0 + r) * a.q.ld + (size_t)h * DIM;
            T* y = a.q_out.p + (size_t)(row0 + r) * a.q_out.ld + (size_t)h * DIM;
            if (e >= pairs) {
                y[e + pairs] = x[e + pairs];
                continue;
            }
            const float2 c = cs[r][e];
            const float x1 = as_float(x[e]), x2 = as_float(x[e + pairs]);
            y[e] = as_type<T>(turned_first(x1, x2, c));
            y[e + pairs] = as_type<T>(turned_second(x1, x2, c));
        }
        return;
    }
    // all lanes of a warp stay together: those without a row write nothing
    for (int i0 = 0; i0 < ROWS * a.c.kv_heads; i0 += kThreads / kLanes) {
        const int i = i0 + tid / kLanes, g = i % a.c.kv_heads, r = i / a.c.kv_heads;
        const bool write = r < rows && at.seq[r] >= 0 && at.position[r] >= 0;
        if (i0 > 0) load_kv(i);
        Vec<T> k, v;
        const T* x = a.k.p + (size_t)(row0 + (write ? r : 0)) * a.k.ld + (size_t)g * DIM;
        if (write) {
            k.load(reinterpret_cast<const T*>(&kv[0]));
            v.load(reinterpret_cast<const T*>(&kv[1]));
            if (e0 < 2 * pairs) {
                if (!a.r.half_layout) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                        if (e0 + e < 2 * pairs) {
                            const float2 c = cs[r][(e0 + e) / 2];
                            const float x1 = k.v[e], x2 = k.v[e + 1];
                            k.v[e] = as_float(as_type<T>(turned_first(x1, x2, c)));
                            k.v[e + 1] = as_float(as_type<T>(turned_second(x1, x2, c)));
                        }
                } else if (whole) {
                    const bool second = e0 >= pairs;
                    Vec<T> o;
                    o.load(reinterpret_cast<const T*>(&kv[2]));
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float2 c = cs[r][(second ? e0 - pairs : e0) + e];
                        k.v[e] = as_float(as_type<T>(second ? turned_second(o.v[e], k.v[e], c) : turned_first(k.v[e], o.v[e], c)));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (e0 + e < 2 * pairs) {
                            const bool second = e0 + e >= pairs;
                            const float2 c = cs[r][second ? e0 + e - pairs : e0 + e];
                            const float o = as_float(x[second ? e0 + e - pairs : e0 + e + pairs]);
                            k.v[e] = as_float(as_type<T>(second ? turned_second(o, k.v[e], c) : turned_first(k.v[e], o, c)));
                        }
                }
            }
        }
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (!write) k.v[e] = v.v[e] = 0.f;
            bad = bad || k.v[e] != k.v[e] || v.v[e] != v.v[e];
        }
        bad = __ballot_sync(0xffffffffu, bad) >> ((tid & 31) / kLanes * kLanes) & ((1u << kLanes) - 1);
        if (bad) {                                         // a NaN counts as 0
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (k.v[e] != k.v[e]) k.v[e] = 0.f;
                if (v.v[e] != v.v[e]) v.v[e] = 0.f;
            }
        }
        const size_t to = write ? cache_row(a.c, at.seq[r], g, at.position[r]) : 0;
        write_group(a.c.kc, a.c.kp, to, DIM / 8, lane, k.v, bad, write);
        write_group(a.c.vc, a.c.vp, to, DIM / 8, lane, v.v, false, write);
    }
}

// A word of codes a thread, eight values.
template <typename T, int DIM, int ROWS>
__global__ void __launch_bounds__(kThreads)
cache4_read_kernel(const Cache4 c, const Seqs s, const Rows<T> k, const Rows<T> v)
{
    __shared__ Places<ROWS> at;
    pdl_launch_dependents();
    const int row0 = blockIdx.x * ROWS;
    pdl_wait();
    find_places<ROWS>(s, row0, at);
    __syncthreads();
    constexpr int kWords = DIM / 8;
    for (int i = threadIdx.x; i < ROWS * c.kv_heads * kWords; i += kThreads) {
        const int word = i % kWords, g = i / kWords % c.kv_heads, r = i / kWords / c.kv_heads;
        if (at.seq[r] < 0) continue;
        const bool held = at.position[r] >= 0;
        const size_t row = held ? cache_row(c, at.seq[r], g, at.position[r]) : 0;
#pragma unroll
        for (int side = 0; side < 2; side++) {
            const Rows<T>& o = side ? v : k;
            if (!o.p) continue;
            const uint32_t w = held ? reinterpret_cast<const uint32_t*>(side ? c.vc : c.kc)[row * kWords + word] : 0;
            const float2 p = held ? __half22float2((side ? c.vp : c.kp)[row * (DIM / 64) + word / 8]) : make_float2(0.f, 0.f);
            T* y = o.p + (size_t)(row0 + r) * o.ld + (size_t)g * DIM + word * 8;
#pragma unroll
            for (int h = 0; h < 8 / Vec<T>::n; h++) {
                Vec<T> x;
#pragma unroll
                for (int e = 0; e < Vec<T>::n; e++) {
                    const int i8 = h * Vec<T>::n + e;
                    x.v[e] = fmaf((float)((w >> (4 * (i8 >> 1) + 16 * (i8 & 1))) & 15), p.x, p.y);
                }
                x.store(y + h * Vec<T>::n);
            }
        }
    }
}

constexpr int kMany = 4, kManyFrom = 4 * 148;              // rows a CTA where the CTAs still fill the SMs

template <typename T, int DIM>
int append(const AppendArgs<T>& a, cudaStream_t stream)
{
    const unsigned parts = a.heads > 0 ? 2 : 1;
    if (a.s.tokens >= kManyFrom)
        return launch_pdl("cache4_append", cache4_append_kernel<T, DIM, kMany>, dim3((a.s.tokens + kMany - 1) / kMany, parts), dim3(kThreads), 0, stream, a);
    return launch_pdl("cache4_append", cache4_append_kernel<T, DIM, 1>, dim3(a.s.tokens, parts), dim3(kThreads), 0, stream, a);
}

template <typename T, int DIM>
int read(const Cache4& c, const Seqs& s, Rows<T> k, Rows<T> v, cudaStream_t stream)
{
    if (s.tokens >= kManyFrom)
        return launch_pdl("cache4_read", cache4_read_kernel<T, DIM, kMany>, dim3((s.tokens + kMany - 1) / kMany), dim3(kThreads), 0, stream, c, s, k, v);
    return launch_pdl("cache4_read", cache4_read_kernel<T, DIM, 1>, dim3(s.tokens), dim3(kThreads), 0, stream, c, s, k, v);
}

}  // namespace

template <typename T>
int launch_cache4_append(const Cache4& c, const Rotary& r, const Seqs& s, Rows<const T> q, Rows<T> q_out, int heads, Rows<const T> k, Rows<const T> v,
                         cudaStream_t stream)
{
    if (s.tokens == 0 || s.batch == 0) return TLLM_OK;
    const AppendArgs<T> a = {c, r, s, heads, q, k, v, q_out};
    return c.dim == 64 ? append<T, 64>(a, stream) : append<T, 128>(a, stream);
}

template <typename T>
int launch_cache4_read(const Cache4& c, const Seqs& s, Rows<T> k, Rows<T> v, cudaStream_t stream)
{
    if (s.tokens == 0 || s.batch == 0) return TLLM_OK;
    return c.dim == 64 ? read<T, 64>(c, s, k, v, stream) : read<T, 128>(c, s, k, v, stream);
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
