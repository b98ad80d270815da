// Rotary positions of queries and keys: (x1, x2) -> a (x1 cos - x2 sin, x2 cos + x1 sin) for the pairs of a
// head's first entries, and the frequencies of long contexts (on the host).
#include <cmath>

#include "cache4.cuh"
#include "launch.cuh"

namespace tllm {

namespace {

constexpr int kThreads = 256;

template <typename T>
struct RotaryArgs {
    Rotary r;
    const int* positions;
    int tokens, heads, kv_heads, dim;
    Rows<const T> q, k;
    Rows<T> q_out, k_out;
};

// A pair, or an entry that does not turn, a thread: half layouts whose pairs are no whole 16-byte units.
template <typename T>
__global__ void __launch_bounds__(kThreads)
rotary_pairs_kernel(const RotaryArgs<T> a)
{
    pdl_launch_dependents();
    pdl_wait();
    const int pairs = a.r.rot / 2, per_head = a.dim - pairs;
    const int row = blockIdx.x, position = a.positions[row];
    for (int i = threadIdx.x; i < (a.heads + a.kv_heads) * per_head; i += kThreads) {
        const int h = i / per_head, e = i % per_head;
        const bool is_q = h < a.heads;
        const size_t at = is_q ? (size_t)h * a.dim : (size_t)(h - a.heads) * a.dim;
        const T* x = is_q ? a.q.p + (size_t)row * a.q.ld + at : a.k.p + (size_t)row * a.k.ld + at;
        T* y = is_q ? a.q_out.p + (size_t)row * a.q_out.ld + at : a.k_out.p + (size_t)row * a.k_out.ld + at;
        if (e >= pairs) {
            y[e + pairs] = x[e + pairs];
            continue;
        }
        const int i1 = a.r.half_layout ? e : 2 * e, i2 = a.r.half_layout ? e + pairs : 2 * e + 1;
        float2 c;
        turn(a.r, a.r.turns[e], position, c.x, c.y);
        const float x1 = as_float(x[i1]), x2 = as_float(x[i2]);
        y[i1] = as_type<T>(turned_first(x1, x2, c));
        y[i2] = as_type<T>(turned_second(x1, x2, c));
    }
}

// ROWS rows a CTA: the angles of their positions once for all heads, in shared memory, while the first units are on their way; then a thread
// takes a unit of a head for all rows, so that ROWS or twice as many loads of 16 bytes are in flight.  Bound by the bytes: 8192 rows of
// 40 BF16 heads of 128 take 35 us (168 MB, 4.8 TB/s) two rows at once, 39 four, 49 eight.
template <typename T, int ROWS>
__global__ void __launch_bounds__(kThreads)
rotary_kernel(const RotaryArgs<T> a)
{
    __shared__ float2 cs[ROWS][256];
    pdl_launch_dependents();
    const int tid = threadIdx.x, row0 = blockIdx.x * ROWS, rows = min(ROWS, a.tokens - row0);
    const Turn<T> t(a.r, a.dim);
    const int units = (a.heads + a.kv_heads) * t.per_head;
    int h = tid / t.per_head, u = tid % t.per_head;
    const int threads = blockDim.x, step_h = threads / t.per_head, step_u = threads % t.per_head;
    pdl_wait();
    uint4 w[ROWS][2];
    const auto load = [&] {
        const bool is_q = h < a.heads;
        const T* x = is_q ? a.q.p + (size_t)h * a.dim : a.k.p + (size_t)(h - a.heads) * a.dim;
        const long long ld = is_q ? a.q.ld : a.k.ld;
#pragma unroll
        for (int r = 0; r < ROWS; r++)
            if (r < rows) t.load(x + (row0 + r) * ld, u, w[r]);
    };
    if (tid < units) load();
    for (int i = tid; i < rows * t.pairs; i += threads) {
        const int r = i / t.pairs, p = i % t.pairs;
        turn(a.r, a.r.turns[p], a.positions[row0 + r], cs[r][p].x, cs[r][p].y);
    }
    __syncthreads();
    for (int i = tid; i < units; i += threads) {
        if (i != tid) load();
        const bool is_q = h < a.heads;
        T* y = is_q ? a.q_out.p + (size_t)h * a.dim : a.k_out.p + (size_t)(h - a.heads) * a.dim;
        const long long ld = is_q ? a.q_out.ld : a.k_out.ld;
#pragma unroll
        for (int r = 0; r < ROWS; r++)
            if (r < rows) t.turn_and_store(y + (row0 + r) * ld, u, w[r], cs[r]);
        h += step_h;
        u += step_u;
        if (u >= t.per_head) {
            u -= t.per_head;
            h++;
        }
    }
}

}  // namespace

template <typename T>
int launch_rotary(const Rotary& r, const int* positions, int tokens, Rows<const T> q, Rows<T> q_out, int heads, Rows<const T> k, Rows<T> k_out,
                  int kv_heads, int dim, cudaStream_t stream)
{
    if (tokens == 0 || heads + kv_heads == 0) return TLLM_OK;
    const RotaryArgs<T> a = {r, positions, tokens, heads, kv_heads, dim, q, k, q_out, k_out};
    if (!Turn<T>::whole(r)) return launch_pdl("rotary", rotary_pairs_kernel<T>, dim3(tokens), dim3(kThreads), 0, stream, a);
    // equal passes over the units; rows together where the CTAs still fill the SMs
    const int units = (heads + kv_heads) * Turn<T>(r, dim).per_head, passes = (units + kThreads - 1) / kThreads;
    const int threads = ((units + passes - 1) / passes + 31) / 32 * 32;
    if (tokens >= 4 * 148) return launch_pdl("rotary", rotary_kernel<T, 2>, dim3((tokens + 1) / 2), dim3(threads), 0, stream, a);
    return launch_pdl("rotary", rotary_kernel<T, 1>, dim3(tokens), dim3(threads), 0, stream, a);
}

#define TLLM_INSTANTIATE(T) \
    template int launch_rotary<T>(const Rotary&, const int*, int, Rows<const T>, Rows<T>, int, Rows<const T>, Rows<T>, int, int, cudaStream_t);
TLLM_INSTANTIATE(half)
TLLM_INSTANTIATE(bf16)
TLLM_INSTANTIATE(float)
#undef TLLM_INSTANTIATE

}  // namespace tllm

extern "C" {

using namespace tllm;

int tllm_b200_rotary_frequencies(int rot_dim, double base, const tllm_b200_rotary_scaling* scaling, double* frequencies_host, float* amplitude_host)
{
    if (!frequencies_host || !amplitude_host) return fail(TLLM_ERR_NULL, "rotary_frequencies: null pointer");
    const tllm_b200_rotary_scaling none = {TLLM_ROTARY_PLAIN, 1, 1, 1, 1};
    const tllm_b200_rotary_scaling& s = scaling ? *scaling : none;
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > 512 || !(base > 1.0) || !std::isfinite(base))
        return fail(TLLM_ERR_SHAPE, "rotary_frequencies: rot_dim=%d base=%g", rot_dim, base);
    if (s.type < TLLM_ROTARY_PLAIN || s.type > TLLM_ROTARY_LLAMA3) return fail(TLLM_ERR_SHAPE, "rotary_frequencies: scaling type %d", s.type);
    if (s.type != TLLM_ROTARY_PLAIN && (!(s.factor >= 1.0) || !std::isfinite(s.factor)))
        return fail(TLLM_ERR_SHAPE, "rotary_frequencies: factor %g is not 1 or more", s.factor);
    if (s.type >= TLLM_ROTARY_YARN && (!(s.original >= 1.0) || !(s.low > 0.0) || !(s.high > s.low) || !std::isfinite(s.original) || !std::isfinite(s.high)))
        return fail(TLLM_ERR_SHAPE, "rotary_frequencies: original=%g low=%g high=%g", s.original, s.low, s.high);
    if (s.type == TLLM_ROTARY_NTK) {
        if (rot_dim < 4) return fail(TLLM_ERR_SHAPE, "rotary_frequencies: rot_dim=%d", rot_dim);
        base *= std::pow(s.factor, (double)rot_dim / (rot_dim - 2));
    }
    const double tau = 6.283185307179586476925286766559;
    // the pair that turns so many times over the original length
    auto pair_of = [&](double turns) { return rot_dim * std::log(s.original / (turns * tau)) / (2 * std::log(base)); };
    double from = 0, to = 0;
    if (s.type == TLLM_ROTARY_YARN) {
        from = std::fmax(std::floor(pair_of(s.high)), 0.0);
        to = std::fmin(std::ceil(pair_of(s.low)), rot_dim - 1.0);
    }
    for (int i = 0; i < rot_dim / 2; i++) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (s.type == TLLM_ROTARY_LINEAR) {
            f /= s.factor;
        } else if (s.type == TLLM_ROTARY_YARN) {
            const double ramp = std::fmin(std::fmax((i - from) / std::fmax(to - from, 0.001), 0.0), 1.0);
            f = f / s.factor * ramp + f * (1 - ramp);
        } else if (s.type == TLLM_ROTARY_LLAMA3) {
            const double mix = std::fmin(std::fmax((s.original * f / tau - s.low) / (s.high - s.low), 0.0), 1.0);
            f = (1 - mix) * f / s.factor + mix * f;
        }
        frequencies_host[i] = f;
    }
    *amplitude_host = s.type == TLLM_ROTARY_YARN ? (float)(0.1 * std::log(s.factor) + 1.0) : 1.f;
    return TLLM_OK;
}

int tllm_b200_rotary_turns(const double* frequencies_host, int pairs, unsigned long long* turns_host)
{
    if (!frequencies_host || !turns_host) return fail(TLLM_ERR_NULL, "rotary_turns: null pointer");
    if (pairs < 1) return fail(TLLM_ERR_SHAPE, "rotary_turns: pairs=%d", pairs);
    for (int i = 0; i < pairs; i++) {
        if (!std::isfinite(frequencies_host[i])) return fail(TLLM_ERR_SHAPE, "rotary_turns: frequency %d is %g", i, frequencies_host[i]);
        // 1 / (2 pi) in 64 bits and more; the whole turns of a position do not count
        long double t = (long double)frequencies_host[i] * 0.159154943091895335768883763372514362L;
        t -= std::floor(t);
        const long double units = std::nearbyint(t * 18446744073709551616.0L);
        turns_host[i] = units >= 18446744073709551616.0L ? 0ull : (unsigned long long)units;
    }
    return TLLM_OK;
}

}  // extern "C"
