// Attention over the 4-bit key/value cache for few rows a sequence: one token of each, or a few.
//
// A key/value head's rows (new tokens times the query heads that share it, up to 8 or 16 at once) go through the
// cache together on mma.sync: codes become FP16 numbers 0..15 in registers (a mask, and one addition or
// multiplication for two), and the scales stay outside the products:
//   s_p,r   = scale sum_groups (s_p c_p . q_r + l_p sum q_r)      positions are the rows of the product, query rows its columns
//   o_r     = sum_p (w_p,r s_p) (c_p - 8) + sum_p w_p,r (l_p + 8 s_p)      channels are the rows; w s rounded to FP16
// so a code is never multiplied by its scale, keys enter exactly, and a value's only rounding is that of w s, 11
// bits of it (with a power of two that follows the largest scale seen, so that small scales do not run out of
// exponents); it meets the difference from the middle of the group's range.  The second sum is FP32.  Weights come out of the first product as pairs of query rows and go into the
// second as pairs of positions: movmatrix, an 8 x 8 transposition in registers.
//
// The running maximum moves when a score exceeds it by more than 2^8; sums are FP32.
//
// Work is cut into chunks of 32 positions.  All chunks of a call are one sequence of which every CTA takes an equal
// part, whatever the lengths; a warp takes every eighth of them, through a ring of its own (cp.async, no barrier).
// What the warps of a CTA find for a head meets in shared memory, what several CTAs find for one in records that a
// second launch joins, in order.
#include <climits>
#include <type_traits>

#include "cache4.cuh"
#include "cache4_work.cuh"
#include "dense.cuh"
#include "launch.cuh"

namespace tllm {

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr float kSlack = 8.f, kLift = 16.f;
constexpr int kPad = 8;                                     // floats behind a row of a warp's outputs

template <int DIM, int NT>
struct Step {
    static constexpr int kRows = 8 * NT, kGroups = DIM / 64;
    static constexpr int kSlots = 2;
    static constexpr int kCodes = kStepChunk * DIM / 2, kParams = kStepChunk * kGroups * 4;
    static constexpr int kSlot = 2 * (kCodes + kParams);    // keys' codes, values' codes, keys' params, values' params
    static constexpr int kOut = kRows * (DIM + kPad);       // floats of a warp's outputs
    static constexpr int kSmem = kWarps * (kSlots * kSlot + (kOut + 2 * kRows) * 4);
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool valid)
{
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(valid ? N : 0) : "memory");
}
__device__ __forceinline__ uint32_t bits(half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ half2 halves(uint32_t u) { return *reinterpret_cast<const half2*>(&u); }
// Nibbles 0, 4 / 1, 5 / 2, 6 / 3, 7 less MID as pairs of FP16 numbers: 1024 + c and 1024 + 16 c are bit patterns.
template <int MID>
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t (&h)[4])
{
    const half2 one = halves(MID ? 0x64086408u : 0x64006400u), sixteenth = halves(0x2c002c00u);              // 1024 + MID, 1 / 16
    const half2 off = halves(MID ? 0xd480d480u : 0xd400d400u);                                              // -(64 + MID)
    static_assert(MID == 0 || MID == 8, "constants above");
    const uint32_t v = w >> 8;
    h[0] = bits(__hsub2(halves((w & 0x000f000fu) | 0x64006400u), one));
    h[1] = bits(__hfma2(halves((w & 0x00f000f0u) | 0x64006400u), sixteenth, off));
    h[2] = bits(__hsub2(halves((v & 0x000f000fu) | 0x64006400u), one));
    h[3] = bits(__hfma2(halves((v & 0x00f000f0u) | 0x64006400u), sixteenth, off));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Rows of a product 0..7 as positions: lanes of a quad-strided read then fall on different banks, for keys (rows 0..3
// and 4..7 at once) and for values (even ones and odd ones at once).
__device__ __forceinline__ int place(int r) { return r < 4 ? r : r ^ 1; }
// 16-byte pieces of a row of 64 bytes, exchanged in every other pair of rows for the same reason.
template <int DIM> __device__ __forceinline__ int swizzle(int row) { return DIM == 128 ? row & 2 : 0; }

template <typename T, int DIM, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1)
cache4_step_kernel(const Cache4Call a, const Rows<const T> q, const Rows<T> out, const bool whole)
{
    using St = Step<DIM, NT>;
    constexpr int GR = St::kGroups;
    extern __shared__ __align__(16) uint8_t smem[];
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * St::kSlots * St::kSlot;
    float* outs = reinterpret_cast<float*>(smem + kWarps * St::kSlots * St::kSlot);
    float* stats = outs + kWarps * St::kOut;                               // [warp][m, l][row]
    const int per = a.heads / a.c.kv_heads;
    pdl_wait();

    if (blockIdx.x == 0 && warp == 0)
        for (int b = lane; b < a.s.batch; b += 32) span_of(a.s, b, true);
    Work<St::kRows, kStepChunk> work(a.s, per, a.c.kv_heads, whole, lane);
    const long long from = work.start(blockIdx.x, gridDim.x), to = work.start(blockIdx.x + 1, gridDim.x);
    if (from >= to) return;
    work.find(from, lane);
    int segment = 0;

    for (long long x = from; x < to; segment++) {
        // ---- the next head's rows and the part of its chunks ----
        const int chunks = work.chunks, j0 = whole ? 0 : work.offset, j1 = whole ? chunks : (int)min((long long)chunks, j0 + (to - x));
        const int tile_rows = min(St::kRows, work.rows - work.tile * St::kRows), r0 = work.tile * St::kRows;
        const Span sp = work.span;
        const size_t base = cache_row(a.c, work.b, work.head, 0);
        const int visible = work.visible;                                  // positions that some row sees

        const auto load = [&](int j, int slot) {
            const uint32_t at = smem_addr(ring + slot * St::kSlot);
            const int p0 = j * kStepChunk;
            constexpr int kPieces = DIM / 32;
#pragma unroll
            for (int i = 0; i < kPieces; i++) {
                const int e = i * 32 + lane, row = e / kPieces, c = e % kPieces;
                const bool valid = p0 + row < visible;
                const size_t src = (base + (valid ? p0 + row : 0)) * (DIM / 2) + c * 16;
                const uint32_t dst = at + row * (DIM / 2) + ((c ^ swizzle<DIM>(row)) * 16);
                copy_async<16>(dst, a.c.kc + src, valid);
                copy_async<16>(dst + St::kCodes, a.c.vc + src, valid);
            }
            const bool valid = p0 + lane < visible;
            const size_t src = (base + (valid ? p0 + lane : 0)) * GR;
            copy_async<4 * GR>(at + 2 * St::kCodes + lane * 4 * GR, a.c.kp + src, valid);
            copy_async<4 * GR>(at + 2 * St::kCodes + St::kParams + lane * 4 * GR, a.c.vp + src, valid);
        };
        int issued = j0 + warp;
#pragma unroll
        for (int i = 0; i < St::kSlots - 1; i++, issued += kWarps) {
            if (issued < j1) load(issued, i);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }

        // ---- the query rows: operands of the first product, sums by group, scales ----
        uint32_t qf[NT][GR][2][2][2];
        float qsum[NT][2][GR], col_scale[NT][2];
        int sees[NT][2], least = INT_MAX;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int r = r0 + 8 * n + g;
            const bool there = 8 * n + g < tile_rows;
            const T* qp = q.p + (size_t)(sp.row0 + (there ? r / per : 0)) * q.ld + (size_t)(work.head * per + (there ? r % per : 0)) * DIM;
            float top = 0.f, f[GR][2][8];
#pragma unroll
            for (int gr = 0; gr < GR; gr++)
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (there) v = *reinterpret_cast<const uint4*>(qp + 64 * gr + 16 * t + 8 * w);
                    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        f[gr][w][i] = as_float(e[i]);
                        top = fmaxf(top, fabsf(f[gr][w][i]));
                    }
                }
            // BF16 numbers become FP16 ones times a power of two of their row, the largest from 2^14 on
            float up = 1.f, down = 1.f;
            if constexpr (sizeof(T) == 2 && !std::is_same<T, half>::value) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = (__float_as_int(top) >> 23) - 127;
                if (top > 0.f && e < 128) {
                    const int sh = min(14 - e, 126);
                    up = __int_as_float((127 + sh) << 23);
                    down = __int_as_float((127 - sh) << 23);
                }
            }
            float sum[GR];
#pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                sum[gr] = 0.f;
#pragma unroll
                for (int w = 0; w < 2; w++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const half2 h = __floats2half2_rn(f[gr][w][4 * j + 2 * i] * up, f[gr][w][4 * j + 2 * i + 1] * up);
                            const float2 v = __half22float2(h);
                            qf[n][gr][w][j][i] = bits(h);
                            sum[gr] += v.x + v.y;
                        }
                sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 1);
                sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 2);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int src = 4 * (2 * t + i), rr = 8 * n + 2 * t + i;
                col_scale[n][i] = __shfl_sync(0xffffffffu, down, src) * a.scale * 1.4426950408889634f;
#pragma unroll
                for (int gr = 0; gr < GR; gr++) qsum[n][i][gr] = __shfl_sync(0xffffffffu, sum[gr], src);
                sees[n][i] = rr < tile_rows ? sp.position((r0 + rr) / per) + 1 : 0;
                if (rr < tile_rows) least = min(least, sees[n][i]);
            }
        }
        least = min(least, __shfl_xor_sync(0xffffffffu, least, 1));
        least = min(least, __shfl_xor_sync(0xffffffffu, least, 2));        // every row of the tile sees so many positions

        float m[NT][2], l[NT][2], lo[NT][2][GR], o[NT][GR][4][4];
        float largest = 0.f, unit = 0.f;                                   // power of two above every scale of values so far, kLift / it
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                m[n][i] = -INFINITY;
                l[n][i] = 0.f;
#pragma unroll
                for (int gr = 0; gr < GR; gr++) lo[n][i][gr] = 0.f;
            }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int gr = 0; gr < GR; gr++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[n][gr][i][e] = 0.f;

        int slot = 0;
#pragma unroll 1
        for (int j = j0 + warp; j < j1; j += kWarps) {
            if (issued < j1) load(issued, slot == 0 ? St::kSlots - 1 : slot - 1);
            issued += kWarps;
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group %0;" ::"n"(St::kSlots - 1) : "memory");
            __syncwarp();
            const uint8_t* kc = ring + slot * St::kSlot;
            const uint8_t *vc = kc + St::kCodes, *kp = vc + St::kCodes, *vp = kp + St::kParams;
            const int p0 = j * kStepChunk;

            // ---- scores ----
            float s[NT][2][4];
            bool grows = false;
            float2 vpar[2][2][GR];                                         // (s, l) of values: product, upper or lower rows, group
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float2 par[2][GR];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int row = 16 * h + 8 * u + place(g);
#pragma unroll
                    for (int gr = 0; gr < GR; gr++) {
                        par[u][gr] = __half22float2(reinterpret_cast<const half2*>(kp)[row * GR + gr]);
                        vpar[h][u][gr] = __half22float2(reinterpret_cast<const half2*>(vp)[row * GR + gr]);
                        vpar[h][u][gr].y = fmaf(8.f, vpar[h][u][gr].x, vpar[h][u][gr].y);
                        grows = grows || vpar[h][u][gr].x > largest;
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[n][h][e] = 0.f;
#pragma unroll
                for (int gr = 0; gr < GR; gr++) {
                    float acc[NT][4] = {};
                    uint2 w[2];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int row = 16 * h + 8 * u + place(g), piece = (2 * gr + (t >> 1)) ^ swizzle<DIM>(row);
                        w[u] = *reinterpret_cast<const uint2*>(kc + row * (DIM / 2) + piece * 16 + (t & 1) * 8);
                    }
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        uint32_t x[4], y[4];
                        unpack8<0>(i ? w[0].y : w[0].x, x);
                        unpack8<0>(i ? w[1].y : w[1].x, y);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            mma_f16(acc[n], x[0], y[0], x[1], y[1], qf[n][gr][i][0][0], qf[n][gr][i][0][1]);
                            mma_f16(acc[n], x[2], y[2], x[3], y[3], qf[n][gr][i][1][0], qf[n][gr][i][1][1]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            s[n][h][e] = fmaf(par[e >> 1][gr].x, acc[n][e], fmaf(par[e >> 1][gr].y, qsum[n][e & 1][gr], s[n][h][e]));
                }
            }
            const bool masked = p0 + kStepChunk > least;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        s[n][h][e] *= col_scale[n][e & 1];
                        if (masked && p0 + 16 * h + 8 * (e >> 1) + place(g) >= sees[n][e & 1]) s[n][h][e] = -INFINITY;
                        grows = grows || s[n][h][e] > m[n][e & 1] + kSlack;
                    }
            if (__any_sync(0xffffffffu, grows)) {
                float top = largest;
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int gr = 0; gr < GR; gr++) top = fmaxf(top, vpar[h][u][gr].x);
                top = warp_max(top);
                if (top > largest) top = __int_as_float(((__float_as_int(top) >> 23) + 1) << 23);
                const float shrink = top > largest ? largest / top : 1.f;
                largest = top;
                unit = top > 0.f ? kLift / top : 0.f;
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        float x = fmaxf(fmaxf(s[n][0][i], s[n][0][2 + i]), fmaxf(s[n][1][i], s[n][1][2 + i]));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                        const float f = x > m[n][i] ? exp2_neg(m[n][i] - x) : 1.f;
                        m[n][i] = fmaxf(m[n][i], x);
                        l[n][i] *= f;
#pragma unroll
                        for (int gr = 0; gr < GR; gr++) {
                            lo[n][i][gr] *= f;
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                o[n][gr][k][i] *= f * shrink;
                                o[n][gr][k][2 + i] *= f * shrink;
                            }
                        }
                    }
            }

            // ---- weights, and outputs ----
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t pw[NT][GR][2];
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        float p[2];
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            p[i] = exp2_neg(s[n][h][2 * u + i] - (m[n][i] == -INFINITY ? 0.f : m[n][i]));
                            l[n][i] += p[i];
                        }
#pragma unroll
                        for (int gr = 0; gr < GR; gr++) {
                            const float2 par = vpar[h][u][gr];
                            const float f = par.x * unit;
                            lo[n][0][gr] = fmaf(p[0], par.y, lo[n][0][gr]);
                            lo[n][1][gr] = fmaf(p[1], par.y, lo[n][1][gr]);
                            pw[n][gr][u] = transposed(bits(__floats2half2_rn(p[0] * f, p[1] * f)));
                        }
                    }
#pragma unroll
                for (int gr = 0; gr < GR; gr++) {
                    uint32_t w[4];                                         // positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of the product
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int row = 16 * h + 8 * (k >> 1) + place(2 * t + (k & 1)), piece = (2 * gr + (g >> 2)) ^ swizzle<DIM>(row);
                        w[k] = *reinterpret_cast<const uint32_t*>(vc + row * (DIM / 2) + piece * 16 + (g & 3) * 4);
                    }
                    uint32_t x0[4], y0[4], x1[4], y1[4];                   // channels 8 g + 2 i and 8 g + 2 i + 1 of two positions each
                    unpack8<8>(__byte_perm(w[0], w[1], 0x5410), x0);
                    unpack8<8>(__byte_perm(w[0], w[1], 0x7632), y0);
                    unpack8<8>(__byte_perm(w[2], w[3], 0x5410), x1);
                    unpack8<8>(__byte_perm(w[2], w[3], 0x7632), y1);
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int n = 0; n < NT; n++) mma_f16(o[n][gr][i], x0[i], y0[i], x1[i], y1[i], pw[n][gr][0], pw[n][gr][1]);
                }
            }
            slot = slot + 1 == St::kSlots ? 0 : slot + 1;
            __syncwarp();
        }
        asm volatile("cp.async.wait_all;" ::: "memory");

        // ---- the warps' parts of this head ----
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int r = 8 * n + 2 * t + i;
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], d);
#pragma unroll
                    for (int gr = 0; gr < GR; gr++) lo[n][i][gr] += __shfl_xor_sync(0xffffffffu, lo[n][i][gr], d);
                }
                if (g == 0) {
                    stats[warp * 2 * St::kRows + r] = m[n][i];
                    stats[(warp * 2 + 1) * St::kRows + r] = l[n][i];
                }
#pragma unroll
                for (int gr = 0; gr < GR; gr++) {
                    float* y = outs + warp * St::kOut + r * (DIM + kPad) + 64 * gr + 8 * g;
                    const float back = largest / kLift;
#pragma unroll
                    for (int k = 0; k < 4; k += 2)
                        *reinterpret_cast<float4*>(y + 2 * k) =
                            make_float4(fmaf(o[n][gr][k][i], back, lo[n][i][gr]), fmaf(o[n][gr][k][2 + i], back, lo[n][i][gr]),
                                        fmaf(o[n][gr][k + 1][i], back, lo[n][i][gr]), fmaf(o[n][gr][k + 1][2 + i], back, lo[n][i][gr]));
                }
            }
        __syncthreads();
        const bool complete = j0 == 0 && j1 == chunks;
        float* rec = complete ? nullptr : static_cast<float*>(a.ws) + ((size_t)blockIdx.x * 2 + (segment > 0)) * kRecord<DIM, St::kRows>;
        for (int e = tid; e < tile_rows * (DIM / 4); e += kThreads) {
            const int r = e / (DIM / 4), c = e % (DIM / 4) * 4;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; w++) top = fmaxf(top, stats[w * 2 * St::kRows + r]);
            const float ref = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float f = exp2_neg(stats[w * 2 * St::kRows + r] - ref);
                const float4 v = *reinterpret_cast<const float4*>(outs + w * St::kOut + r * (DIM + kPad) + c);
                sum = fmaf(stats[(w * 2 + 1) * St::kRows + r], f, sum);
                y = make_float4(fmaf(v.x, f, y.x), fmaf(v.y, f, y.y), fmaf(v.z, f, y.z), fmaf(v.w, f, y.w));
            }
            if (complete) {
                const int i = (r0 + r) / per, head = work.head * per + (r0 + r) % per;
                store_row<T>(out.p + (size_t)(sp.row0 + i) * out.ld + (size_t)head * DIM + c, y, sum, sp.position(i) >= 0);
            } else {
                if (c == 0) {
                    rec[r] = top;
                    rec[St::kRows + r] = sum;
                }
                *reinterpret_cast<float4*>(rec + 2 * St::kRows + r * DIM + c) = y;
            }
        }
        __syncthreads();
        x += whole ? 1 : j1 - j0;
        if (x < to) work.next();
    }
}

template <typename T, int DIM, int NT>
int launch(const Cache4Call& a, Rows<const T> q, Rows<T> out, const StepPlan& p, cudaStream_t stream)
{
    using St = Step<DIM, NT>;
    static bool attr[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return fail(TLLM_ERR_LAUNCH, "cache4_step: no current device");
    if (!attr[dev]) {
        cudaFuncSetAttribute(cache4_step_kernel<T, DIM, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, St::kSmem);
        attr[dev] = true;
    }
    int st = launch_pdl("cache4_step", cache4_step_kernel<T, DIM, NT>, dim3(p.ctas), dim3(kThreads), St::kSmem, stream, a, q, out, p.whole);
    if (st || p.whole) return st;
    return launch_cache4_join<T>(a, out, St::kRows, p.ctas, p.items, stream);
}

}  // namespace

// Rows of a tile: 8, or 16 where that saves a walk over the cache.
StepPlan step_plan(const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    StepPlan p;
    const int per = heads / c.kv_heads, most = max_new > 0 ? max_new : (tokens + c.batch - 1) / (c.batch > 0 ? c.batch : 1);
    const long long rows = (long long)most * per;
    p.tiles = rows > 8 ? 2 : 1;
    const long long items = (long long)c.batch * c.kv_heads * ((rows + 8 * p.tiles - 1) / (8 * p.tiles));
    p.items = (int)(items < 1 ? 1 : items < 65536 ? items : 65536);
    const int len = max_len > 0 && max_len < c.rows ? max_len : c.rows;
    const int at_once = p.tiles == 1 ? 296 : 148;
    p.whole = len <= 512;
    p.ctas = p.whole ? p.items : at_once;
    p.bytes = p.whole ? 0 : (size_t)p.ctas * 2 * (size_t)(8 * p.tiles) * (c.dim + 2) * sizeof(float);
    return p;
}

template <typename T>
int launch_cache4_step(const Cache4Call& a, Rows<const T> q, Rows<T> out, const StepPlan& p, cudaStream_t stream)
{
    if (a.c.dim == 64) return p.tiles == 1 ? launch<T, 64, 1>(a, q, out, p, stream) : launch<T, 64, 2>(a, q, out, p, stream);
    return p.tiles == 1 ? launch<T, 128, 1>(a, q, out, p, stream) : launch<T, 128, 2>(a, q, out, p, stream);
}

template int launch_cache4_step<half>(const Cache4Call&, Rows<const half>, Rows<half>, const StepPlan&, cudaStream_t);
template int launch_cache4_step<bf16>(const Cache4Call&, Rows<const bf16>, Rows<bf16>, const StepPlan&, cudaStream_t);

}  // namespace tllm
