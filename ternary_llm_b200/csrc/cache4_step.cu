// Attention over the 4-bit key/value cache for few rows a sequence: one token of each, or a few.
//
// A key/value head's rows (new tokens times the query heads that share it, up to 4, 8 or 16 at once) go through the
// cache together on mma.sync.  With keys k = l + s c and values alike, scales and lowest values stay outside the products:
//   scores   sum_groups s (c . q) + l sum q   c . q in integers: codes, or codes times 16, are bytes after one mask, a
//            query is 16 bits of its largest entry in the group, as two signed bytes in neighbouring columns of the
//            product (m16n8k32), whose sums are joined exactly.  Positions are the rows of the product.
//   outputs  sum_p (w s) (c - 8) + sum_p w (l + 8 s)   codes are FP16 numbers after a mask and an addition or
//            multiplication for two, w s is rounded to FP16 (11 bits of it) and meets the difference from the middle of
//            the group's range; the second sum is FP32.  w s is in units of its row and group that follow the largest w |s| of
//            the positions that the row sees, so that a scale far above it without weight takes no bits: they are lost from
//            2^-20 of it on, in steps of 2^-30 of it.  Channels are the rows of the product (m16n8k16), columns the query
//            rows, or with up to four of them the four for the first and the four for the second group.
// Weights come out of the first product by position and go into the second as pairs of positions: movmatrix, an 8 x 8
// transposition in registers.  The running maximum moves when a score exceeds it by more than 2^8; sums are FP32.
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
constexpr float kSlack = 8.f, kLift = 64.f, kMost = 32768.f;          // kMost: of a weight times a scale in units, inside FP16
constexpr int kPad = 8;                                     // floats behind a row of a warp's outputs
constexpr float kDigits = 32512.f;                          // largest query entry in the integer product: 127 * 256

template <int DIM, int ROWS>
struct Step {
    static constexpr int kGroups = DIM / 64;
    static constexpr int kSets = ROWS / 4;                  // column tiles of the first product: four rows, two digits each
    static constexpr int kCols = ROWS == 4 ? 1 : ROWS / 8;  // column tiles of the second
    static constexpr int kSlots = 2;
    static constexpr int kCodes = kStepChunk * DIM / 2, kParams = kStepChunk * kGroups * 4;
    static constexpr int kSlot = 2 * (kCodes + kParams);    // keys' codes, values' codes, keys' params, values' params
    static constexpr int kOut = ROWS * (DIM + kPad);        // floats of a warp's outputs
    static constexpr int kSmem = kWarps * (kSlots * kSlot + (kOut + 2 * ROWS) * 4);
    // row of set n that lane t of a quad has in the sums of the first product
    static __device__ __forceinline__ int row(int n, int t) { return ROWS == 4 ? t : 8 * (n >> 1) + 2 * t + (n & 1); }
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
// Nibbles 0, 4 / 1, 5 / 2, 6 / 3, 7 less 8 as pairs of FP16 numbers: 1024 + c and 1024 + 16 c are bit patterns.
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t (&h)[4])
{
    const half2 one = halves(0x64086408u), sixteenth = halves(0x2c002c00u), off = halves(0xd480d480u);      // 1032, 1 / 16, -72
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
__device__ __forceinline__ void mma_u8s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// The largest of the eight lanes that hold a row.
__device__ __forceinline__ float row_max(float v)
{
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}

// The same of one or two numbers that are not negative, by their upper 16 bits.
template <int N>
__device__ __forceinline__ void row_max_upper(float (&v)[N])
{
    uint32_t x = __byte_perm(__float_as_uint(v[0]), __float_as_uint(v[N - 1]), 0x7632);
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) x = __vmaxu2(x, __shfl_xor_sync(0xffffffffu, x, d));
    v[0] = __uint_as_float(x << 16);
    v[N - 1] = __uint_as_float(x & 0xffff0000u);
}

// The power of two that takes v to kLift .. 2 kLift, for v of 2^-100 .. 2^30, and kLift divided by it (0 for 0).
__device__ __forceinline__ float unit_of(float v) { return __int_as_float(((260 - (__float_as_int(v) >> 23)) << 23)); }
__device__ __forceinline__ float unit_back(float unit) { return unit > 0.f ? unit_of(unit) : 0.f; }

// Rows of a product 0..7 as positions: lanes of a quad-strided read then fall on different banks, for keys (rows 0..3
// and 4..7 at once) and for values (even ones and odd ones at once).
__device__ __forceinline__ int place(int r) { return r < 4 ? r : r ^ 1; }
// 16-byte pieces of a row of 64 bytes, exchanged in every other pair of rows for the same reason.
template <int DIM> __device__ __forceinline__ int swizzle(int row) { return DIM == 128 ? row & 2 : 0; }

template <typename T, int DIM, int ROWS>
__global__ void __launch_bounds__(kThreads, ROWS == 16 ? 1 : 2)
cache4_step_kernel(const Cache4Call a, const Rows<const T> q, const Rows<T> out, const bool whole)
{
    using St = Step<DIM, ROWS>;
    constexpr int GR = St::kGroups, NS = St::kSets, NC = St::kCols, kStep = kWarps * kStepChunk;
    extern __shared__ __align__(16) uint8_t smem[];
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * St::kSlots * St::kSlot;
    float* outs = reinterpret_cast<float*>(smem + kWarps * St::kSlots * St::kSlot);
    float* stats = outs + kWarps * St::kOut;                               // [warp][m, l][row]
    const int per = a.heads / a.c.kv_heads;
    pdl_wait();

    __shared__ typename Work<ROWS, kStepChunk>::Start start;
    __shared__ uint32_t digits[NS * GR * 4][32];
    __shared__ float2 worth[NS * GR][4];
    Work<ROWS, kStepChunk> work(a.s, per, a.c.kv_heads, whole);
    if (warp == 0) work.find(blockIdx.x, gridDim.x, lane, &start);
    if (!whole && tid == 0) entry_of(a.ws, blockIdx.x)->parts = 0;
    __syncthreads();
    work.begin(start);
    const int to = work.to;

    int segment = 0;
    for (int x = work.x; x < to; segment++) {
        // ---- the next head's rows and the part of its chunks ----
        const int chunks = work.chunks, units = work.kFixed + chunks;
        const int j0 = whole ? 0 : work.chunk_at(work.offset), j1 = whole ? chunks : work.chunk_at(min(units, work.offset + (to - x)));
        x += whole ? 1 : units - work.offset;
        if (j0 == j1) {
            if (x < to) work.next();
            continue;
        }
        const int r0 = work.tile * ROWS, tile_rows = min(ROWS, work.rows - r0);
        const Span sp = work.span;
        const int visible = work.visible;                                  // positions that some row sees

        // a lane copies the same piece of every (32 / pieces of a row)-th row, and a row's params
        constexpr int kPieces = DIM / 32, kSpan = 32 / kPieces;
        const int my_row = lane / kPieces;
        const size_t first_row = cache_row(a.c, work.b, work.head, 0) + (size_t)(j0 + warp) * kStepChunk;
        const size_t code = (first_row + my_row) * (DIM / 2) + lane % kPieces * 16, par = (first_row + lane) * GR;
        const uint8_t *k_src = a.c.kc + code, *v_src = a.c.vc + code;
        const half2 *kp_src = a.c.kp + par, *vp_src = a.c.vp + par;
        const uint32_t to_codes = smem_addr(ring) + my_row * (DIM / 2) + ((lane % kPieces) ^ swizzle<DIM>(my_row)) * 16;
        const uint32_t to_params = smem_addr(ring) + 2 * St::kCodes + lane * 4 * GR;
        int issued = j0 + warp;
        const auto load = [&](int slot) {
            if (issued < j1) {
                const int left = visible - issued * kStepChunk;            // positions behind hold anything: nothing of them is read
                const uint32_t at = slot * St::kSlot;
                if (left >= kStepChunk) {
#pragma unroll
                    for (int i = 0; i < kPieces; i++) {
                        constexpr int kNext = kSpan * (DIM / 2);
                        copy_async<16>(to_codes + at + i * kNext, k_src + i * kNext, true);
                        copy_async<16>(to_codes + at + St::kCodes + i * kNext, v_src + i * kNext, true);
                    }
                    copy_async<4 * GR>(to_params + at, kp_src, true);
                    copy_async<4 * GR>(to_params + at + St::kParams, vp_src, true);
                } else {
#pragma unroll 1
                    for (int i = 0; i < kPieces; i++) {
                        const bool valid = my_row + i * kSpan < left;
                        const int off = i * kSpan * (DIM / 2);
                        copy_async<16>(to_codes + at + off, valid ? k_src + off : a.c.kc, valid);
                        copy_async<16>(to_codes + at + St::kCodes + off, valid ? v_src + off : a.c.vc, valid);
                    }
                    const bool valid = lane < left;
                    copy_async<4 * GR>(to_params + at, valid ? kp_src : a.c.kp, valid);
                    copy_async<4 * GR>(to_params + at + St::kParams, valid ? vp_src : a.c.vp, valid);
                }
                k_src += kStep * (DIM / 2);
                v_src += kStep * (DIM / 2);
                kp_src += kStep * GR;
                vp_src += kStep * GR;
            }
            issued += kWarps;
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < St::kSlots - 1; i++) load(i);

        // ---- the query rows: digits for the first product, their sums, what a unit of a digit is worth ----
        // A warp makes those of four rows and a group, all read them.
        for (int k = warp; k < NS * GR; k += kWarps) {
            const int n = k / GR, gr = k % GR, rr = St::row(n, g >> 1), r = r0 + rr;       // columns 2 i and 2 i + 1: digits of a row
            const bool there = rr < tile_rows;
            const T* qp = q.p + (size_t)(sp.row0 + (there ? r / per : 0)) * q.ld + (size_t)(work.head * per + (there ? r % per : 0)) * DIM + 64 * gr + 16 * t;
            float f[2][8], top = 0.f;
            bool odd = false;
            uint4 v[2];
#pragma unroll
            for (int w = 0; w < 2; w++) v[w] = there ? reinterpret_cast<const uint4*>(qp)[w] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < 2; w++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    f[w][i] = as_float(reinterpret_cast<const T*>(&v[w])[i]);
                    top = fmaxf(top, fabsf(f[w][i]));
                    odd = odd || !(fabsf(f[w][i]) < INFINITY);
                }
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                odd = __shfl_xor_sync(0xffffffffu, odd, d) || odd;
            }
            // sizes that a quotient of FP32 numbers can hold; smaller ones are zero in FP16 scores
            top = fmaxf(top, 1e-30f);
            const float by = kDigits / top;
            int total = 0;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                uint32_t b[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int x = odd ? 0 : __float2int_rn(f[w][i] * by), hi = (x + 128) >> 8;
                    total += x;
                    b[i] = (uint32_t)(g & 1 ? x - hi * 256 : hi) & 0xff;
                }
                // bytes as the codes lie in a word: low nibbles 0, 2, 4, 6 are entries 0, 4, 1, 5, high ones 2, 6, 3, 7
                digits[k * 4 + w][lane] = b[0] | b[4] << 8 | b[1] << 16 | b[5] << 24;
                digits[k * 4 + 2 + w][lane] = b[2] | b[6] << 8 | b[3] << 16 | b[7] << 24;
            }
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
            // a query that is not finite has no scores
            if (t == 0 && !(g & 1)) worth[k][g >> 1] = make_float2(16.f * (float)total, odd ? NAN : top / (16.f * kDigits) * (a.scale * 1.4426950408889634f));
        }
        __syncthreads();
        uint32_t qd[NS][GR][2][2];
        float qsum[NS][GR], unit_q[NS][GR];
        int sees[NS], least = INT_MAX;
#pragma unroll
        for (int n = 0; n < NS; n++) {
#pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                const int k = n * GR + gr;
#pragma unroll
                for (int w = 0; w < 4; w++) qd[n][gr][w >> 1][w & 1] = digits[k * 4 + w][lane];
                const float2 u = worth[k][t];
                qsum[n][gr] = u.x;
                unit_q[n][gr] = u.y;
            }
            const int rt = St::row(n, t);
            sees[n] = rt < tile_rows ? sp.position((r0 + rt) / per) + 1 : 0;
            if (rt < tile_rows) least = min(least, sees[n]);
        }
        least = min(least, __shfl_xor_sync(0xffffffffu, least, 1));
        least = min(least, __shfl_xor_sync(0xffffffffu, least, 2));        // every row of the tile sees so many positions

        float m[NS], ref[NS], l[NS], lo[NS][GR], o[NC][GR][4][4];          // ref: m, 0 before the first position
        float unit[NS][GR];                                                // what weights times scales of values are multiplied with, 0 before the first
#pragma unroll
        for (int n = 0; n < NS; n++) {
            m[n] = -INFINITY;
            ref[n] = l[n] = 0.f;
#pragma unroll
            for (int gr = 0; gr < GR; gr++) lo[n][gr] = unit[n][gr] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int gr = 0; gr < GR; gr++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[n][gr][i][e] = 0.f;

        int slot = 0;
#pragma unroll 1
        for (int j = j0 + warp; j < j1; j += kWarps) {
            load(slot == 0 ? St::kSlots - 1 : slot - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(St::kSlots - 1) : "memory");
            __syncwarp();
            const uint8_t* kc = ring + slot * St::kSlot;
            const uint8_t *vc = kc + St::kCodes, *kp = vc + St::kCodes, *vp = kp + St::kParams;
            const int p0 = j * kStepChunk;

            // ---- scores ----
            float s[NS][2][2];                                             // set, half of the chunk, row g or g + 8 of the product
            float2 vpar[2][2][GR];                                         // (s, l + 8 s) of values
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float2 par[2][GR];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int row = 16 * h + 8 * u + place(g);
                    uint32_t kw[GR], vw[GR];
                    if constexpr (GR == 2) {
                        const uint2 x2 = *reinterpret_cast<const uint2*>(kp + row * 8), y2 = *reinterpret_cast<const uint2*>(vp + row * 8);
                        kw[0] = x2.x, kw[1] = x2.y, vw[0] = y2.x, vw[1] = y2.y;
                    } else {
                        kw[0] = *reinterpret_cast<const uint32_t*>(kp + row * 4), vw[0] = *reinterpret_cast<const uint32_t*>(vp + row * 4);
                    }
#pragma unroll
                    for (int gr = 0; gr < GR; gr++) {
                        par[u][gr] = __half22float2(halves(kw[gr]));
                        vpar[h][u][gr] = __half22float2(halves(vw[gr]));
                        vpar[h][u][gr].y = fmaf(8.f, vpar[h][u][gr].x, vpar[h][u][gr].y);
                    }
                }
#pragma unroll
                for (int gr = 0; gr < GR; gr++) {
                    int low[NS][4] = {}, high[NS][4] = {};                  // of low nibbles, and of high ones sixteen times as large
                    uint2 w[2];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int row = 16 * h + 8 * u + place(g), piece = (2 * gr + (t >> 1)) ^ swizzle<DIM>(row);
                        w[u] = *reinterpret_cast<const uint2*>(kc + row * (DIM / 2) + piece * 16 + (t & 1) * 8);
                    }
#pragma unroll
                    for (int n = 0; n < NS; n++) {
                        mma_u8s8(low[n], w[0].x & 0x0f0f0f0fu, w[1].x & 0x0f0f0f0fu, w[0].y & 0x0f0f0f0fu, w[1].y & 0x0f0f0f0fu, qd[n][gr][0][0], qd[n][gr][0][1]);
                        mma_u8s8(high[n], w[0].x & 0xf0f0f0f0u, w[1].x & 0xf0f0f0f0u, w[0].y & 0xf0f0f0f0u, w[1].y & 0xf0f0f0f0u, qd[n][gr][1][0], qd[n][gr][1][1]);
                    }
#pragma unroll
                    for (int n = 0; n < NS; n++)
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const float dot = (float)(low[n][2 * u] * 4096 + low[n][2 * u + 1] * 16 + high[n][2 * u] * 256 + high[n][2 * u + 1]);
                            const float v = fmaf(par[u][gr].x, dot, par[u][gr].y * qsum[n][gr]);
                            s[n][h][u] = gr == 0 ? v * unit_q[n][gr] : fmaf(v, unit_q[n][gr], s[n][h][u]);
                        }
                }
            }
            if (p0 + kStepChunk > least) {
#pragma unroll
                for (int n = 0; n < NS; n++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int u = 0; u < 2; u++)
                            if (p0 + 16 * h + 8 * u + place(g) >= sees[n]) s[n][h][u] = -INFINITY;
            }
            // A row's maximum moves with its scores, its unit with its weights times scales; the largest of either says whether they may have to.
            bool grows = false;
            float scales[GR];
#pragma unroll
            for (int gr = 0; gr < GR; gr++) scales[gr] = fmaxf(fmaxf(fabsf(vpar[0][0][gr].x), fabsf(vpar[0][1][gr].x)), fmaxf(fabsf(vpar[1][0][gr].x), fabsf(vpar[1][1][gr].x)));
#pragma unroll
            for (int n = 0; n < NS; n++) {
                const float v = fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][1][0], s[n][1][1])), p = exp2_neg(v - ref[n]);
                grows = grows || v > m[n] + kSlack;
#pragma unroll
                for (int gr = 0; gr < GR; gr++) grows = grows || p * unit[n][gr] * scales[gr] > kMost;
            }
            if (__any_sync(0xffffffffu, grows)) {
                // each row by what it sees itself: its result does not depend on the others of the tile
#pragma unroll
                for (int n = 0; n < NS; n++) {
                    const float v = row_max(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][1][0], s[n][1][1])));
                    const bool up = v > m[n] + kSlack;
                    const float f = up ? exp2_neg(m[n] - v) : 1.f;
                    if (up) m[n] = ref[n] = v;
                    l[n] *= f;
                    float here[GR] = {};
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const float p = exp2_neg(s[n][h][u] - ref[n]);
#pragma unroll
                            for (int gr = 0; gr < GR; gr++) here[gr] = fmaxf(here[gr], p * fabsf(vpar[h][u][gr].x));
                        }
                    row_max_upper(here);
#pragma unroll
                    for (int gr = 0; gr < GR; gr++) {
                        const float most = here[gr];
                        float by = f;
                        if (up || most * unit[n][gr] > kMost) {
                            const float back = unit_back(unit[n][gr]), now = unit_of(fmaxf(fmaxf(back * f, most), 0x1p-100f));
                            by = f * (back * now * (1.f / kLift));
                            unit[n][gr] = now;
                        }
                        lo[n][gr] *= f;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            if constexpr (ROWS == 4) {
                                o[0][gr][k][gr] *= by;
                                o[0][gr][k][2 + gr] *= by;
                            } else {
                                o[n >> 1][gr][k][n & 1] *= by;
                                o[n >> 1][gr][k][2 + (n & 1)] *= by;
                            }
                        }
                    }
                }
            }

            // ---- weights, and outputs ----
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t pw[NC][GR][2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    float p[NS], ps[NS][GR];                               // weights; times the scales of values, in units
#pragma unroll
                    for (int n = 0; n < NS; n++) {
                        p[n] = exp2_neg(s[n][h][u] - ref[n]);
                        l[n] += p[n];
#pragma unroll
                        for (int gr = 0; gr < GR; gr++) {
                            ps[n][gr] = p[n] * (vpar[h][u][gr].x * unit[n][gr]);
                            lo[n][gr] = fmaf(p[n], vpar[h][u][gr].y, lo[n][gr]);
                        }
                    }
                    if constexpr (ROWS == 4) {
                        pw[0][0][u] = transposed(bits(__floats2half2_rn(ps[0][0], GR == 2 ? ps[0][GR - 1] : 0.f)));
#pragma unroll
                        for (int gr = 1; gr < GR; gr++) pw[0][gr][u] = pw[0][0][u];
                    } else {
#pragma unroll
                        for (int n = 0; n < NC; n++)
#pragma unroll
                            for (int gr = 0; gr < GR; gr++) pw[n][gr][u] = transposed(bits(__floats2half2_rn(ps[2 * n][gr], ps[2 * n + 1][gr])));
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
                    unpack8(__byte_perm(w[0], w[1], 0x5410), x0);
                    unpack8(__byte_perm(w[0], w[1], 0x7632), y0);
                    unpack8(__byte_perm(w[2], w[3], 0x5410), x1);
                    unpack8(__byte_perm(w[2], w[3], 0x7632), y1);
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int n = 0; n < NC; n++) mma_f16(o[n][gr][i], x0[i], y0[i], x1[i], y1[i], pw[n][gr][0], pw[n][gr][1]);
                }
            }
            slot = slot + 1 == St::kSlots ? 0 : slot + 1;
            __syncwarp();
        }
        asm volatile("cp.async.wait_all;" ::: "memory");

        // ---- the warps' parts of this head ----
#pragma unroll
        for (int n = 0; n < NS; n++) {
            const int r = St::row(n, t);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                l[n] += __shfl_xor_sync(0xffffffffu, l[n], d);
#pragma unroll
                for (int gr = 0; gr < GR; gr++) lo[n][gr] += __shfl_xor_sync(0xffffffffu, lo[n][gr], d);
            }
            if (g == 0) {
                stats[warp * 2 * ROWS + r] = m[n];
                stats[(warp * 2 + 1) * ROWS + r] = l[n];
            }
#pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                float* y = outs + warp * St::kOut + r * (DIM + kPad) + 64 * gr + 8 * g;
                const float back = unit_back(unit[n][gr]) * (1.f / kLift);
                const int nc = ROWS == 4 ? 0 : n >> 1, e = ROWS == 4 ? gr : n & 1;
#pragma unroll
                for (int k = 0; k < 4; k += 2)
                    *reinterpret_cast<float4*>(y + 2 * k) =
                        make_float4(fmaf(o[nc][gr][k][e], back, lo[n][gr]), fmaf(o[nc][gr][k][2 + e], back, lo[n][gr]),
                                    fmaf(o[nc][gr][k + 1][e], back, lo[n][gr]), fmaf(o[nc][gr][k + 1][2 + e], back, lo[n][gr]));
            }
        }
        __syncthreads();
        const bool complete = j0 == 0 && j1 == chunks;
        float* rec = complete ? nullptr : record_of<DIM, ROWS>(a.ws, gridDim.x, blockIdx.x, segment > 0);
        if (!complete && j0 == 0 && tid == 0)
            *entry_of(a.ws, blockIdx.x) = Shared4{work.owner(x - 1) - (int)blockIdx.x + 1, segment > 0, work.head, work.tile, sp.row0, sp.n, sp.len, 0};
        for (int e = tid; e < tile_rows * (DIM / 4); e += kThreads) {
            const int r = e / (DIM / 4), c = e % (DIM / 4) * 4;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; w++) top = fmaxf(top, stats[w * 2 * ROWS + r]);
            const float zero = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float f = exp2_neg(stats[w * 2 * ROWS + r] - zero);
                const float4 v = *reinterpret_cast<const float4*>(outs + w * St::kOut + r * (DIM + kPad) + c);
                sum = fmaf(stats[(w * 2 + 1) * ROWS + r], f, sum);
                y = make_float4(fmaf(v.x, f, y.x), fmaf(v.y, f, y.y), fmaf(v.z, f, y.z), fmaf(v.w, f, y.w));
            }
            if (complete) {
                const int i = (r0 + r) / per, head = work.head * per + (r0 + r) % per;
                store_row<T>(out.p + (size_t)(sp.row0 + i) * out.ld + (size_t)head * DIM + c, y, sum, sp.position(i) >= 0);
            } else {
                if (c == 0) {
                    rec[r] = top;
                    rec[ROWS + r] = sum;
                }
                *reinterpret_cast<float4*>(rec + 2 * ROWS + r * DIM + c) = y;
            }
        }
        __syncthreads();
        if (x < to) work.next();
    }
}

template <typename T, int DIM, int ROWS>
int launch(const Cache4Call& a, Rows<const T> q, Rows<T> out, const StepPlan& p, cudaStream_t stream)
{
    static bool attr[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return fail(TLLM_ERR_LAUNCH, "cache4_step: no current device");
    if (!attr[dev]) {
        cudaFuncSetAttribute(cache4_step_kernel<T, DIM, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Step<DIM, ROWS>::kSmem);
        attr[dev] = true;
    }
    int st = launch_pdl("cache4_step", cache4_step_kernel<T, DIM, ROWS>, dim3(p.ctas), dim3(kThreads), Step<DIM, ROWS>::kSmem, stream, a, q, out, p.whole);
    if (st || p.whole) return st;
    return launch_cache4_join<T>(a, out, ROWS, p.ctas, stream);
}

template <typename T, int DIM>
int launch_rows(const Cache4Call& a, Rows<const T> q, Rows<T> out, const StepPlan& p, cudaStream_t stream)
{
    return p.rows == 4 ? launch<T, DIM, 4>(a, q, out, p, stream) : p.rows == 8 ? launch<T, DIM, 8>(a, q, out, p, stream) : launch<T, DIM, 16>(a, q, out, p, stream);
}

}  // namespace

StepPlan step_plan(const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    StepPlan p;
    const long long rows = (long long)new_rows(c, tokens, max_new) * (heads / c.kv_heads);
    p.rows = rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
    const long long items = (long long)c.batch * c.kv_heads * ((rows + p.rows - 1) / p.rows);
    const int len = max_len > 0 && max_len < c.rows ? max_len : c.rows;
    // A tile's positions stay in one CTA while that takes no longer than a second launch and what it waits for.  Both ways, us, one / 48
    // sequences of 32 heads over 8, caches beyond L2 in turn: heads of 128 behind 300 6.3 / 15.3 in one CTA, 12.1 / 18.5 cut; behind 800 9.3 / 21.2, 12.3 /
    // 23.9; behind 1200 10.9 / 24.9, 12.8 / 27.9; behind 2000 14.5 / 34.2, 13.1 / 36.4; heads of 64 behind 2000 9.4 / 21.6, 11.1 / 24.1.
    p.whole = len <= kStepWhole / c.dim;
    // More than two such rounds of CTAs: one round, each with an equal number of tiles in a row, which saves what a CTA does before its first
    // tile, and costs where lengths differ.  One token each, 32 heads of 128 over 8, up to 800 positions, us, one round / a CTA a tile: equal
    // lengths 48 sequences 21.3 / 20.1, 96 31.9 / 35.0, 256 72.1 / 92.2; lengths between 1 and that 21.4 / 19.0, 29.9 / 27.3, 64.4 / 76.0;
    // 1024 of 8 heads over one 70 / 102.
    const int round = p.rows == 16 ? 148 : 296;
    p.ctas = p.whole && items <= 2 * round ? (int)items : round;
    p.bytes = p.whole ? 0 : join_bytes(c.dim, p.rows, p.ctas);
    return p;
}

template <typename T>
int launch_cache4_step(const Cache4Call& a, Rows<const T> q, Rows<T> out, const StepPlan& p, cudaStream_t stream)
{
    return a.c.dim == 64 ? launch_rows<T, 64>(a, q, out, p, stream) : launch_rows<T, 128>(a, q, out, p, stream);
}

template int launch_cache4_step<half>(const Cache4Call&, Rows<const half>, Rows<half>, const StepPlan&, cudaStream_t);
template int launch_cache4_step<bf16>(const Cache4Call&, Rows<const bf16>, Rows<bf16>, const StepPlan&, cudaStream_t);

}  // namespace tllm
