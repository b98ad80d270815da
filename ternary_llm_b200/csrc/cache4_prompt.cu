// Attention over the 4-bit key/value cache for many rows a sequence, on the 5th-generation tensor cores.
//
// A CTA takes 256 rows of a key/value head (new tokens times the query heads that share it) as two tiles of 128 and
// walks over tiles of 128 positions.  Roles: four warps turn the codes of a tile into FP16 numbers in shared memory,
// rounded once (l + s c, 11 bits); one warp issues tcgen05.mma; four warps for each tile of rows have a row a thread.
//   S = Q K^T    both operands in shared memory, 128 FP32 columns of tensor memory for each tile of rows
//   softmax      a thread reads its row; the weights go back over S as FP16, with a factor of 2^6 that leaves small
//                ones their bits (the sum of the weights takes it out)
//   O += P V     weights from tensor memory, values feature-major
// so a tile of the cache is unpacked once for 256 rows, and one tile's products run beside the other's softmax.
// BF16 queries become FP16 numbers times a power of two of their row.  The running maximum moves when it grows by more
// than 2^8; sums are FP32.  A position that a row does not see is masked before the maximum, and values are finite
// (append marks a NaN in the key), so nothing behind a row's own position reaches it.
//
// Work: tiles of rows, longest first; or, where there are too few, all tiles of positions as one sequence of which
// every CTA takes an equal part, parts of a tile of rows joined by a second launch in their order.
// All mbarrier waits are bounded.
#include <type_traits>

#include "cache4.cuh"
#include "cache4_work.cuh"
#include "dense.cuh"
#include "f32x2.cuh"
#include "launch.cuh"
#include "tcgen05.cuh"

namespace tllm {

namespace {

using namespace gemm;

constexpr int kTile = kPromptChunk, kRows = kPromptRows, kRowTiles = kRows / kTile;
constexpr int kThreads = 512;                        // row tiles' softmax 0-3, 4-7, unpacking 8-11, products 12
constexpr int kBlock = kTile * 128;                  // bytes of 64 columns of a tile: 128-byte rows
constexpr int kStages = 2;
constexpr float kSlack = 8.f, kLift = 6.f, kLog2e = 1.4426950408889634f;

template <int DIM>
struct Prompt {
    static constexpr int kBlocks = DIM / 64;
    static constexpr int kOperand = kBlocks * kBlock;                              // bytes of a tile
    static constexpr int kSmem = (kRowTiles + 2 * kStages) * kOperand + 1024;
    static constexpr uint32_t kTmemCols = kRowTiles * (kTile + DIM) <= 384 && kRowTiles * (kTile + DIM) > 256 ? 512 : kRowTiles * (kTile + DIM);
};

__device__ __forceinline__ uint32_t idesc(int n, bool feature_major)
{
    return (1u << 4) | ((feature_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
// operand whose rows are the contracted index: blocks of 64 features kBlock apart, groups of 8 rows 1024 bytes apart
__device__ __forceinline__ uint64_t feature_major_desc(uint32_t addr)
{
    return (make_sw128_desc(addr) & ~((uint64_t)0x3fff << 16)) | ((uint64_t)(kBlock >> 4) << 16);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc)
{
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc)
{
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }"
        ::"r"(d), "r"(a), "l"(b), "r"(id), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                 "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                 "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// A tile's rows of a key/value head and the tiles of positions [j0, j1) of its `chunks`, one after the other for this CTA;
// every role walks over the same.
struct Walk : Work<kRows, kTile> {
    long long x, to;
    int from_top, step, j0, j1, segment;
    __device__ __forceinline__ Walk(const Cache4Call& a, bool whole_, int lane) : Work(a.s, a.heads / a.c.kv_heads, a.c.kv_heads, whole_, lane), segment(-1)
    {
        if (whole) {
            const int pairs = s.batch * kv_heads;
            from_top = (int)(blockIdx.x / pairs);
            step = max((int)gridDim.x / pairs, 1);
            b = (int)(blockIdx.x % pairs) / kv_heads;
            head = (int)(blockIdx.x % pairs) % kv_heads;
            span = span_of(s, b, false);
            rows = span.n * per;
            from_top -= step;
        } else {
            x = start(blockIdx.x, gridDim.x);
            to = start(blockIdx.x + 1, gridDim.x);
            if (x < to) find(x, lane);
        }
    }
    __device__ __forceinline__ bool advance()
    {
        segment++;
        if (whole) {
            from_top += step;
            const int tl = (rows + kRows - 1) / kRows - 1 - from_top;
            if (tl < 0) return false;
            set_tile(tl);
            j0 = 0;
            j1 = chunks;
            return true;
        }
        if (x >= to) return false;
        if (segment > 0) next();
        j0 = offset;
        j1 = (int)min((long long)chunks, j0 + (to - x));
        x += j1 - j0;
        return true;
    }
    __device__ __forceinline__ bool complete() const { return j0 == 0 && j1 == chunks; }
    __device__ __forceinline__ int tile_rows(int i) const { return min(kTile, rows - tile * kRows - i * kTile); }
};

enum Bar { kQFull = 0, kKFull = 2, kKEmpty = 4, kVFull = 6, kVEmpty = 8, kSFull = 10, kPReady = 12, kPvDone = 14, kLast = 16, kBars = 17 };

template <typename T, int DIM>
__global__ void __launch_bounds__(kThreads, 1)
cache4_prompt_kernel(const Cache4Call a, const Rows<const T> q, const Rows<T> out, const bool whole)
{
    using P = Prompt<DIM>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t bars[kBars];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t *qs = smem, *ks = qs + kRowTiles * P::kOperand, *vs = ks + kStages * P::kOperand;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    volatile int* abortp = &abort_flag;
    int never = 0;

    if (tid == 0) {
        for (int i = 0; i < kBars; i++) {
            const bool by_threads = i < kKFull || i / 2 * 2 == kKFull || i / 2 * 2 == kVFull || i / 2 * 2 == kPReady;
            mbar_init(bar(i), by_threads ? kTile : 1);
        }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(P::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;                                       // S of both tiles of rows, then O of both
    pdl_wait();
    if (blockIdx.x == 0 && warp == 13)
        for (int b = lane; b < a.s.batch; b += 32) span_of(a.s, b, true);

    if (warp >= 12) {
        fewer_registers<56>();
        if (warp == 12) {
            // ---------------- products ----------------
            const bool leader = elect_one();
            const uint32_t id_s = idesc(kTile, false), id_o = idesc(DIM, true);
            Walk w(a, whole, lane);
            uint32_t n = 0, items[2] = {0, 0}, rounds[2] = {0, 0};         // tiles of positions so far; by tile of rows: segments, weights
            bool ok = true;
            // S of tile of rows i against the tile of positions in stage st
            auto scores = [&](int i, uint32_t st) {
                fence_after();
                if (leader) {
                    const uint64_t qd = make_sw128_desc(smem_u32(qs + i * P::kOperand)), kd = make_sw128_desc(smem_u32(ks + st * P::kOperand));
#pragma unroll
                    for (int j = 0; j < P::kBlocks; j++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint32_t o = j * (kBlock >> 4) + k * 2;
                            mma_ss(tmem + i * kTile, qd + o, kd + o, id_s, j > 0 || k > 0);
                        }
                    mma_commit(bar(kSFull + i));
                }
            };
            while (ok && w.advance()) {
                const int active = w.tile_rows(1) > 0 ? 2 : 1, tiles = w.j1 - w.j0;
                ok = mbar_wait(bar(kKFull + (n & 1)), (n >> 1) & 1, abortp);
                for (int i = 0; ok && i < active; i++) {
                    if (!(ok = mbar_wait(bar(kQFull + i), items[i]++ & 1, abortp))) break;
                    scores(i, n & 1);
                }
                if (ok && leader) mma_commit(bar(kKEmpty + (n & 1)));
                for (int j = 0; ok && j < tiles; j++, n++) {
                    const uint32_t st = n & 1, next = st ^ 1;
                    ok = mbar_wait(bar(kVFull + st), (n >> 1) & 1, abortp);
                    for (int i = 0; ok && i < active; i++) {
                        if (!(ok = mbar_wait(bar(kPReady + i), rounds[i] & 1, abortp))) break;
                        fence_after();
                        if (leader) {
                            const uint64_t vd = feature_major_desc(smem_u32(vs + st * P::kOperand));
#pragma unroll
                            for (int k = 0; k < kTile / 16; k++)
                                mma_ts(tmem + kRowTiles * kTile + i * DIM, tmem + i * kTile + k * 8, vd + k * (2048 >> 4), id_o, j > 0 || k > 0);
                            mma_commit(bar(kPvDone + i));
                        }
                        if (j + 1 < tiles) {
                            // the weights lie where the next scores go
                            ok = (i > 0 || mbar_wait(bar(kKFull + next), ((n + 1) >> 1) & 1, abortp)) && mbar_wait(bar(kPvDone + i), rounds[i] & 1, abortp);
                            if (!ok) break;
                            scores(i, next);
                        }
                        rounds[i]++;
                    }
                    if (ok && leader) {
                        mma_commit(bar(kVEmpty + st));
                        if (j + 1 < tiles) mma_commit(bar(kKEmpty + next));
                    }
                }
            }
            if (!ok) {
                abort_flag = 1;
                // what was issued completes before the memory is given up
                if (leader) mma_commit(bar(kLast));
                __syncwarp();
                mbar_wait(bar(kLast), 0, &never);
            }
        }
    } else if (warp >= 8) {
        fewer_registers<104>();
        // ---------------- unpacking: a position a thread ----------------
        const int row = tid - 256;
        Walk w(a, whole, lane);
        uint32_t n = 0;
        bool ok = true;
        // codes c to l + s c, rounded to FP16
        auto unpack = [&](uint8_t* dst, const uint4 (&code)[DIM / 32], const half2 (&par)[P::kBlocks]) {
            const half2 one = __halves2half2(__ushort_as_half(0x6400), __ushort_as_half(0x6400));
            const half2 sixteenth = __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00)), off = __halves2half2(__ushort_as_half(0xd400), __ushort_as_half(0xd400));
#pragma unroll
            for (int c = 0; c < DIM / 32; c++) {
                const half2 s = __low2half2(par[c / 2]), l = __high2half2(par[c / 2]);
                const uint32_t word[4] = {code[c].x, code[c].y, code[c].z, code[c].w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    half2 h[4];
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint32_t v = k ? word[i] >> 8 : word[i], lo = (v & 0x000f000fu) | 0x64006400u, hi = (v & 0x00f000f0u) | 0x64006400u;
                        h[2 * k] = __hfma2(__hsub2(*reinterpret_cast<const half2*>(&lo), one), s, l);
                        h[2 * k + 1] = __hfma2(__hfma2(*reinterpret_cast<const half2*>(&hi), sixteenth, off), s, l);
                    }
                    const int piece = c * 4 + i;                            // of 16 bytes
                    *reinterpret_cast<uint4*>(dst + (piece >> 3) * kBlock + row * 128 + (((piece & 7) ^ (row & 7)) << 4)) = *reinterpret_cast<const uint4*>(h);
                }
            }
        };
        while (ok && w.advance()) {
            const size_t base = cache_row(a.c, w.b, w.head, 0);
            uint4 kc[DIM / 32], vc[DIM / 32];
            half2 kp[P::kBlocks], vp[P::kBlocks];
            auto load = [&](int j) {
                const int p = j * kTile + row;
                const bool valid = p < w.visible;                           // positions behind hold anything: they become 0
#pragma unroll
                for (int c = 0; c < DIM / 32; c++) {
                    kc[c] = valid ? reinterpret_cast<const uint4*>(a.c.kc + (base + p) * (DIM / 2))[c] : make_uint4(0, 0, 0, 0);
                    vc[c] = valid ? reinterpret_cast<const uint4*>(a.c.vc + (base + p) * (DIM / 2))[c] : make_uint4(0, 0, 0, 0);
                }
                const half2 zero = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
#pragma unroll
                for (int c = 0; c < P::kBlocks; c++) {
                    kp[c] = valid ? a.c.kp[(base + p) * P::kBlocks + c] : zero;
                    vp[c] = valid ? a.c.vp[(base + p) * P::kBlocks + c] : zero;
                }
            };
            load(w.j0);
            for (int j = w.j0; j < w.j1; j++, n++) {
                const uint32_t st = n & 1, parity = ((n >> 1) & 1) ^ 1;
                uint4 k_now[DIM / 32], v_now[DIM / 32];
                half2 kp_now[P::kBlocks], vp_now[P::kBlocks];
#pragma unroll
                for (int c = 0; c < DIM / 32; c++) {
                    k_now[c] = kc[c];
                    v_now[c] = vc[c];
                }
#pragma unroll
                for (int c = 0; c < P::kBlocks; c++) {
                    kp_now[c] = kp[c];
                    vp_now[c] = vp[c];
                }
                if (j + 1 < w.j1) load(j + 1);
                if (!(ok = mbar_wait(bar(kKEmpty + st), parity, abortp))) break;
                unpack(ks + st * P::kOperand, k_now, kp_now);
                fence_async();
                mbar_arrive(bar(kKFull + st));
                if (!(ok = mbar_wait(bar(kVEmpty + st), parity, abortp))) break;
                unpack(vs + st * P::kOperand, v_now, vp_now);
                fence_async();
                mbar_arrive(bar(kVFull + st));
            }
        }
        if (!ok) abort_flag = 1;
    } else {
        more_registers<176>();
        // ---------------- softmax: a row a thread ----------------
        const int i = warp >> 2, row = tid & (kTile - 1);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, row_s = tmem + i * kTile + lanes, row_o = tmem + kRowTiles * kTile + i * DIM + lanes;
        Walk w(a, whole, lane);
        uint32_t rounds = 0;
        bool ok = true;
        while (ok && w.advance()) {
            const int tile_rows = w.tile_rows(i), r = w.tile * kRows + i * kTile + row;
            if (tile_rows <= 0) continue;
            const bool there = row < tile_rows;
            const int token = there ? r / w.per : 0, head = w.head * w.per + (there ? r % w.per : 0);
            const int sees = there ? w.span.position(token) + 1 : 0, least = w.span.position((r - row) / w.per) + 1;
            // ---- the row of queries ----
            float scale2 = a.scale * kLog2e;
            {
                const uint4* src = reinterpret_cast<const uint4*>(q.p + (size_t)(w.span.row0 + token) * q.ld + (size_t)head * DIM);
                uint4 v[DIM / 8];
#pragma unroll
                for (int c = 0; c < DIM / 8; c++) v[c] = there ? src[c] : make_uint4(0, 0, 0, 0);
                if constexpr (!std::is_same<T, half>::value) {
                    float top = 0.f;
#pragma unroll
                    for (int c = 0; c < DIM / 8; c++)
#pragma unroll
                        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(as_float(reinterpret_cast<const T*>(&v[c])[e])));
                    const int e = (__float_as_int(top) >> 23) - 127;
                    float up = 1.f;
                    if (top > 0.f && e < 128) {
                        const int sh = min(14 - e, 126);
                        up = __int_as_float((127 + sh) << 23);
                        scale2 *= __int_as_float((127 - sh) << 23);
                    }
#pragma unroll
                    for (int c = 0; c < DIM / 8; c++) {
                        half2 h[4];
#pragma unroll
                        for (int e2 = 0; e2 < 4; e2++)
                            h[e2] = __floats2half2_rn(as_float(reinterpret_cast<const T*>(&v[c])[2 * e2]) * up, as_float(reinterpret_cast<const T*>(&v[c])[2 * e2 + 1]) * up);
                        v[c] = *reinterpret_cast<const uint4*>(h);
                    }
                }
#pragma unroll
                for (int c = 0; c < DIM / 8; c++)
                    *reinterpret_cast<uint4*>(qs + i * P::kOperand + (c >> 3) * kBlock + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v[c];
                fence_async();
                mbar_arrive(bar(kQFull + i));
            }
            float m = -INFINITY, l = 0.f;
            for (int j = w.j0; j < w.j1; j++, rounds++) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar(kSFull + i), rounds & 1, abortp));
                if (!ok) break;
                fence_after();
                uint32_t raw[4][32];
#pragma unroll
                for (int k = 0; k < 4; k++) tmem_ld32(row_s + k * 32, raw[k]);
                wait_ld();
                f32x2 s[64];
                const f32x2 scale = pair_f32(scale2, scale2);
#pragma unroll
                for (int k = 0; k < 64; k++) s[k] = mul_pair(pair_f32(raw[k >> 4][2 * (k & 15)], raw[k >> 4][2 * (k & 15) + 1]), scale);
                if ((j + 1) * kTile > least) {                              // some (row, position) of the tile is masked
                    const int seen = sees - j * kTile;
#pragma unroll
                    for (int k = 0; k < 64; k++) {
                        const float2 v = split_f32(s[k]);
                        s[k] = pair_f32(2 * k >= seen ? -INFINITY : v.x, 2 * k + 1 >= seen ? -INFINITY : v.y);
                    }
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < 64; k++) {
                    const float2 v = split_f32(s[k]);
                    top[k & 3] = fmaxf(top[k & 3], fmaxf(v.x, v.y));
                }
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                const bool grows = mx > m + kSlack;
                if (__any_sync(0xffffffffu, grows)) {
                    const float f = grows ? exp2_neg(m - mx) : 1.f;         // 0 where nothing was seen before
                    if (grows) {
                        m = mx;
                        l *= f;
                    }
                    if (j > w.j0) {
#pragma unroll 1
                        for (int c = 0; c < DIM; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(row_o + c, o);
                            wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st32(row_o + c, o);
                        }
                    }
                }
                const float ref = kLift - (m == -INFINITY ? 0.f : m);
                const f32x2 off = pair_f32(ref, ref);
                f32x2 sum[2] = {0ull, 0ull};
#pragma unroll
                for (int part = 0; part < 2; part++) {
                    uint32_t pw[32];
#pragma unroll
                    for (int k = 0; k < 32; k++) {
                        const float2 e = split_f32(add_pair(s[part * 32 + k], off));
                        const float x = exp2_neg(e.x), y = exp2_neg(e.y);
                        sum[k & 1] = add_pair(sum[k & 1], pair_f32(x, y));
                        pw[k] = Pair2<half>::of(x, y);
                    }
                    tmem_st32(row_s + part * 32, pw);
                }
                l += sum_pair(add_pair(sum[0], sum[1]));
                wait_st();
                fence_before();
                mbar_arrive(bar(kPReady + i));
            }
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(kPvDone + i), (rounds - 1) & 1, abortp));
            if (!ok) break;
            fence_after();
            if (w.complete()) {
                T* y = out.p + (size_t)(w.span.row0 + token) * out.ld + (size_t)head * DIM;
#pragma unroll 1
                for (int c = 0; c < DIM; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(row_o + c, o);
                    wait_ld();
                    if (there)
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            store_row<T>(y + c + e, make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3])), l,
                                         sees > 0);
                }
            } else {
                float* rec = static_cast<float*>(a.ws) + ((size_t)blockIdx.x * 2 + (w.segment > 0)) * kRecord<DIM, kRows>;
                const int at = i * kTile + row;
                if (there) {
                    rec[at] = m;
                    rec[kRows + at] = l;
                }
#pragma unroll 1
                for (int c = 0; c < DIM; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(row_o + c, o);
                    wait_ld();
                    if (there)
#pragma unroll
                        for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(rec + 2 * kRows + at * DIM + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            fence_before();                                                 // the next products come after these reads
        }
        if (!ok) abort_flag = 1;
    }
    fence_before();
    __syncthreads();
    if (abort_flag && tid == 0) atomicExch(a.s.err, TLLM_ERR_TIMEOUT);
    if (warp == 12) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::kTmemCols) : "memory");
    }
}

template <typename T, int DIM>
int launch(const Cache4Call& a, Rows<const T> q, Rows<T> out, const PromptPlan& p, cudaStream_t stream)
{
    static bool attr[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return fail(TLLM_ERR_LAUNCH, "cache4_prompt: no current device");
    const auto kernel = cache4_prompt_kernel<T, DIM>;
    if (!attr[dev]) {
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Prompt<DIM>::kSmem);
        attr[dev] = true;
    }
    const int st = launch_pdl("cache4_prompt", kernel, dim3(p.ctas), dim3(kThreads), Prompt<DIM>::kSmem, stream, a, q, out, p.whole);
    return st || p.whole ? st : launch_cache4_join<T>(a, out, kRows, p.ctas, p.items, stream);
}

}  // namespace

PromptPlan prompt_plan(const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    PromptPlan p;
    const int per = heads / c.kv_heads, most = max_new > 0 && max_new < tokens ? max_new : tokens;
    const long long tiles = ((long long)most * per + kRows - 1) / kRows, pairs = (long long)c.batch * c.kv_heads;
    // tiles of rows that there are at most, and at most in all
    const long long all = ((long long)tokens * per + kRows - 1) / kRows * c.kv_heads + pairs;
    const long long grid = tiles * pairs < (1 << 20) ? tiles * pairs : (1 << 20) / pairs * pairs;
    p.whole = all >= 222;
    p.items = (int)(all < 65535 ? all : 65535);
    p.ctas = p.whole ? (int)(grid < pairs ? pairs : grid) : 148;
    p.bytes = p.whole ? 0 : (size_t)p.ctas * 2 * kRows * (c.dim + 2) * sizeof(float);
    return p;
}

template <typename T>
int launch_cache4_prompt(const Cache4Call& a, Rows<const T> q, Rows<T> out, const PromptPlan& p, cudaStream_t stream)
{
    return a.c.dim == 64 ? launch<T, 64>(a, q, out, p, stream) : launch<T, 128>(a, q, out, p, stream);
}

template int launch_cache4_prompt<half>(const Cache4Call&, Rows<const half>, Rows<half>, const PromptPlan&, cudaStream_t);
template int launch_cache4_prompt<bf16>(const Cache4Call&, Rows<const bf16>, Rows<bf16>, const PromptPlan&, cudaStream_t);

}  // namespace tllm
