// Attention over the 4-bit key/value cache for many rows a sequence, on the 5th-generation tensor cores.
//
// A CTA takes 256 rows of a key/value head (new tokens times the query heads that share it) as two tiles of 128 and
// walks over tiles of 128 positions.  Roles: four warps turn the codes of keys into FP16 numbers in shared memory,
// rounded once (l + s c, 11 bits), three those of values; one issues tcgen05.mma; four for each tile of rows have a row
// a thread.
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
constexpr int kThreads = 512;                        // warps: rows' softmax 0-3 and 4-7, keys 8-11, products 12, values 13-15
constexpr int kValueThreads = 96;
// registers of a softmax thread, of the others: 2 * many + 2 * few = 4 * 128
template <bool UNPACK> constexpr int kMany = UNPACK ? 184 : 200;
template <bool UNPACK> constexpr int kFew = 256 - kMany<UNPACK>;
constexpr int kBlock = kTile * 128;                  // bytes of 64 columns of a tile: 128-byte rows
constexpr int kStages = 2;
constexpr float kSlack = 8.f, kLift = 6.f, kLog2e = 1.4426950408889634f;

template <int DIM>
struct Prompt {
    static constexpr int kBlocks = DIM / 64;
    static constexpr int kOperand = kBlocks * kBlock;                              // bytes of a tile
    static constexpr int kValueRounds = (DIM / 32 * kTile + kValueThreads - 1) / kValueThreads;
    static constexpr int kRawKeys = kTile * (DIM / 2 + 4 * kBlocks), kRaw = kRawKeys + kValueRounds * kValueThreads * 20;     // the next tile's codes and params
    static constexpr int kSmem = (kRowTiles + 2 * kStages) * kOperand + kRaw + 1024;
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
// Issued by the lane that has `leader`; no branch, so that the operands stay in uniform registers.
__device__ __forceinline__ void mma_ss(bool leader, uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc)
{
    asm volatile(
        "{ .reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc), "r"((uint32_t)leader) : "memory");
}
__device__ __forceinline__ void mma_ts(bool leader, uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc)
{
    asm volatile(
        "{ .reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }"
        ::"r"(d), "r"(a), "l"(b), "r"(id), "r"((uint32_t)acc), "r"((uint32_t)leader) : "memory");
}
__device__ __forceinline__ void commit(bool leader, uint32_t bar)
{
    asm volatile("{ .reg .pred q; setp.ne.b32 q, %1, 0;\n"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(bar), "r"((uint32_t)leader) : "memory");
}
__device__ __forceinline__ int uniform(int x) { return (int)__reduce_or_sync(0xffffffffu, (unsigned)x); }
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool valid)
{
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(valid ? N : 0) : "memory");
}
__device__ __forceinline__ void copies_landed() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                 "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                 "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ f32x2 fma_pairs(f32x2 a, f32x2 b, f32x2 c)
{
    fma_pair(c, a, b);
    return c;
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Keys and values as FP16 rows: [batch * kv_heads][cap][dim].
struct Expanded {
    CUtensorMap k, v;
    int cap;
};

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
        if (whole) {
            segment++;
            from_top += step;
            const int tl = (rows + kRows - 1) / kRows - 1 - from_top;
            if (tl < 0) return false;
            set_tile(tl);
            j0 = 0;
            j1 = chunks;
            return true;
        }
        do {
            if (x >= to) return false;
            if (++segment > 0) next();
            j0 = chunk_at(offset);
            j1 = chunk_at(min((long long)kFixed + chunks, offset + (to - x)));
            x += kFixed + chunks - offset;
        } while (j0 == j1);
        return true;
    }
    __device__ __forceinline__ bool complete() const { return j0 == 0 && j1 == chunks; }
    __device__ __forceinline__ int tile_rows(int i) const { return min(kTile, rows - tile * kRows - i * kTile); }
};

enum Bar { kQFull = 0, kKFull = 2, kKEmpty = 4, kVFull = 6, kVEmpty = 8, kSFull = 10, kPvDone = 12, kPReady = 14, kLast = 18, kBars = 19 };

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 32 codes as l + s c, rounded to FP16.
__device__ __forceinline__ void expand32(const uint4& code, half2 par, uint4 (&y)[4])
{
    const half2 one = __halves2half2(__ushort_as_half(0x6400), __ushort_as_half(0x6400));
    const half2 sixteenth = __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00)), off = __halves2half2(__ushort_as_half(0xd400), __ushort_as_half(0xd400));
    const half2 s = __low2half2(par), l = __high2half2(par);
    const uint32_t word[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        half2 h[4];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint32_t v = k ? word[i] >> 8 : word[i], lo = (v & 0x000f000fu) | 0x64006400u, hi = (v & 0x00f000f0u) | 0x64006400u;
            h[2 * k] = __hfma2(__hsub2(*reinterpret_cast<const half2*>(&lo), one), s, l);
            h[2 * k + 1] = __hfma2(__hfma2(*reinterpret_cast<const half2*>(&hi), sixteenth, off), s, l);
        }
        y[i] = *reinterpret_cast<const uint4*>(h);
    }
}
// The same to the four 16-byte pieces of a tile's row from `piece` on.
__device__ __forceinline__ void unpack32(uint8_t* tile, int row, int piece, const uint4& code, half2 par)
{
    uint8_t* dst = tile + (piece >> 3) * kBlock + row * 128;
    uint4 y[4];
    expand32(code, par, y);
#pragma unroll
    for (int i = 0; i < 4; i++) *reinterpret_cast<uint4*>(dst + ((((piece & 7) + i) ^ (row & 7)) << 4)) = y[i];
}

// UNPACK: from the cache; else keys and values are FP16 rows in the workspace, copied by TMA (rows b * kv_heads + head of `cap`
// positions each).
template <typename T, int DIM, bool UNPACK>
__global__ void __launch_bounds__(kThreads, 1)
cache4_prompt_kernel(const Cache4Call a, const Rows<const T> q, const Rows<T> out, const bool whole, const __grid_constant__ Expanded x)
{
    using P = Prompt<DIM>;
    constexpr int kCodes = DIM / 32;                                       // 16-byte pieces of a row of codes
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t bars[kBars];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t *qs = smem, *ks = qs + kRowTiles * P::kOperand, *vs = ks + kStages * P::kOperand, *raw = vs + kStages * P::kOperand;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    volatile int* abortp = &abort_flag;
    int never = 0;

    if (tid == 0) {
        for (int i = 0; i < kBars; i++) {
            const int pair = i & ~1;
            mbar_init(bar(i), pair == kQFull || (UNPACK && pair == kKFull) || (i >= kPReady && i < kLast) ? kTile : UNPACK && pair == kVFull ? kValueThreads : 1);
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
        fewer_registers<kFew<UNPACK>>();
        if (warp == 12) {
            // ---------------- products ----------------
            // Every value that a branch or an operand depends on is uniform by a vote or a reduction of the warp: operands then come from
            // uniform registers (some 150 clocks an MMA otherwise).
            const bool leader = elect_one();
            const uint32_t id_s = idesc(kTile, false), id_o = idesc(DIM, true), base = uniform(smem_u32(smem)), t0 = uniform(tmem);
            const auto wait = [&](int i, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar(i), parity, abortp)) != 0; };
            const auto score = [&](int i, uint32_t st) {
                const uint64_t qd = make_sw128_desc(base + i * P::kOperand), kd = make_sw128_desc(base + (kRowTiles + st) * P::kOperand);
#pragma unroll
                for (int j = 0; j < P::kBlocks; j++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t o = j * (kBlock >> 4) + k * 2;
                        mma_ss(leader, t0 + i * kTile, qd + o, kd + o, id_s, j > 0 || k > 0);
                    }
                commit(leader, bar(kSFull + i));
            };
            // half of the positions of a tile
            const auto output = [&](int i, uint32_t st, int part, bool first) {
                const uint64_t vd = feature_major_desc(base + (kRowTiles + kStages + st) * P::kOperand);
#pragma unroll
                for (int k = part * 4; k < part * 4 + 4; k++)
                    mma_ts(leader, t0 + kRowTiles * kTile + i * DIM, t0 + i * kTile + k * 8, vd + k * (2048 >> 4), id_o, !first || k > 0);
                if (part) commit(leader, bar(kPvDone + i));
            };
            Walk w(a, whole, lane);
            uint32_t n = 0, items[2] = {0, 0}, rounds[2] = {0, 0};         // tiles of positions so far; by tile of rows: segments, weights
            bool ok = true;
            while (ok && __any_sync(0xffffffffu, w.advance())) {
                const int active = uniform(w.tile_rows(1) > 0 ? 2 : 1), tiles = uniform(w.j1 - w.j0);
                ok = wait(kKFull + (n & 1), (n >> 1) & 1);
#pragma unroll
                for (int i = 0; i < 2; i++)
                    if (ok && i < active) {
                        ok = wait(kQFull + i, items[i]++ & 1);
                        fence_after();
                        if (ok) score(i, n & 1);
                    }
                if (ok) commit(leader, bar(kKEmpty + (n & 1)));
                for (int j = 0; ok && j < tiles; j++, n++) {
                    const uint32_t st = n & 1;
                    const bool more = j + 1 < tiles;
                    ok = wait(kVFull + st, (n >> 1) & 1);
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        if (i < active) {
#pragma unroll
                            for (int part = 0; part < 2; part++) {
                                ok = ok && wait(kPReady + 2 * i + part, rounds[i] & 1);
                                if (!ok) break;
                                fence_after();
                                output(i, st, part, j == 0);
                            }
                            if (ok && more) {
                                // the weights lie where the next scores go
                                ok = (i > 0 || wait(kKFull + (st ^ 1), ((n + 1) >> 1) & 1)) && wait(kPvDone + i, rounds[i] & 1);
                                fence_after();
                                if (ok) score(i, st ^ 1);
                            }
                            rounds[i]++;
                        }
                    if (ok) {
                        commit(leader, bar(kVEmpty + st));
                        if (more) commit(leader, bar(kKEmpty + (st ^ 1)));
                    }
                }
            }
            if (!ok) {
                abort_flag = 1;
                // what was issued completes before the memory is given up
                commit(leader, bar(kLast));
                __syncwarp();
                mbar_wait(bar(kLast), 0, &never);
            }
        } else if constexpr (!UNPACK) {
            if (warp == 13) {
                // ---------------- copies of expanded keys and values ----------------
                const bool leader = elect_one();
                Walk w(a, whole, lane);
                uint32_t n = 0, issued[2] = {0, 0};
                bool ok = true;
                while (ok && w.advance()) {
                    const int row0 = (w.b * w.kv_heads + w.head) * x.cap;
                    for (int j = w.j0; ok && j < w.j1; j++, n++) {
                        const uint32_t st = n & 1, parity = ((n >> 1) & 1) ^ 1;
#pragma unroll
                        for (int side = 0; side < 2; side++) {
                            const uint32_t full = bar((side ? kVFull : kKFull) + st);
                            if (!(ok = mbar_wait(bar((side ? kVEmpty : kKEmpty) + st), parity, abortp))) break;
                            if (leader) {
                                mbar_expect_tx(full, P::kOperand);
#pragma unroll
                                for (int c = 0; c < P::kBlocks; c++)
                                    tma_load_2d(smem_u32((side ? vs : ks) + st * P::kOperand + c * kBlock), side ? &x.v : &x.k, c * 64, row0 + j * kTile, full);
                            }
                            issued[side] = n + 1;
                        }
                    }
                }
                if (!ok) abort_flag = 1;
                __syncwarp();
                // after an abort the copies still in flight must land before the shared memory goes away
                if (*abortp)
                    for (int side = 0; side < 2; side++)
                        for (uint32_t i = issued[side] > 2 ? issued[side] - 2 : 0; i < issued[side]; i++)
                            mbar_wait(bar((side ? kVFull : kKFull) + (i & 1)), (i >> 1) & 1, &never);
            }
        } else {
            // ---------------- values: 16 bytes of a position at once ----------------
            constexpr int kRounds = P::kValueRounds;
            const int first = tid - 13 * 32;
            const uint8_t* mine = raw + P::kRawKeys + first * 16;            // a thread reads what it copied
            const half2* my_par = reinterpret_cast<const half2*>(raw + P::kRawKeys + kRounds * kValueThreads * 16) + first;
            Walk w(a, whole, lane);
            uint32_t n = 0;
            bool ok = true;
            while (ok && w.advance()) {
                const size_t row0 = cache_row(a.c, w.b, w.head, 0);
                const auto load = [&](int j, int k) {
                    const int e = first + k * kValueThreads, c = e / kTile, p = j * kTile + e % kTile;
                    const bool valid = c < kCodes && p < w.visible;         // positions behind hold anything: they become 0
                    const size_t at = row0 + (valid ? p : 0);
                    copy_async<16>(smem_u32(mine) + k * kValueThreads * 16, a.c.vc + at * (DIM / 2) + (valid ? c * 16 : 0), valid);
                    copy_async<4>(smem_u32(my_par) + k * kValueThreads * 4, a.c.vp + at * P::kBlocks + (valid ? c / 2 : 0), valid);
                };
#pragma unroll
                for (int k = 0; k < kRounds; k++) load(w.j0, k);
                for (int j = w.j0; j < w.j1; j++, n++) {
                    const uint32_t st = n & 1;
                    copies_landed();
                    if (!(ok = mbar_wait(bar(kVEmpty + st), ((n >> 1) & 1) ^ 1, abortp))) break;
#pragma unroll
                    for (int k = 0; k < kRounds; k++) {
                        const int e = first + k * kValueThreads, c = e / kTile;
                        if (c < kCodes)
                            unpack32(vs + st * P::kOperand, e % kTile, c * 4, *reinterpret_cast<const uint4*>(mine + k * kValueThreads * 16), my_par[k * kValueThreads]);
                        if (j + 1 < w.j1) load(j + 1, k);
                    }
                    fence_async();
                    mbar_arrive(bar(kVFull + st));
                }
            }
            copies_landed();
            if (!ok) abort_flag = 1;
        }
    } else if (warp >= 8) {
        fewer_registers<kFew<UNPACK>>();
        // ---------------- keys: a position a thread ----------------
        if constexpr (UNPACK) {
        const int row = tid - 256;
        const uint8_t* mine = raw + row * 16;
        const half2* my_par = reinterpret_cast<const half2*>(raw + kCodes * kTile * 16 + row * 4 * P::kBlocks);
        Walk w(a, whole, lane);
        uint32_t n = 0;
        bool ok = true;
        while (ok && w.advance()) {
            const size_t row0 = cache_row(a.c, w.b, w.head, 0);
            const auto load = [&](int j, int c) {
                const int p = j * kTile + row;
                const bool valid = p < w.visible;
                const size_t at = row0 + (valid ? p : 0);
                copy_async<16>(smem_u32(mine) + c * kTile * 16, a.c.kc + at * (DIM / 2) + c * 16, valid);
            };
            const auto load_par = [&](int j) {
                const int p = j * kTile + row;
                const bool valid = p < w.visible;
                copy_async<4 * P::kBlocks>(smem_u32(my_par), a.c.kp + (row0 + (valid ? p : 0)) * P::kBlocks, valid);
            };
            load_par(w.j0);
#pragma unroll
            for (int c = 0; c < kCodes; c++) load(w.j0, c);
            for (int j = w.j0; j < w.j1; j++, n++) {
                const uint32_t st = n & 1;
                copies_landed();
                if (!(ok = mbar_wait(bar(kKEmpty + st), ((n >> 1) & 1) ^ 1, abortp))) break;
                half2 par[P::kBlocks];
#pragma unroll
                for (int c = 0; c < P::kBlocks; c++) par[c] = my_par[c];
                if (j + 1 < w.j1) load_par(j + 1);
#pragma unroll
                for (int c = 0; c < kCodes; c++) {
                    unpack32(ks + st * P::kOperand, row, c * 4, *reinterpret_cast<const uint4*>(mine + c * kTile * 16), par[c / 2]);
                    if (j + 1 < w.j1) load(j + 1, c);
                }
                fence_async();
                mbar_arrive(bar(kKFull + st));
            }
        }
        copies_landed();
        if (!ok) abort_flag = 1;
        }
    } else {
        more_registers<kMany<UNPACK>>();
        // ---------------- softmax: a row a thread ----------------
        const int i = warp >> 2, row = tid & (kTile - 1);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, row_s = tmem + i * kTile + lanes, row_o = tmem + kRowTiles * kTile + i * DIM + lanes;
        Walk w(a, whole, lane);
        if (!whole && tid == 0) entry_of(a.ws, blockIdx.x)->parts = 0;
        uint32_t rounds = 0;
        bool ok = true;
        while (ok && w.advance()) {
            const int tile_rows = w.tile_rows(i), r = w.tile * kRows + i * kTile + row;
            if (tile_rows <= 0) continue;
            const bool there = row < tile_rows;
            const int token = there ? r / w.per : 0, head = w.head * w.per + (there ? r % w.per : 0);
            const int sees = there ? w.span.position(token) + 1 : 0, least = w.span.position((r - row) / w.per) + 1;
            // ---- the row of queries, with the sign of the scale ----
            float scale2 = fabsf(a.scale) * kLog2e;
            {
                const uint4* src = reinterpret_cast<const uint4*>(q.p + (size_t)(w.span.row0 + token) * q.ld + (size_t)head * DIM);
                uint4 v[DIM / 8];
#pragma unroll
                for (int c = 0; c < DIM / 8; c++) v[c] = there ? src[c] : make_uint4(0, 0, 0, 0);
                float up = a.scale < 0.f ? -1.f : 1.f;
                if constexpr (!std::is_same<T, half>::value) {
                    float top = 0.f;
#pragma unroll
                    for (int c = 0; c < DIM / 8; c++)
#pragma unroll
                        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(as_float(reinterpret_cast<const T*>(&v[c])[e])));
                    const int e = (__float_as_int(top) >> 23) - 127;
                    if (top > 0.f && e < 128) {
                        const int sh = min(14 - e, 126);
                        up *= __int_as_float((127 + sh) << 23);
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
                } else if (up < 0.f) {
#pragma unroll
                    for (int c = 0; c < DIM / 8; c++) v[c] = make_uint4(v[c].x ^ 0x80008000u, v[c].y ^ 0x80008000u, v[c].z ^ 0x80008000u, v[c].w ^ 0x80008000u);
                }
#pragma unroll
                for (int c = 0; c < DIM / 8; c++)
                    *reinterpret_cast<uint4*>(qs + i * P::kOperand + (c >> 3) * kBlock + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v[c];
                fence_async();
                mbar_arrive(bar(kQFull + i));
            }
            scale2 = fmaxf(scale2, 1e-37f);                                 // a masked score times it stays -infinity
            const f32x2 scale = pair_f32(scale2, scale2);
            float m = -INFINITY, l = 0.f;
            for (int j = w.j0; j < w.j1; j++, rounds++) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar(kSFull + i), rounds & 1, abortp));
                if (!ok) break;
                fence_after();
                uint32_t s[4][32];
                tmem_ld32(row_s, s[0]);
                tmem_ld32(row_s + 32, s[1]);
                wait_ld();
                tmem_ld32(row_s + 64, s[2]);
                tmem_ld32(row_s + 96, s[3]);
                const bool masked = (j + 1) * kTile > least;                // some (row, position) of the tile is
                const int seen = sees - j * kTile;
                float top[2] = {-INFINITY, -INFINITY};
                const auto mask = [&](int part) {
                    if (masked)
#pragma unroll
                        for (int k = 0; k < 64; k++)
                            if (part * 64 + k >= seen) s[part * 2 + k / 32][k % 32] = 0xff800000u;
                };
                const auto largest = [&](int k) {                            // of four scores
                    const uint32_t(&v)[32] = s[k / 32];
                    top[0] = max3(top[0], __uint_as_float(v[k % 32]), __uint_as_float(v[k % 32 + 1]));
                    top[1] = max3(top[1], __uint_as_float(v[k % 32 + 2]), __uint_as_float(v[k % 32 + 3]));
                };
                f32x2 sum[2], off;
                uint32_t pw[32];
                const auto weights = [&](int part, auto between) {           // of 64 positions
#pragma unroll
                    for (int k = 0; k < 32; k++) {
                        const uint32_t(&v)[32] = s[part * 2 + k / 16];
                        const float2 e = split_f32(fma_pairs(pair_f32(v[k % 16 * 2], v[k % 16 * 2 + 1]), scale, off));
                        const float x = exp2_neg(e.x), y = exp2_neg(e.y);
                        sum[k & 1] = add_pair(sum[k & 1], pair_f32(x, y));
                        pw[k] = Pair2<half>::of(x, y);
                        between(k);
                    }
                };
                const auto hand_over = [&](int part) {
                    tmem_st32(row_s + part * 32, pw);
                    wait_st();
                    fence_before();
                    mbar_arrive(bar(kPReady + 2 * i + part));
                };
                const auto reference = [&] {
                    const float ref = kLift - (m == -INFINITY ? 0.f : m);
                    off = pair_f32(ref, ref);
                    sum[0] = sum[1] = 0ull;
                };
                mask(0);
                // with the maximum so far, which rarely has to move: its own search runs beside the exponentials
                const bool guess = !UNPACK && j > w.j0;
                if (guess) {
                    wait_ld();
                    mask(1);
                    reference();
                    weights(0, [&](int k) { largest(4 * k); });
                } else {
#pragma unroll
                    for (int k = 0; k < 64; k += 4) largest(k);
                    wait_ld();
                    mask(1);
#pragma unroll
                    for (int k = 64; k < 128; k += 4) largest(k);
                }
                const float mx = fmaxf(top[0], top[1]) * scale2;
                const bool grows = mx > m + kSlack;
                const bool any = __any_sync(0xffffffffu, grows);
                if (any) {
                    const float f = grows ? exp2_neg(m - mx) : 1.f;         // 0 where nothing was seen before
                    if (grows) {
                        m = mx;
                        l *= f;
                    }
                    if (j > w.j0) {
#pragma unroll 1
                        for (int c = 0; c < DIM; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(row_o + c, o);
                            wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16(row_o + c, o);
                        }
                    }
                }
                if (any || !guess) {
                    reference();
                    weights(0, [](int) {});
                }
                hand_over(0);
                weights(1, [](int) {});
                hand_over(1);
                l += sum_pair(add_pair(sum[0], sum[1]));
            }
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(kPvDone + i), (rounds - 1) & 1, abortp));
            if (!ok) break;
            fence_after();
            T* y = out.p + (size_t)(w.span.row0 + token) * out.ld + (size_t)head * DIM;
            const int at = i * kTile + row;
            const bool complete = w.complete();
            float* rec = complete ? nullptr : record_of<DIM, kRows>(a.ws, gridDim.x, blockIdx.x, w.segment > 0);
            if (!complete && w.j0 == 0 && tid == 0)
                *entry_of(a.ws, blockIdx.x) =
                    Shared4{w.owner(w.x - 1, gridDim.x) - (int)blockIdx.x + 1, w.segment > 0, w.head, w.tile, w.span.row0, w.span.n, w.span.len, 0};
            if (!complete && there) {
                rec[at] = m;
                rec[kRows + at] = l;
            }
#pragma unroll 1
            for (int c = 0; c < DIM; c += 32) {
                uint32_t o[32];
                tmem_ld32(row_o + c, o);
                wait_ld();
                if (there) {
                    if (complete) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            store_row<T>(y + c + e, make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3])), l,
                                         sees > 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(rec + 2 * kRows + at * DIM + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
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

// Rows of keys and values of the sequences of a call as FP16, rounded once; zeros up to the end of a tile of positions.
template <int DIM>
__global__ void __launch_bounds__(256)
cache4_expand_kernel(const Cache4Call a, uint8_t* k, uint8_t* v, const int cap)
{
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.z, g = blockIdx.y;
    const Span sp = span_of(a.s, b, blockIdx.x == 0 && g == 0 && threadIdx.x == 0);
    const int end = sp.n > 0 ? min((sp.len + kTile - 1) / kTile * kTile, cap) : 0;
    constexpr int kPieces = DIM / 32, kPositions = 256 / kPieces;          // 16 bytes of codes a thread, of keys and of values
    const int c = threadIdx.x % kPieces;
    for (int p = blockIdx.x * kPositions + threadIdx.x / kPieces; p < end; p += gridDim.x * kPositions) {
        const size_t row = cache_row(a.c, b, g, min(p, sp.len - 1)), to = ((size_t)(b * a.c.kv_heads + g) * cap + p) * DIM * 2 + c * 64;
#pragma unroll
        for (int side = 0; side < 2; side++) {
            uint4 code = make_uint4(0, 0, 0, 0);
            half2 par = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
            if (p < sp.len) {
                code = reinterpret_cast<const uint4*>((side ? a.c.vc : a.c.kc) + row * (DIM / 2))[c];
                par = (side ? a.c.vp : a.c.kp)[row * (DIM / 64) + c / 2];
            }
            uint4 y[4];
            expand32(code, par, y);
#pragma unroll
            for (int i = 0; i < 4; i++) reinterpret_cast<uint4*>((side ? v : k) + to)[i] = y[i];
        }
    }
}

int encode(CUtensorMap* map, const uint8_t* p, int dim, size_t rows)
{
    const EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(TLLM_ERR_LAUNCH, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)dim * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)kTile}, estr[2] = {1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<uint8_t*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? TLLM_OK : fail(TLLM_ERR_LAUNCH, "cache4_prompt: cuTensorMapEncodeTiled failed with %d", (int)r);
}

template <typename T, int DIM, bool UNPACK>
int launch_form(const Cache4Call& a, Rows<const T> q, Rows<T> out, const PromptPlan& p, cudaStream_t stream)
{
    static bool attr[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return fail(TLLM_ERR_LAUNCH, "cache4_prompt: no current device");
    const auto kernel = cache4_prompt_kernel<T, DIM, UNPACK>;
    if (!attr[dev]) {
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Prompt<DIM>::kSmem);
        attr[dev] = true;
    }
    Expanded x = {};
    int st;
    if (!UNPACK) {
        const size_t rows = (size_t)a.c.batch * a.c.kv_heads * p.cap;
        uint8_t *k = static_cast<uint8_t*>(a.ws) + p.join_bytes, *v = k + rows * DIM * 2;
        x.cap = p.cap;
        if ((st = encode(&x.k, k, DIM, rows)) || (st = encode(&x.v, v, DIM, rows))) return st;
        const int positions = 256 / (DIM / 32), blocks = (p.cap + positions - 1) / positions;
        st = launch_pdl("cache4_expand", cache4_expand_kernel<DIM>, dim3(blocks < 1024 ? blocks : 1024, a.c.kv_heads, a.c.batch), dim3(256), 0, stream, a, k, v, p.cap);
        if (st) return st;
    }
    st = launch_pdl("cache4_prompt", kernel, dim3(p.ctas), dim3(kThreads), Prompt<DIM>::kSmem, stream, a, q, out, p.whole, x);
    return st || p.whole ? st : launch_cache4_join<T>(a, out, kRows, p.ctas, stream);
}

template <typename T, int DIM>
int launch(const Cache4Call& a, Rows<const T> q, Rows<T> out, const PromptPlan& p, cudaStream_t stream)
{
    return p.cap ? launch_form<T, DIM, false>(a, q, out, p, stream) : launch_form<T, DIM, true>(a, q, out, p, stream);
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
    p.ctas = p.whole ? (int)(grid < pairs ? pairs : grid) : 148;
    p.join_bytes = p.whole ? 0 : (join_bytes(c.dim, kRows, p.ctas) + 255) / 256 * 256;
    const int len = max_len > 0 && max_len < c.rows ? max_len : c.rows;
    p.cap = tiles >= 3 && pairs * len < (1 << 30) ? (len + kTile - 1) / kTile * kTile : 0;
    p.bytes = p.join_bytes + (size_t)pairs * p.cap * c.dim * 4;
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
