// Attention over the 4-bit key/value cache for many rows a sequence, on the 5th-generation tensor cores.
//
// A CTA takes 256 rows of a key/value head (new tokens times the query heads that share it) as two tiles of 128, or one
// tile of 128 where there are SMs for it, and walks over tiles of 128 positions.  Roles: three warps turn codes of keys into FP16 numbers in shared memory, rounded
// once (l + s c, 11 bits), three those of values; one for each tile of rows issues tcgen05.mma; four for each tile of
// rows have a row a thread.
//   S = Q K^T    128 FP32 columns of tensor memory for each tile of rows; keys in shared memory, queries too, or for heads
//                of 64, where it has room, in tensor memory (nine prompts 3 % quicker)
//   softmax      a thread reads its row; the weights go back over S as FP16, with a factor of 2^6 that leaves small
//                ones their bits (the sum of the weights takes it out): 11 of them down to 2^-20 of the largest, steps of 2^-30 of it below
//   O += P V     weights from tensor memory, values feature-major
// so a tile of the cache is unpacked once for 256 rows, and one tile's products run beside the other's softmax.
// BF16 queries become FP16 numbers times a power of two of their row.  The running maximum moves when a score exceeds it
// by more than 2^8; sums are FP32.  A position that a row does not see is masked before the maximum, and values are
// finite (append marks a NaN in the key), so nothing behind a row's own position reaches it.
//
// Work: tiles of rows, longest first; or, where there are too few, all tiles of positions as one sequence of which
// every CTA takes an equal part, parts of a tile of rows joined by a second launch in their order.
// All mbarrier waits are bounded.
//
// What bounds it: 512 tokens of 32 heads of 128 over 8 behind 16000 take 149 - 168 us from card to card, 0.81 - 0.92 PFLOP/s (the power
// limit decides), 14 of them the join; 149 were 136 without the exponentials, and 158, before the scores were read twice, 125 without any softmax
// arithmetic and 149 without the products: the softmax warps, then the tensor pipe.  Heads of 64 have half the products for the same
// softmax: nine prompts of 4529 tokens in all take 115, 99 without the exponentials, of which 28 are their full rate.
#include <cmath>
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

constexpr int kTile = kPromptChunk;
constexpr int kThreads = 512;                        // warps: softmax of a tile of rows 0-3, of the other 4-7, its products 12, 13, keys and values the rest
constexpr int kUnpackThreads = 96;                   // of keys, and of values
constexpr int kBlock = kTile * 128;                  // bytes of 64 columns of a tile: 128-byte rows
constexpr int kStages = 2, kHalf = kTile / 2;
constexpr float kLift = 6.f, kSlack = 8.f, kLog2e = 1.4426950408889634f;             // 2^(kLift + kSlack) fits FP16

template <int DIM, int ROW_TILES>
struct Prompt {
    static constexpr int kRows = ROW_TILES * kTile;
    static constexpr int kBlocks = DIM / 64;
    static constexpr int kOperand = kBlocks * kBlock;                              // bytes of a tile
    static constexpr int kRounds = (DIM / 32 * kTile + kUnpackThreads - 1) / kUnpackThreads;      // of 16 bytes a thread, of keys or values
    static constexpr int kRawSide = kRounds * kUnpackThreads * 20;                                // the next tile's codes and params
    static constexpr int kSmem = (ROW_TILES + 2 * kStages) * kOperand + 2 * kRawSide + 1024;
    static constexpr int kQueryCols = DIM == 64 ? DIM / 2 : 0;                     // of tensor memory for a tile's queries, where there is room
    static constexpr uint32_t kTmemCols = ROW_TILES == 2 ? 512 : 256;                // a power of two that holds ROW_TILES (kTile + DIM + kQueryCols)
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

// A tile's rows of a key/value head and the tiles of positions [j0, j1) of its `chunks`, one after the other for this CTA;
// every role walks over the same.
template <int ROWS>
struct Walk : Work<ROWS, kTile> {
    using Base = Work<ROWS, kTile>;
    using Base::s, Base::per, Base::kv_heads, Base::whole, Base::x, Base::to, Base::b, Base::head, Base::tile, Base::offset, Base::rows, Base::chunks,
        Base::span, Base::kFixed, Base::chunk_at;
    int from_top, step, j0, j1, segment;
    __device__ __forceinline__ Walk(const Cache4Call& a, bool whole_, const typename Base::Start& f) : Base(a.s, a.heads / a.c.kv_heads, a.c.kv_heads, whole_), segment(-1)
    {
        if (whole) {
            const int pairs = s.batch * kv_heads, pair = blockIdx.x % pairs;
            step = max((int)gridDim.x / pairs, 1);
            from_top = (int)blockIdx.x / pairs - step;
            b = pair / kv_heads;
            head = pair % kv_heads;
            span = span_of(s, b, blockIdx.x / pairs == 0 && head == 0 && threadIdx.x == 0);
            rows = span.n * per;
        } else {
            Base::begin(f);
        }
    }
    __device__ __forceinline__ bool advance()
    {
        if (whole) {
            segment++;
            from_top += step;
            const int tl = (rows + ROWS - 1) / ROWS - 1 - from_top;
            if (tl < 0) return false;
            Base::set_tile(tl);
            j0 = 0;
            j1 = chunks;
            return true;
        }
        do {
            if (x >= to) return false;
            if (++segment > 0) Base::next();
            j0 = chunk_at(offset);
            j1 = chunk_at(min(kFixed + chunks, offset + (to - x)));
            x += kFixed + chunks - offset;
        } while (j0 == j1);
        return true;
    }
    __device__ __forceinline__ bool complete() const { return j0 == 0 && j1 == chunks; }
    __device__ __forceinline__ int tile_rows(int i) const { return min(kTile, rows - tile * ROWS - i * kTile); }
};

// the last three by tile of rows and half of a tile of positions
enum Bar { kQFull = 0, kKFull = 2, kKEmpty = 4, kVFull = 6, kVEmpty = 8, kSFull = 10, kPvDone = 14, kPReady = 18, kLast = 22, kBars = 24 };

// the largest; NaN where one of them is
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 32 codes of a row as l + s c, rounded to FP16, to four 16-byte pieces of a tile at `dst`, exchanged as `turn` says.
__device__ __forceinline__ void unpack32(uint32_t dst, uint32_t turn, const uint4& code, half2 par)
{
    const half2 one = __halves2half2(__ushort_as_half(0x6400), __ushort_as_half(0x6400));
    const half2 sixteenth = __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00)), off = __halves2half2(__ushort_as_half(0xd400), __ushort_as_half(0xd400));
    const half2 s = __low2half2(par), l = __high2half2(par);
    const uint32_t word[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint32_t v = k ? word[i] >> 8 : word[i], lo = (v & 0x000f000fu) | 0x64006400u, hi = (v & 0x00f000f0u) | 0x64006400u;
            const half2 x = __hfma2(__hsub2(*reinterpret_cast<const half2*>(&lo), one), s, l);
            const half2 y = __hfma2(__hfma2(*reinterpret_cast<const half2*>(&hi), sixteenth, off), s, l);
            h[2 * k] = *reinterpret_cast<const uint32_t*>(&x);
            h[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&y);
        }
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + (turn ^ (uint32_t)(i << 4))), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
    }
}

template <typename T, int DIM, int ROW_TILES>
__global__ void __launch_bounds__(kThreads, 1)
cache4_prompt_kernel(const Cache4Call a, const Rows<const T> q, const Rows<T> out, const bool whole)
{
    using P = Prompt<DIM, ROW_TILES>;
    using W = Walk<P::kRows>;
    constexpr int kRows = P::kRows;
    constexpr int kCodes = DIM / 32;                                       // 16-byte pieces of a row of codes
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t bars[kBars];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, falls;
    __shared__ typename W::Base::Start start;
    __shared__ float row_scale[kRows];
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t *qs = smem, *ks = qs + ROW_TILES * P::kOperand, *vs = ks + kStages * P::kOperand, *raw = vs + kStages * P::kOperand;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    volatile int *abortp = &abort_flag, *fallsp = &falls;
    int never = 0;

    if (tid == 0) {
        for (int i = 0; i < kBars; i++) {
            const int pair = i & ~1;
            mbar_init(bar(i), pair == kQFull || (i >= kPReady && i < kLast) ? kTile : pair == kKFull || pair == kVFull ? kUnpackThreads :
                              pair == kKEmpty || pair == kVEmpty ? ROW_TILES : 1);
        }
        abort_flag = falls = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(P::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    if (warp == 13 && !whole) typename W::Base(a.s, a.heads / a.c.kv_heads, a.c.kv_heads, false).find(blockIdx.x, gridDim.x, lane, &start);
    if (!whole && tid == 0) entry_of(a.ws, blockIdx.x)->parts = 0;
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;                                       // S of both tiles of rows, then O of both

    if (warp >= 12 && warp < 12 + ROW_TILES) {
        // ---------------- products of a tile of rows ----------------
        // Every value that a branch or an operand depends on is uniform by a vote or a reduction of the warp: operands then come from
        // uniform registers (115 clocks an MMA, 155 otherwise).
        const int i = warp - 12;
        const bool leader = elect_one();
        const uint32_t id_s = idesc(kHalf, false), id_o = idesc(DIM, true), t0 = uniform(tmem), base = uniform(smem_u32(smem));
        const uint64_t qd = make_sw128_desc(base + i * P::kOperand);
        const uint32_t to_s = t0 + i * kTile, to_o = t0 + ROW_TILES * kTile + i * DIM, to_q = t0 + ROW_TILES * (kTile + DIM) + i * P::kQueryCols;
        const auto wait = [&](int k, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar(k), parity, abortp)) != 0; };
        // half h of a tile of positions
        const auto score = [&](int h, uint32_t st) {
            const uint64_t kd = make_sw128_desc(base + (ROW_TILES + st) * P::kOperand) + h * (kHalf * 128 >> 4);
            fence_after();
#pragma unroll
            for (int j = 0; j < P::kBlocks; j++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t o = j * (kBlock >> 4) + k * 2;
                    if constexpr (P::kQueryCols > 0) mma_ts(leader, to_s + h * kHalf, to_q + k * 8, kd + o, id_s, k > 0);
                    else mma_ss(leader, to_s + h * kHalf, qd + o, kd + o, id_s, j > 0 || k > 0);
                }
            commit(leader, bar(kSFull + i + 2 * h));
        };
        const auto output = [&](int h, uint32_t st, bool first) {
            const uint64_t vd = feature_major_desc(base + (ROW_TILES + kStages + st) * P::kOperand) + h * (kHalf * 128 >> 4);
            fence_after();
#pragma unroll
            for (int k = 0; k < kHalf / 16; k++) mma_ts(leader, to_o, to_s + h * kHalf + k * 8, vd + k * (2048 >> 4), id_o, !first || k > 0);
            commit(leader, bar(kPvDone + i + 2 * h));
        };
        W w(a, whole, start);
        uint32_t n = 0, items = 0, rounds = 0;                             // tiles of positions so far; with rows here: segments, tiles
        bool ok = true;
        while (ok && __any_sync(0xffffffffu, w.advance())) {
            const int tiles = uniform(w.j1 - w.j0);
            if (!uniform(w.tile_rows(i) > 0)) {
                // no rows here: the stages are free as soon as they are full
                for (int j = 0; ok && j < tiles; j++, n++) {
                    ok = wait(kKFull + (n & 1), (n >> 1) & 1) && wait(kVFull + (n & 1), (n >> 1) & 1);
                    if (ok && lane == 0) {
                        mbar_arrive(bar(kKEmpty + (n & 1)));
                        mbar_arrive(bar(kVEmpty + (n & 1)));
                    }
                }
                continue;
            }
            ok = wait(kKFull + (n & 1), (n >> 1) & 1) && wait(kQFull + i, items++ & 1);
            if (ok) {
                score(0, n & 1);
                score(1, n & 1);
                commit(leader, bar(kKEmpty + (n & 1)));
            }
            for (int j = 0; ok && j < tiles; j++, n++, rounds++) {
                const uint32_t st = n & 1, parity = rounds & 1;
                ok = wait(kVFull + st, (n >> 1) & 1);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    ok = ok && wait(kPReady + i + 2 * h, parity);
                    if (!ok) break;
                    output(h, st, j == 0 && h == 0);
                    if (h == 1) commit(leader, bar(kVEmpty + st));
                    if (j + 1 < tiles) {
                        // the weights lie where the next scores go
                        ok = (h > 0 || wait(kKFull + (st ^ 1), ((n + 1) >> 1) & 1)) && wait(kPvDone + i + 2 * h, parity);
                        if (!ok) break;
                        score(h, st ^ 1);
                        if (h == 1) commit(leader, bar(kKEmpty + (st ^ 1)));
                    }
                }
            }
        }
        if (!ok) {
            abort_flag = 1;
            // what was issued completes before the memory is given up
            commit(leader, bar(kLast + i));
            __syncwarp();
            mbar_wait(bar(kLast + i), 0, &never);
        }
    } else if (warp >= 8 && warp != 13) {
        // ---------------- unpacking: 16 bytes of a position at once ----------------
        // A thread copies what it unpacks for the tile after this one (cp.async), and reads it back itself.
        // Three warps for keys and three for values, so that neither waits for the other's stage.  Piece e is piece e / 128 of row e % 128; the
        // rows of a thread agree in their last three bits, so what is exchanged is fixed.
        constexpr int kRounds = P::kRounds;
        const bool values = warp == 11 || warp > 13;
        const int first = (values ? max(warp - 13, 0) : warp - 8) * 32 + lane;
        const uint32_t mine = smem_u32(raw) + (values ? P::kRawSide : 0), mine_par = mine + kRounds * kUnpackThreads * 16, turn = (lane & 3) << 4;
        const uint32_t tile0 = smem_u32(values ? vs : ks);
        const int full = values ? kVFull : kKFull, empty = values ? kVEmpty : kKEmpty;
        const uint8_t* codes = values ? a.c.vc : a.c.kc;
        const half2* params = values ? a.c.vp : a.c.kp;
        W w(a, whole, start);
        uint32_t n = 0;
        bool ok = true;
        while (ok && w.advance()) {
            size_t at = cache_row(a.c, w.b, w.head, w.j0 * kTile);           // of the tile to be copied
            const auto load = [&](int j) {
                const int left = w.visible - j * kTile;                     // positions behind hold anything: they become 0
#pragma unroll
                for (int k = 0; k < kRounds; k++) {
                    const int e = first + k * kUnpackThreads, c = e / kTile, row = e % kTile;
                    if (k < kRounds - 1 || e < kCodes * kTile) {
                        const bool valid = row < left;
                        const size_t from = at + (valid ? row : 0);
                        copy_async<16>(mine + e * 16, codes + from * (DIM / 2) + c * 16, valid);
                        copy_async<4>(mine_par + e * 4, params + from * P::kBlocks + c / 2, valid);
                    }
                }
                at += kTile;
            };
            load(w.j0);
            for (int j = w.j0; j < w.j1; j++, n++) {
                const uint32_t st = n & 1;
                asm volatile("cp.async.wait_all;" ::: "memory");
                if (!(ok = mbar_wait(bar(empty + st), ((n >> 1) & 1) ^ 1, abortp))) break;
                const uint32_t to = tile0 + st * P::kOperand;
#pragma unroll
                for (int k = 0; k < kRounds; k++) {
                    const int e = first + k * kUnpackThreads, c = e / kTile;
                    if (k < kRounds - 1 || e < kCodes * kTile) {
                        uint4 code;
                        uint32_t par;
                        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(code.x), "=r"(code.y), "=r"(code.z), "=r"(code.w) : "r"(mine + e * 16) : "memory");
                        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(par) : "r"(mine_par + e * 4) : "memory");
                        unpack32(to + (c >> 1) * kBlock + e % kTile * 128 + (((c & 1) ^ (lane >> 2 & 1)) << 6), turn, code, *reinterpret_cast<const half2*>(&par));
                    }
                }
                fence_async();
                mbar_arrive(bar(full + st));
                if (j + 1 < w.j1) load(j + 1);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
        if (!ok) abort_flag = 1;
    } else if (warp < 4 * ROW_TILES) {
        // ---------------- softmax: a row a thread ----------------
        const int i = warp >> 2, row = tid & (kTile - 1);
        // Sequences of a call whose `first` falls may share rows: nothing is written then, as Work::find has it for work that is cut.  The 128 threads
        // share the comparisons; each reads the others' answer behind kSFull, which comes behind their kQFull.
        const bool mine = whole && row < a.s.batch;
        const int from = mine ? a.s.first[row] : 0, upto = mine ? a.s.first[row + 1] : 0;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, row_s = tmem + i * kTile + lanes, row_o = tmem + ROW_TILES * kTile + i * DIM + lanes;
        W w(a, whole, start);
        if (upto < from) *fallsp = 1;
        if (whole)
            for (int k = row + kTile; k < a.s.batch; k += kTile)
                if (a.s.first[k + 1] < a.s.first[k]) *fallsp = 1;
        const bool wide = ((reinterpret_cast<uintptr_t>(out.p) | (uintptr_t)out.ld * sizeof(T)) & 31) == 0;     // outputs on whole sectors
        uint32_t rounds = 0;
        bool ok = true;
        while (ok && w.advance()) {
            const int tile_rows = w.tile_rows(i), r = w.tile * kRows + i * kTile + row;
            if (tile_rows <= 0) continue;
            const bool there = row < tile_rows;
            const int token = there ? r / w.per : 0, head = w.head * w.per + (there ? r % w.per : 0);
            const int sees = there ? w.span.position(token) + 1 : 0, least = w.span.position((r - row) / w.per) + 1;
            // ---- the warp's rows of queries, with the sign of the scale: kLanes lanes take a row, whole sectors at a time ----
            constexpr int kLanes = DIM / 8, kAtOnce = 32 / kLanes;
            const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;
            const auto piece = [&](int k) {
                const int at = (warp & 3) * 32 + k * kAtOnce + lane / kLanes;
                return qs + i * P::kOperand + (lane % kLanes >> 3) * kBlock + at * 128 + (((lane & 7) ^ (at & 7)) << 4);
            };
            int at0 = (warp & 3) * 32 + lane / kLanes, tok = (w.tile * kRows + i * kTile + at0) / w.per, sub = (w.tile * kRows + i * kTile + at0) - tok * w.per;
#pragma unroll 2
            for (int k = 0; k < 32 / kAtOnce; k++, at0 += kAtOnce, sub += kAtOnce) {
                for (; sub >= w.per; sub -= w.per) tok++;
                const bool valid = at0 < tile_rows;
                const T* src = q.p + (size_t)(w.span.row0 + (valid ? tok : 0)) * q.ld + (size_t)(w.head * w.per + (valid ? sub : 0)) * DIM + lane % kLanes * 8;
                copy_async<16>(smem_u32(piece(k)), src, valid);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (!std::is_same<T, half>::value || sign) {
                // a lane changes what it copied.  BF16 numbers become FP16 ones times a power of two of their row, the largest from 2^14 on:
                // their exponents order the sizes
#pragma unroll 4
                for (int k = 0; k < 32 / kAtOnce; k++) {
                    const uint4 v = *reinterpret_cast<const uint4*>(piece(k));
                    uint32_t x[4] = {v.x ^ sign, v.y ^ sign, v.z ^ sign, v.w ^ sign};
                    if constexpr (!std::is_same<T, half>::value) {
                        uint32_t top = 0;
#pragma unroll
                        for (int e = 0; e < 4; e++) top = max(top, max(x[e] & 0x7f80u, x[e] >> 16 & 0x7f80u));
#pragma unroll
                        for (int d = 1; d < kLanes; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
                        const int exponent = (int)(top >> 7) - 127, sh = exponent == 128 || top == 0 ? 0 : min(14 - exponent, 126);
                        const float up = __int_as_float((127 + sh) << 23);
#pragma unroll
                        for (int e = 0; e < 4; e++) x[e] = Pair2<half>::of(__uint_as_float(x[e] << 16) * up, __uint_as_float(x[e] & 0xffff0000u) * up);
                        if (lane % kLanes == 0) row_scale[i * kTile + (warp & 3) * 32 + k * kAtOnce + lane / kLanes] = __int_as_float((127 - sh) << 23);
                    }
                    *reinterpret_cast<uint4*>(piece(k)) = make_uint4(x[0], x[1], x[2], x[3]);
                }
            }
            if constexpr (P::kQueryCols > 0) {
                __syncwarp();
                uint32_t x[32];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint4 v = *reinterpret_cast<const uint4*>(qs + i * P::kOperand + row * 128 + ((e ^ (row & 7)) << 4));
                    x[4 * e] = v.x, x[4 * e + 1] = v.y, x[4 * e + 2] = v.z, x[4 * e + 3] = v.w;
                }
                tmem_st32(tmem + ROW_TILES * (kTile + DIM) + i * P::kQueryCols + lanes, x);
                wait_st();
                fence_before();
            } else {
                fence_async();
            }
            __syncwarp();
            mbar_arrive(bar(kQFull + i));
            float scale2 = fabsf(a.scale) * kLog2e;
            if constexpr (!std::is_same<T, half>::value) scale2 *= row_scale[i * kTile + row];
            scale2 = fmaxf(scale2, 1e-37f);                                 // a masked score times it stays -infinity
            const f32x2 scale = pair_f32(scale2, scale2);
            float m = -INFINITY, l = 0.f;
            for (int j = 2 * w.j0; j < 2 * w.j1; j++) {
                const int h = j & 1, u = i + 2 * h;
                const uint32_t at_s = row_s + h * kHalf, parity = rounds & 1;
                rounds += h;
                ok = __all_sync(0xffffffffu, mbar_wait(bar(kSFull + u), parity, abortp));
                if (!ok) break;
                fence_after();
                const int seen = sees - j * kHalf;
                const bool masked = (j + 1) * kHalf > least;                // some (row, position)
                float mx;
                {
                    uint32_t s[2][32];
                    tmem_ld32(at_s, s[0]);
                    tmem_ld32(at_s + 32, s[1]);
                    wait_ld();
                    if (masked) {
#pragma unroll
                        for (int k = 0; k < kHalf; k++)
                            if (k >= seen) s[k / 32][k % 32] = 0xff800000u;
                    }
                    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < 32; k++) top[k / 16] = max3(top[k / 16], __uint_as_float(s[k / 16][k % 16 * 2]), __uint_as_float(s[k / 16][k % 16 * 2 + 1]));
                    mx = max3(top[0], top[0], top[1]) * scale2;
                }
                const bool grows = !(mx <= m + kSlack);                     // a row's result does not depend on the others' of its warp
                if (__any_sync(0xffffffffu, grows)) {
                    const float f = grows ? exp2_neg(m - mx) : 1.f;         // 0 where nothing was seen before
                    if (grows) {
                        m = mx;
                        l *= f;
                    }
                    if (!(mx < INFINITY)) l = NAN;                          // a score that is no number
                    if (j > 2 * w.j0) {
                        // the output of the half before may be under way
                        ok = __all_sync(0xffffffffu, mbar_wait(bar(kPvDone + i + 2 * (h ^ 1)), h ? parity : parity ^ 1, abortp));
                        if (!ok) break;
                        fence_after();
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
                // The scores are read again, 32 at once: kept since the search for the maximum they take the registers that exponentials ahead
                // of their use need (512 behind 16000 158 us, 148.5 read again, 16 at once 156).
                const float ref = kLift - (m == -INFINITY ? 0.f : m);
                const f32x2 off = pair_f32(ref, ref);
                f32x2 sum[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < kHalf; c += 32) {
                    uint32_t s[32], pw[16];
                    tmem_ld32(at_s + c, s);
                    wait_ld();
                    if (masked) {
#pragma unroll
                        for (int k = 0; k < 32; k++)
                            if (c + k >= seen) s[k] = 0xff800000u;
                    }
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        const float2 e = split_f32(fma_pairs(pair_f32(s[2 * k], s[2 * k + 1]), scale, off));
                        const float x = exp2_neg(e.x), y = exp2_neg(e.y);
                        sum[k & 1] = add_pair(sum[k & 1], pair_f32(x, y));
                        pw[k] = Pair2<half>::of(x, y);
                    }
                    tmem_st16(at_s + c / 2, pw);                            // over scores that were read
                }
                l += sum_pair(add_pair(sum[0], sum[1]));
                wait_st();
                fence_before();
                mbar_arrive(bar(kPReady + u));
            }
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(kPvDone + i + 2), (rounds - 1) & 1, abortp));
            if (!ok) break;
            fence_after();
            T* y = out.p + (size_t)(w.span.row0 + token) * out.ld + (size_t)head * DIM;
            const int at = i * kTile + row;
            const bool complete = w.complete();
            float* rec = complete ? nullptr : record_of<DIM, kRows>(a.ws, gridDim.x, blockIdx.x, w.segment > 0);
            if (!complete && w.j0 == 0 && tid == 0)
                *entry_of(a.ws, blockIdx.x) =
                    Shared4{w.owner(w.x - 1) - (int)blockIdx.x + 1, w.segment > 0, w.head, w.tile, w.span.row0, w.span.n, w.span.len, 0};
            if (!complete && there) {
                rec[at] = m;
                rec[kRows + at] = l;
            }
            const float f = sees > 0 ? 1.f / l : 0.f;
            const bool stores = there && !*fallsp;
#pragma unroll 1
            for (int c = 0; c < DIM; c += 32) {
                uint32_t o[32];
                tmem_ld32(row_o + c, o);
                wait_ld();
                if (stores && complete) {
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        p[e] = sees > 0 ? Pair2<T>::of(__uint_as_float(o[2 * e]) * f, __uint_as_float(o[2 * e + 1]) * f) : 0u;
                    if (wide) {
                        store32(y + c, p);
                        store32(y + c + 16, p + 8);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) reinterpret_cast<uint4*>(y + c)[e] = make_uint4(p[4 * e], p[4 * e + 1], p[4 * e + 2], p[4 * e + 3]);
                    }
                } else if (stores) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) store32(rec + 2 * kRows + at * DIM + c + e, o + e);
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

template <typename T, int DIM, int ROW_TILES>
int launch(const Cache4Call& a, Rows<const T> q, Rows<T> out, const PromptPlan& p, cudaStream_t stream)
{
    static bool attr[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return fail(TLLM_ERR_LAUNCH, "cache4_prompt: no current device");
    const auto kernel = cache4_prompt_kernel<T, DIM, ROW_TILES>;
    if (!attr[dev]) {
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Prompt<DIM, ROW_TILES>::kSmem);
        attr[dev] = true;
    }
    const int st = launch_pdl("cache4_prompt", kernel, dim3(p.ctas), dim3(kThreads), Prompt<DIM, ROW_TILES>::kSmem, stream, a, q, out, p.whole);
    return st || p.whole ? st : launch_cache4_join<T>(a, out, p.rows, p.ctas, stream);
}

}  // namespace

PromptPlan prompt_plan(const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    PromptPlan p;
    const int per = heads / c.kv_heads, most = max_new > 0 && max_new < tokens ? max_new : tokens, len = max_len > 0 && max_len < c.rows ? max_len : c.rows;
    const double longest = (len + kTile - 1) / kTile, mean = longest - (most < len ? most : len) / (2.0 * kTile);
    // Tiles of `rows` rows, where every sequence has as many rows as it may.
    const auto tiles_of = [&](int rows) {
        const double by_tokens = (double)tokens * per / rows + c.batch, by_most = (double)c.batch * (((long long)most * per + rows - 1) / rows);
        return (by_tokens < by_most ? by_tokens : by_most) * c.kv_heads;
    };
    // Whole tiles take CTAs for as many in every sequence as one may have, and 0.02 us a CTA that finds none: us, 32 heads of 128 over 8, whole / cut,
    // 2000 tokens beside 3 single ones (740 such CTAs) 68 / 78, 15 (3700) 117 / 90, nine prompts of unknown length (3800) 137 / 117, 4000 beside 63 (31000) 630 / 256.
    const long long pairs = (long long)c.batch * c.kv_heads;
    const auto grid_of = [&](int rows) {
        const long long grid = ((long long)most * per + rows - 1) / rows * pairs;
        return grid < (1 << 20) ? grid : (1 << 20) / pairs * pairs;
    };
    const auto idle = [&](int rows) { return fmax(grid_of(rows) - ((double)tokens * per / rows + c.batch) * c.kv_heads, 0.0); };
    if (tiles_of(128) <= 148) {
        // An SM for each tile of 128 rows: the quickest of these tiles whole, cut, and tiles of 256 rows cut, as they measure, us: 8 + 1.9 for each
        // tile of positions, or 19 + 1.85 for each that a CTA takes, or 27 + 2.35; sequences of a batch differ, so that cut ones have fewer.
        // 32 heads of 128 over 8, one sequence: 79 tokens behind 500 15.1 / 20.4 / 24.8, behind 2500 40.7 / 21.6 / 27.8, behind 16000 209 / 51 /
        // 54; 500 behind 1200 30.4 / 40.2 / 38.2, behind 6000 90 / 95 / 75.  Tiles of 256 whole take 18.7, 52.2, 268, 37.2 and 116.
        const double few = c.batch > 1 ? 0.85 : 1;
        const auto cut = [&](int rows) { return fmax(tiles_of(rows) * (few * mean + Work<128, kTile>::kFixed) / 148, (double)Work<128, kTile>::kLeast); };
        const double whole = 8 + 1.9 * longest + idle(128) / 75, halves = 19 + 1.85 * cut(128), full = 27 + 2.35 * cut(256);
        p.rows = full < fmin(whole, halves) ? 256 : 128;
        p.whole = whole <= fmin(halves, full);
    } else {
        // A tile of rows stays in one CTA unless the longest would keep its SM busy for more than seven tiles of positions (some 2 us each) after
        // the others are done, which is what cutting costs in records and a second launch.  Both ways, us, 32 heads over 8: of 128, a prompt of
        // 1500 34 whole, 50 cut, 2000 48 / 69; of 64, four prompts of 700 34 / 43.
        const double rows = (double)tokens * per / 256 > (double)c.batch ? (double)tokens * per / 256 : (double)c.batch;
        p.rows = 256;
        p.whole = longest - rows * c.kv_heads * mean / 148 <= 7 && idle(256) <= 1500;
    }
    p.whole = p.whole || !work_fits(c, tokens, heads, len, p.rows, kTile, false);
    p.ctas = p.whole ? (int)fmax(grid_of(p.rows), pairs) : 148;
    p.bytes = p.whole ? 0 : join_bytes(c.dim, p.rows, p.ctas);
    return p;
}

template <typename T, int DIM>
static int launch_rows(const Cache4Call& a, Rows<const T> q, Rows<T> out, const PromptPlan& p, cudaStream_t stream)
{
    return p.rows == kTile ? launch<T, DIM, 1>(a, q, out, p, stream) : launch<T, DIM, 2>(a, q, out, p, stream);
}

template <typename T>
int launch_cache4_prompt(const Cache4Call& a, Rows<const T> q, Rows<T> out, const PromptPlan& p, cudaStream_t stream)
{
    return a.c.dim == 64 ? launch_rows<T, 64>(a, q, out, p, stream) : launch_rows<T, 128>(a, q, out, p, stream);
}

template int launch_cache4_prompt<half>(const Cache4Call&, Rows<const half>, Rows<half>, const PromptPlan&, cudaStream_t);
template int launch_cache4_prompt<bf16>(const Cache4Call&, Rows<const bf16>, Rows<bf16>, const PromptPlan&, cudaStream_t);

}  // namespace tllm
