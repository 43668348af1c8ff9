// attend.cu — kvops_attend_hot: attention of drafted tokens over the hot rows that their top-K
// lists name and over one another's drafted rows along a tree (the formulas are in
// include/kvops_b200.h).
//
// A key row is read once for its score and its value, and every head and drafted token of a
// request shares it, so both products are matrix products over tiles of 64 keys:
//   S^T [64 keys x NQ queries] = K [64 x 576] Q^T,   O^T [512 x NQ] += V^T [512 x 64] P^T,
// with V the first 512 columns of K: one copy of the rows in shared memory serves both, K-major for
// the first and MN-major for the second. The transposed form keeps the matrix unit's 128 rows full of
// value dimensions for any number of queries: with the queries as rows, a tile of 64 would run at half
// rate, and 128 rows of 512 fp32 outputs would fill tensor memory and leave no room for the scores.
// Operands come from shared memory at 128 bytes a cycle, which bounds both products: 48 cycles for
// 16 dimensions (or keys) at NQ = 64, 36 + 16 of them a tile. Tiles of 128 keys would take 48 cycles
// for twice the keys in the first product, but leave no room for a second tile beside the queries:
// rows, products and softmax then take turns (12200 cycles for 128 keys, where this takes 2 x 3300).
//
// One CTA per SM takes a run of (query tile, key tile) pairs. Warps 0-7: the softmax, a thread for two keys
// and two of each eight queries of its half, and the outputs. Warps 8-15: the rows, by asynchronous 16-byte
// copies, four rows of 128 bytes an instruction (38 bytes a cycle and SM; gathering tensor copies of the
// same 512 bytes reach 48 alone, but cost the thread that issues them 190 cycles each beside the other
// warps, which left 18). 16-bit rows land where the products read them; stored rows' codes land in a
// warp's own place and are converted from there. Warps 16 and 17 issue the two products: the first of the
// next tile goes ahead of the second of this one, whose probabilities the softmax is still working out.
// Warp 18 finds the rows that the lists name, a few tiles ahead. (Their lines prefetched into L2 from there
// gave 2% at NQ = 64 and cost up to 10% elsewhere.) A key tile is four groups of 128 dimensions (16 KB)
// and the 64 rotary dimensions (8 KB). The groups go through a ring of places that the second product
// frees one by one, so rows travel while earlier ones are still in use.
//
// Measured, 2048 keys a request (here and below without the call from Python: a captured graph of 20 launches):
// 64 requests x 128 heads, fp16 rows, 65 us (2.6 TB/s, 563 TFLOP/s; 3300 cycles a tile, of which the operands take
// 2500, and 20 of 148 SMs have no list); four tokens each 253 us (577 TFLOP/s); 64 requests x 16 heads
// 37 us (154 MB, 4.2 TB/s), with 8-bit rows 45 us: a load warp has one place for codes, so the next tile's are
// fetched behind the conversion of this one's only, 1450 of 3700 cycles a tile; one request x 128 heads
// 13 us, chains of loads (the count, the slots, the rows), two products, the outputs and the joining.
#include <cuda_runtime.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include <string>
#include <type_traits>

#include "kvops_internal.cuh"
#include "quant.cuh"
#include "tcgen05.cuh"

namespace kvb {
namespace {

constexpr int kValueDim = 512;          // values of a row that the output sums
constexpr int kKeyDim = 576;            // values of a row that the scores use
constexpr uint32_t kStoredBytes = 656;  // of a stored row of 512 + 64 values
constexpr uint32_t kStoredPlain = 528;  // where its 64 rotary values start
constexpr int kTile = 64;               // keys per tile
constexpr uint32_t kChunkBytes = kTile * 128;  // 64 dimensions of a tile's keys, in 128-byte rows
constexpr uint32_t kGroupBytes = 2 * kChunkBytes;
constexpr int kSoftmaxWarps = 8;

constexpr int kLoadWarps = 8;
constexpr int kScoreWarp = kSoftmaxWarps + kLoadWarps, kWeighWarp = kScoreWarp + 1, kFindWarp = kScoreWarp + 2;
constexpr int kThreads = (kFindWarp + 1) * 32;  // five warps to a scheduler leave a thread 96 registers, six 80
constexpr uint32_t kAhead = 4;  // tiles whose rows are known at a time

// A column's running reference: probabilities are 2^(score - reference), and it is set Plan::lift (in powers of
// two) below the largest score so far when a score passes it by kMost. They stay below 2^kMost, which is an
// fp16 number; moving the reference means scaling the outputs in tensor memory, so it should be rare: what a
// later score may exceed the first tile's largest by is kMost less the lift. (Normal scores of variance 3,
// as of unit-variance queries and rows, 64 requests x 128 heads: 4 of it 106 us, 11 of it 81.)
// fp16's smallest step is 2^-24: each probability that the second product takes is off by 2^-25 at the most
// besides its relative rounding (those below become 0), while the sum, which has them in fp32, is 2^lift or
// more. n keys all rounded the same way are off by n 2^-(25 + lift) of the largest value: with a lift of 4, 2^-13 for
// 2^16 keys, below the output's own rounding. n counts the keys of one CTA's part, each of which has its own
// references; where that can be more, the lift is 14, which leaves 2^-15 for 2^24 keys. (It costs less the longer
// a part is: in us with 4 and 14, 64 requests x 128 heads, 32 tiles a part, 65 and 94; 8 requests x 16 heads x 2^17 keys,
// 111 tiles, 197 and 203; 148 requests x 16 heads x 2^17, 2048 tiles, 2906 and 2913.)
// bf16 has the range of fp32: what is lost is below 2^-121 of the largest.
constexpr float kMost = 15.f;
constexpr float kLiftFp16 = 4.f, kLiftFp16Long = 14.f, kLiftBf16 = -5.f;
constexpr uint32_t kLongPart = 1u << 16;

// How the (query tile, key tile) pairs are dealt out. Units are query tiles: group (a request, or a
// request's token where every token has its own list) by group.
struct Plan {
    uint32_t lists;       // lists per request: 1, or tokens
    uint32_t group_rows;  // query rows that share a list
    uint32_t qtiles;      // query tiles per group
    uint32_t list_end;    // top_k rounded up to four: where the drafted rows start among the keys
    uint32_t tiles;       // key tiles per unit
    uint32_t ctas;
    uint32_t run_at_most; // pairs of a run, with every request real
    float lift;           // see kMost
    uint32_t whole;       // > 0: every CTA takes this many whole units; 0: runs of pairs of one length
    float2 *part_ml;      // [2 * ctas][NQ] reference and sum of a unit's part
    float *part_o;        // [2 * ctas][NQ * 512] its weighted sums, in part_at's order
};

// Where (as float4) a part keeps the sums of dimension block * 128 + quarter * 32 + lane of the four
// queries 4 i .. 4 i + 3 of a half: the order in which the softmax warps hold them.
template <int NQ>
__device__ __forceinline__ uint64_t part_at(uint32_t slot, uint32_t block, uint32_t quarter, uint32_t half, uint32_t i,
                                            uint32_t lane)
{
    return ((((static_cast<uint64_t>(slot) * 4 + block) * 4 + quarter) * 2 + half) * (NQ / 8) + i) * 32 + lane;
}

__device__ __forceinline__ uint32_t real_units(const KvopsAttend &a, const Plan &p)
{
    const int32_t n = *reinterpret_cast<const int32_t *>(a.num_real);
    const uint32_t reqs = n < 0 ? 0u : min(static_cast<uint32_t>(n), a.max_num_reqs);
    return reqs * p.lists * p.qtiles;
}

// Pairs of a CTA's run; CTA c has those from c * run_length on.
__device__ __forceinline__ uint32_t run_length(const Plan &p, uint32_t units)
{
    return p.whole > 0 ? p.whole * p.tiles : (units * p.tiles + p.ctas - 1) / p.ctas;
}

struct Unit {
    uint32_t req;       // batch row
    uint32_t token;     // its token, where every token has its own list
    uint32_t row0;      // first query row within the group
    uint32_t rows;      // query rows (at most NQ)
    uint64_t out_row;   // output row of query row row0
};

template <int NQ>
__device__ __forceinline__ Unit unit_at(const Plan &p, uint32_t unit)
{
    Unit u;
    const uint32_t group = unit / p.qtiles;
    u.req = group / p.lists;
    u.token = group - u.req * p.lists;
    u.row0 = (unit - group * p.qtiles) * NQ;
    u.rows = min(static_cast<uint32_t>(NQ), p.group_rows - u.row0);
    u.out_row = static_cast<uint64_t>(group) * p.group_rows + u.row0;
    return u;
}

// The token of query row `row` of a unit's group (its head is the remainder).
__device__ __forceinline__ uint32_t token_of(const KvopsAttend &a, const Plan &p, const Unit &u, uint32_t row)
{
    return p.lists > 1 ? u.token : row / a.heads;
}

// Shared memory: a ring of groups, the rotary dimensions of two tiles, the queries, and for stored
// rows the codes of a tile, 32 rows x 128 bytes of it each load warp's own. A tile's probabilities [64 keys]
// [64 x 16 bit] take the place of its rotary dimensions, which only the scores need.
template <int NQ, bool kStored>
struct Layout {
    // as many as fit beside the queries; a tile has four groups
    static constexpr int places = kStored ? (NQ == 64 ? 6 : 8) : NQ == 64 ? 8 : NQ == 32 ? 10 : 11;
    static constexpr uint32_t rope = places * kGroupBytes;
    static constexpr uint32_t q = rope + 2 * kChunkBytes;
    static constexpr uint32_t stage = q + NQ * 2 * kKeyDim;
    static constexpr uint32_t bytes = stage + (kStored ? kTile * kValueDim : 0) + 1024;
    static_assert(bytes + 6 * 1024 <= 227 * 1024, "with the static part");
};
constexpr int kMostPlaces = 11;

struct Shared {
    alignas(16) float per_warp[kSoftmaxWarps][32];  // read four at a time
    float top[2][4][32];       // a tile's maxima by column, by half and lane quarter
    uint64_t tree[64];         // of the unit's query rows
    // full: rows have landed; empty: the second product is done with them; done: with a tile; rope_*:
    // a tile's rotary dimensions, then probabilities
    uint64_t q_full, full[kMostPlaces], empty[kMostPlaces], rope_full[2], rope_empty[2], s_full[2], p_full[2], done[2],
        meta_full[kAhead], meta_empty[kAhead];
    uint64_t row[kAhead][kTile];  // where the tile's hot rows start, 0: no hot row
    uint8_t kind[kAhead][kTile];  // of the tile's keys: kNone, kList, kDraft or kBadDraft
    // 0 for a tile without any key, else kKeys | lo << 8 | hi << 16: rows 4 lo .. 4 hi - 1 are drafted ones
    uint32_t tile[kAhead];
    uint64_t drained[2];  // the products of the score and the weigh warp
    uint32_t tmem, stop;  // stop: a wait has given up
};
enum : uint8_t { kNone = 0, kList = 1, kDraft = 2, kBadDraft = 3 };

__device__ __forceinline__ void group_barrier(int id, int threads)
{
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool group_any(int id, int threads, bool mine)
{
    uint32_t r;
    asm volatile("{ .reg .pred p, q; setp.ne.u32 p, %3, 0; bar.red.or.pred q, %1, %2, p; selp.u32 %0, 1, 0, q; }"
                 : "=r"(r) : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(mine)) : "memory");
    return r != 0;
}

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Of the threads of a warp with the same columns (those whose lanes differ in bits 2-4), the largest
// values or the sums; returns the one of the thread's own column, number `own`.
template <bool kMax, int kN>
__device__ __forceinline__ float join_columns(float (&v)[kN], int own)
{
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
#pragma unroll
        for (int w = 4; w < 32; w *= 2) {
            const float other = __shfl_xor_sync(0xFFFFFFFFu, v[i], w);
            v[i] = kMax ? fmaxf(v[i], other) : v[i] + other;
        }
        if (own == i) mine = v[i];
    }
    return mine;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool some)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(some ? 16u : 0u) : "memory");
}
// An arrival of this thread once all its copies so far have landed.
__device__ __forceinline__ void copies_arrive(uint32_t bar)
{
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void copy_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void store16(uint32_t dst, const uint4 &v)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Whether any of eight 16-bit values is inf or NaN.
template <typename T>
__device__ __forceinline__ bool not_finite(const uint4 &v)
{
    const uint32_t m = T::kInf | (T::kInf << 16);
    return (__vcmpeq2(v.x & m, m) | __vcmpeq2(v.y & m, m) | __vcmpeq2(v.z & m, m) | __vcmpeq2(v.w & m, m)) != 0;
}

// ---- the rows ----------------------------------------------------------------------------------

// A place in the ring of groups and the parity of its use.
template <int kPlaces>
struct Ring {
    uint32_t place = 0, turn = 0;
    __device__ __forceinline__ void next()
    {
        if (++place == kPlaces) {
            place = 0;
            ++turn;
        }
    }
};

// The unit's queries, K-major in blocks of 64 dimensions, rows behind the last as zeros; warp w takes rows w,
// w + 8, ... The run's first unit's are always loaded, before its rows are known; a later unit's with its
// first tile that has a key, once the `done` tiles before are done with the place (or, if there were
// none, once the first unit's are there).
template <int NQ>
__device__ __forceinline__ void load_queries(const KvopsAttend &a, const Plan &plan, Shared &sh, uint32_t q_at,
                                             const Unit &u, bool later, uint32_t done, int warp, int lane)
{
    using namespace tc;
    uint64_t from = 0;  // lane i: where row w + 8 i starts, 0: none
    {
        const uint32_t r = warp + kLoadWarps * lane, row = u.row0 + r;
        if (r < u.rows) {
            const uint32_t t = token_of(a, plan, u, row), h = plan.lists > 1 ? row : row - t * a.heads;
            from = a.q + 2 * (u.req * a.q_stride_req + t * a.q_stride_token + h * a.q_stride_head);
        }
    }
    if (later && done > 0) mbar_wait(smem_addr(&sh.s_full[(done - 1) & 1]), ((done - 1) >> 1) & 1, &sh.stop);
    else if (later) mbar_wait(smem_addr(&sh.q_full), 0, &sh.stop);
#pragma unroll 4
    for (int i = 0; i < NQ / kLoadWarps; ++i) {
        const uint64_t row = __shfl_sync(0xFFFFFFFFu, from, i);
        const uint32_t r = warp + kLoadWarps * i;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const uint32_t c = k * 32 + lane;
            if (c < 72)
                copy16(q_at + (c >> 3) * (NQ * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                       reinterpret_cast<const uint8_t *>(row != 0 ? row + c * 16 : a.q), row != 0);
        }
    }
    copies_arrive(smem_addr(&sh.q_full));
}

__device__ __forceinline__ const int32_t *list_of(const KvopsAttend &a, const Unit &u)
{
    return reinterpret_cast<const int32_t *>(a.topk_device_slots) + u.req * a.slots_stride_req +
           u.token * a.slots_stride_token;
}
__device__ __forceinline__ const uint8_t *draft_row(const KvopsAttend &a, const Unit &u, uint32_t j)
{
    return reinterpret_cast<const uint8_t *>(a.draft_rows) + 2 * (u.req * a.draft_stride_req + j * a.draft_stride_row);
}

// 16 bytes of a drafted row. Not every query sees it: a value that is not finite would turn their
// zero probability into NaN, so it is left out and the row marked.
template <typename T>
__device__ __forceinline__ uint4 draft_unit(const uint8_t *from, uint8_t *kind)
{
    uint4 v = *reinterpret_cast<const uint4 *>(from);
    if (not_finite<T>(v)) {
        v = make_uint4(0u, 0u, 0u, 0u);
        *kind = kBadDraft;
    }
    return v;
}

constexpr uint32_t kKeys = 1, kOver = 2;  // of a tile's word: it has a key; no tile, a wait has given up
// Whether a wait of the CTA has given up (the lanes may see it at different times).
__device__ __forceinline__ bool given_up(const Shared &sh)
{
    return *const_cast<const volatile uint32_t *>(&sh.stop) != 0;
}

// The rows of each tile, for the other warps: lane l looks at keys l and l + 32.
template <int NQ, bool kStored>
__device__ __forceinline__ void find_warp(const KvopsAttend &a, const Plan &plan, Shared &sh, uint32_t begin, uint32_t end)
{
    using namespace tc;
    constexpr uint32_t kRowBytes = kStored ? kStoredBytes : 2 * kKeyDim;
    const int lane = threadIdx.x & 31;
    uint32_t unit = begin / plan.tiles, tile = begin - unit * plan.tiles;  // the next to fetch
    const int32_t *list = nullptr;
    const int64_t *pool_at = nullptr;
    const auto enter = [&]() {
        const Unit u = unit_at<NQ>(plan, unit);
        list = list_of(a, u);
        pool_at = reinterpret_cast<const int64_t *>(a.req_pool_indices) + u.req;
    };
    // A tile on its way: its request's pool index and two slots, as they come from memory. Nothing is
    // worked out of them before its turn: a warp stands still at the first use of a load.
    struct Fetched {
        int64_t pool;
        int32_t slot[2];
        uint32_t tile;
    };
    const auto fetch = [&]() {
        Fetched f;
        f.pool = -1;
        if (a.top_k > 0) f.pool = *pool_at;
        f.tile = tile;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t k = tile * kTile + lane + 32 * j;
            f.slot[j] = -1;
            if (k < a.top_k) f.slot[j] = list[k];
        }
        if (++tile == plan.tiles) {
            tile = 0;
            ++unit;
            enter();
        }
        return f;
    };
    enter();
    Fetched next[2];  // two tiles on their way
    if (begin < end) next[0] = fetch();
    if (begin + 1 < end) next[1] = fetch();
    const long long limit = a.wait_clocks != 0 ? a.wait_clocks : kWaitClocks;
    bool behind = false;  // whether a slot named a row behind the request's last
    for (uint32_t at = begin, n = 0; at < end; ++at, ++n) {
        const Fetched f = next[0];
        next[0] = next[1];
        if (at + 2 < end) next[1] = fetch();
        const uint32_t buf = n % kAhead;
        if (n >= kAhead) {
            // The caller's limit is looked at here, where a wait lasts as long as the slowest warp's tile, and after
            // the wait, since the barrier instruction itself may take longer than a short limit. (The other
            // waits have a constant one: read from shared memory it cost 4%.)
            const long long start = clock64();
            mbar_wait(smem_addr(&sh.meta_empty[buf]), (n / kAhead - 1) & 1, &sh.stop);
            if (clock64() - start > limit) *const_cast<volatile uint32_t *>(&sh.stop) = 1u;
            __syncwarp();
        }
        if (__any_sync(0xFFFFFFFFu, given_up(sh))) break;
        const bool in_pool = f.pool >= 0 && f.pool < static_cast<int64_t>(a.pool_size);
        bool mine = false;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t k = f.tile * kTile + lane + 32 * j;
            const bool named = in_pool && f.slot[j] >= 0, listed = named && static_cast<uint32_t>(f.slot[j]) < a.hot_rows;
            const bool drafted = k >= plan.list_end && k - plan.list_end < a.drafts;
            sh.row[buf][lane + 32 * j] =
                listed ? a.hot_row_base + (f.pool * a.hot_req_stride_rows + f.slot[j]) * kRowBytes : 0;
            sh.kind[buf][lane + 32 * j] = listed ? kList : drafted ? kDraft : kNone;
            mine |= listed || drafted;
            behind |= named && !listed;
        }
        const bool any = __any_sync(0xFFFFFFFFu, mine);
        if (lane == 0) {
            const uint32_t t0 = f.tile * kTile;
            const uint32_t lo = plan.list_end <= t0 ? 0 : min(plan.list_end - t0, static_cast<uint32_t>(kTile));
            const uint32_t till = plan.list_end + ((a.drafts + 3) & ~3u);
            const uint32_t hi = a.drafts == 0 || till <= t0 ? lo : max(lo, min(till - t0, static_cast<uint32_t>(kTile)));
            sh.tile[buf] = any ? kKeys | (lo / 4) << 8 | (hi / 4) << 16 : 0u;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&sh.meta_full[buf]));
    }
    if (a.report_slots != 0 && __any_sync(0xFFFFFFFFu, behind) && lane == 0 && a.err_word != 0)
        atomicCAS_system(reinterpret_cast<uint32_t *>(a.err_word), 0u, KVOPS_ERR_ATTEND_SLOT);
}

// The word of the n-th tile of the run, once it is known, the same in every lane; and the end of its use.
// After a wait has given up it is kOver, which has no key: rows' addresses may never have been written. A warp that
// got it asks for no further tile, for which each time it would wait as long as the barrier instruction does.
__device__ __forceinline__ uint32_t tile_word(Shared &sh, uint32_t n)
{
    tc::mbar_wait(tc::smem_addr(&sh.meta_full[n % kAhead]), (n / kAhead) & 1, &sh.stop);
    const uint32_t word = *const_cast<volatile uint32_t *>(&sh.tile[n % kAhead]);
    return __shfl_sync(0xFFFFFFFFu, given_up(sh) ? kOver : word, 0);
}
__device__ __forceinline__ void tile_done(Shared &sh, uint32_t n, int lane)
{
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(tc::smem_addr(&sh.meta_empty[n % kAhead]));
}

// Copies 128 bytes from byte `column` of kFours fours of rows (from `from` on, an even four) of tile n to `to`,
// four rows an instruction, leaving out the fours [lo, hi); rows that are none become zeros.
template <int kFours>
__device__ __forceinline__ void copy_rows(const KvopsAttend &a, const Shared &sh, uint32_t n, int from, int lo, int hi,
                                          uint32_t to, uint32_t column)
{
    constexpr int kBatch = kFours < 8 ? kFours : 8;
    const uint32_t n16 = threadIdx.x & 7, r4 = threadIdx.x >> 3 & 3;
    const uint64_t *row = &sh.row[n % kAhead][4 * from + r4];
    const uint64_t add = column + n16 * 16;
    to += r4 * 128;
    const uint32_t even = (n16 ^ r4) << 4, odd = (n16 ^ (r4 + 4)) << 4;
#pragma unroll
    for (int b = 0; b < kFours; b += kBatch) {
        uint64_t at[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) at[i] = row[4 * (b + i)];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const bool some = at[i] != 0, skip = from + b + i >= lo && from + b + i < hi;
            if (!skip)
                copy16(to + (b + i) * 512 + ((b + i) & 1 ? odd : even),
                       reinterpret_cast<const uint8_t *>(some ? at[i] + add : a.q), some);
        }
    }
}

// Drafted rows' values from 64 * chunk on, of the fours from .. till of tile n, the tile-th of its unit, to `to`, where
// the tile's first row is; zeros behind the last row.
template <typename T>
__device__ __forceinline__ void bring_drafts(const KvopsAttend &a, const Plan &plan, Shared &sh, const Unit &u, uint32_t n,
                                             uint32_t tile, uint32_t to, uint32_t chunk, uint32_t chunks, int from, int till)
{
    for (uint32_t i = 4 * from * chunks * 8 + (threadIdx.x & 31); i < 4 * till * chunks * 8; i += 32) {
        const uint32_t c16 = i & 7, c = chunks == 2 ? i >> 3 & 1 : 0, r = chunks == 2 ? i >> 4 : i >> 3;
        const uint32_t j = tile * kTile + r - plan.list_end;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (j < a.drafts) v = draft_unit<T>(draft_row(a, u, j) + (chunk + c) * 128 + c16 * 16, &sh.kind[n % kAhead][r]);
        store16(to + c * kChunkBytes + r * 128 + ((c16 ^ (r & 7)) << 4), v);
    }
}

// Every lane's arrival, after its copies and (if any) the drafted rows that it stored itself.
__device__ __forceinline__ void rows_arrive(uint64_t *bar, bool stored_some)
{
    using namespace tc;
    if (stored_some) {
        copy_close();
        copy_wait<0>();
        fence_async_shared();
        mbar_arrive(smem_addr(bar));
    } else {
        copies_arrive(smem_addr(bar));
    }
}

// Load warp w brings, of 16-bit rows, chunk w (64 dimensions) of all 64 rows; of stored rows, the codes
// of group w / 2 of 32 rows, which it converts; and of either, the rotary dimensions of eight rows. (A warp of
// their own for these makes them late: they wait for the probabilities of the tile before last.) Drafted
// rows, whose first is at a multiple of four, come through registers.
template <typename T, typename Code, bool kStored, int NQ>
__device__ __forceinline__ void load_warps(const KvopsAttend &a, const Plan &plan, Shared &sh, uint32_t smem,
                                           uint32_t begin, uint32_t end)
{
    using namespace tc;
    using L = Layout<NQ, kStored>;
    const int warp = (threadIdx.x >> 5) - kSoftmaxWarps, lane = threadIdx.x & 31;
    const uint32_t group = warp >> 1, side = warp & 1;
    const uint32_t stage = smem + L::stage + warp * (32 * 128);
    float next_scale = 0.f;  // stored: of row 32 side + lane, group `group`, of the codes on their way
    const auto send = [&](uint32_t n, int lo, int hi) {  // the codes of this warp's rows of tile n, and their scales
        const uint64_t mine = sh.row[n % kAhead][side * 32 + lane];
        next_scale = 0.f;
        // (not the read-only path: the kernel ahead may write the rows while this one has begun and waits)
        if (mine != 0) next_scale = reinterpret_cast<const float *>(mine + kValueDim)[group];
        copy_rows<8>(a, sh, n, side * 8, lo, hi, stage, group * 128);
        copy_close();
    };

    uint32_t unit = begin / plan.tiles, tile = begin - unit * plan.tiles, done = 0;
    Unit u = unit_at<NQ>(plan, unit);
    Ring<L::places> ring;  // of group 0 of the tile
    bool q_loaded = false, sent = false;  // sent: the tile's codes are on their way
    if (begin < end) {
        load_queries<NQ>(a, plan, sh, smem + L::q, u, false, 0, warp, lane);
        q_loaded = true;
    }
    for (uint32_t at = begin, n = 0; at < end; ++at, ++n) {
        const uint32_t word = tile_word(sh, n);
        if ((word & kKeys) != 0) {
            const int lo = word >> 8 & 0xFF, hi = word >> 16;
            const bool first = !q_loaded;
            q_loaded = true;
            const auto bring_rope = [&]() {
                // the place was the probabilities' of the tile before last
                const uint32_t half = done & 1, rope = smem + L::rope + half * kChunkBytes;
                if (done > 1) mbar_wait(smem_addr(&sh.rope_empty[half]), ((done >> 1) - 1) & 1, &sh.stop);
                copy_rows<2>(a, sh, n, 2 * warp, lo, hi, rope + warp * 1024, kStored ? kStoredPlain : 2 * kValueDim);
                const int from = max(lo, 2 * warp), till = min(hi, 2 * warp + 2);
                if (from < till) bring_drafts<T>(a, plan, sh, u, n, tile, rope, 8, 1, from, till);
                rows_arrive(&sh.rope_full[half], from < till);
            };
            // this warp's group and its place
            uint32_t place = ring.place + group, turn = ring.turn;
            if (place >= L::places) {
                place -= L::places;
                ++turn;
            }
            uint64_t *full = &sh.full[place];
            if constexpr (kStored) {
                if (!sent) send(n, lo, hi);
                if (first) load_queries<NQ>(a, plan, sh, smem + L::q, u, true, done, warp, lane);
                copy_wait<0>();
                __syncwarp();
                uint4 code[8];
                const uint32_t r = side * 32 + lane;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(code[i].x), "=r"(code[i].y), "=r"(code[i].z), "=r"(code[i].w)
                                 : "r"(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) : "memory");
                const float scale = next_scale;
                __syncwarp();
                bring_rope();  // ahead of the codes, whose landing its arrival would wait for as well
                sent = false;
                if (at + 1 < end) {  // the next tile's, into the place that was just read
                    const uint32_t w = tile_word(sh, n + 1);
                    sent = (w & kKeys) != 0;
                    if (sent) send(n + 1, w >> 8 & 0xFF, w >> 16);
                }
                if (turn > 0) mbar_wait(smem_addr(&sh.empty[place]), (turn - 1) & 1, &sh.stop);
                const uint32_t to = smem + place * kGroupBytes;
                const int from = max(lo, static_cast<int>(side) * 8), till = min(hi, static_cast<int>(side) * 8 + 8);
                if (!(static_cast<int>(r >> 2) >= lo && static_cast<int>(r >> 2) < hi)) {
                    // A loop, with the codes moving down to the registers that its next round reads: see
                    // attend_kernel on instructions.
                    constexpr int kRound = 2;
#pragma unroll 1
                    for (int i0 = 0; i0 < 8; i0 += kRound) {
#pragma unroll
                        for (int i = 0; i < 2 * kRound; ++i) {
                            const uint4 &w = code[i >> 1];
                            const uint32_t unit = 2 * i0 + i;
                            store16(to + (unit >> 3) * kChunkBytes + r * 128 + (((unit & 7) ^ (r & 7)) << 4),
                                    decode_unit<T, Code>(i & 1 ? make_uint2(w.z, w.w) : make_uint2(w.x, w.y), scale));
                        }
#pragma unroll
                        for (int i = 0; i + kRound < 8; ++i) code[i] = code[i + kRound];
                    }
                }
                if (from < till) bring_drafts<T>(a, plan, sh, u, n, tile, to, 2 * group, 2, from, till);
                fence_async_shared();
                mbar_arrive(smem_addr(full));
            } else {
                if (first) load_queries<NQ>(a, plan, sh, smem + L::q, u, true, done, warp, lane);
                if (turn > 0) mbar_wait(smem_addr(&sh.empty[place]), (turn - 1) & 1, &sh.stop);
                const uint32_t to = smem + place * kGroupBytes + side * kChunkBytes;
                copy_rows<kTile / 4>(a, sh, n, 0, lo, hi, to, warp * 128);
                if (lo < hi) bring_drafts<T>(a, plan, sh, u, n, tile, to, warp, 1, lo, hi);
                rows_arrive(full, lo < hi);
                bring_rope();
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) ring.next();
            ++done;
        } else if (word == kOver) {
            break;
        }
        tile_done(sh, n, lane);
        if (++tile == plan.tiles) {
            tile = 0;
            q_loaded = false;
            u = unit_at<NQ>(plan, ++unit);
        }
    }
    copy_close();
    copy_wait<0>();
}

// ---- the products ------------------------------------------------------------------------------

// A product warp's walk over the tiles: body(starts, at) for each one with a key, `starts` telling whether
// it is the first of its unit.
template <typename Body>
__device__ __forceinline__ void each_tile(const Plan &plan, Shared &sh, uint32_t begin, uint32_t end, const Body &body)
{
    using namespace tc;
    uint32_t tile = begin % plan.tiles;
    bool starts = true;
    const int lane = threadIdx.x & 31;
    for (uint32_t at = begin, n = 0; at < end; ++at, ++n) {
        const uint32_t word = tile_word(sh, n);
        const bool any = (word & kKeys) != 0;
        tile_done(sh, n, lane);
        if (any) body(starts, at);
        else if (word == kOver) break;
        starts = !any && starts;
        if (++tile == plan.tiles) {
            tile = 0;
            starts = true;
        }
    }
}

template <typename T>
constexpr uint32_t kType = std::is_same<T, Bf16>::value ? 1u : 0u;

// The first product of each tile, as soon as its rows are there and the scores of the tile before
// last have been read. (A warp of its own: one that issued both products would do the second only
// after the next tile's rows, since a look at a barrier that is not there yet takes until it is.)
template <typename T, bool kStored, int NQ>
__device__ __forceinline__ void score_warp(const Plan &plan, Shared &sh, uint32_t smem, uint32_t begin, uint32_t end)
{
    using namespace tc;
    using L = Layout<NQ, kStored>;
    constexpr uint32_t inst = instruction(kType<T>, false, kTile, NQ);
    const uint32_t elected = elect(), tmem = __shfl_sync(0xFFFFFFFFu, sh.tmem, 0);
    // operands at their start; a descriptor counts addresses in units of 16 bytes
    const uint64_t keys0 = operand(smem, 16, 1024), queries = operand(smem + L::q, 16, 1024);
    const uint64_t rotary0 = operand(smem + L::rope, 16, 1024);
    Ring<L::places> in;
    uint32_t n = 0, units = 0;
    each_tile(plan, sh, begin, end, [&](bool starts, uint32_t at) {
        const uint32_t buf = n & 1, s_at = tmem + buf * NQ;
        if (starts) {
            // (the first unit's queries are loaded even if it has no key)
            if (n == 0 && at / plan.tiles != begin / plan.tiles) mbar_wait(smem_addr(&sh.q_full), units++ & 1, &sh.stop);
            mbar_wait(smem_addr(&sh.q_full), units++ & 1, &sh.stop);
        }
        if (n > 1) mbar_wait(smem_addr(&sh.p_full[buf]), ((n >> 1) - 1) & 1, &sh.stop);
#pragma unroll 1
        for (int g = 0; g < 4; ++g) {
            mbar_wait(smem_addr(&sh.full[in.place]), in.turn & 1, &sh.stop);
            fence_async_shared();  // what the copies wrote
            fence_after_sync();
            const uint64_t keys = keys0 + in.place * (kGroupBytes >> 4);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                mma(elected, s_at, keys + ((i / 4 * kChunkBytes + (i & 3) * 32) >> 4),
                    queries + (((2 * g + i / 4) * (NQ * 128) + (i & 3) * 32) >> 4), inst, g > 0 || i > 0);
            in.next();
        }
        mbar_wait(smem_addr(&sh.rope_full[buf]), (n >> 1) & 1, &sh.stop);
        fence_async_shared();
        fence_after_sync();
        const uint64_t rotary = rotary0 + buf * (kChunkBytes >> 4);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            mma(elected, s_at, rotary + ((i * 32) >> 4), queries + ((8 * (NQ * 128) + i * 32) >> 4), inst, true);
        commit(elected, smem_addr(&sh.s_full[buf]));
        ++n;
    });
    if (n > 0) drain(elected, smem_addr(&sh.drained[0]));
}

// The second product of each tile, as soon as its probabilities are there.
template <typename T, bool kStored, int NQ>
__device__ __forceinline__ void weigh_warp(const Plan &plan, Shared &sh, uint32_t smem, uint32_t begin, uint32_t end)
{
    using namespace tc;
    using L = Layout<NQ, kStored>;
    constexpr uint32_t inst = instruction(kType<T>, true, 128, NQ);
    const uint32_t elected = elect(), o_at = __shfl_sync(0xFFFFFFFFu, sh.tmem, 0) + 2 * NQ;
    const uint64_t values0 = operand(smem, kChunkBytes, 1024), probs0 = operand(smem + L::rope, 16, 1024);
    Ring<L::places> out;
    uint32_t n = 0;
    each_tile(plan, sh, begin, end, [&](bool starts, uint32_t) {
        const uint32_t buf = n & 1;
        mbar_wait(smem_addr(&sh.p_full[buf]), (n >> 1) & 1, &sh.stop);
        fence_async_shared();
        fence_after_sync();
        const uint64_t probs = probs0 + buf * (kChunkBytes >> 4);
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {
            const uint64_t values = values0 + out.place * (kGroupBytes >> 4);
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i)
                mma(elected, o_at + b * NQ, values + ((i * 2048) >> 4), probs + ((i * 2048) >> 4), inst, !starts || i > 0);
            commit(elected, smem_addr(&sh.empty[out.place]));
            out.next();
        }
        commit(elected, smem_addr(&sh.rope_empty[buf]));
        commit(elected, smem_addr(&sh.done[buf]));
        ++n;
    });
    if (n > 0) drain(elected, smem_addr(&sh.drained[1]));
}

// ---- the softmax and the outputs ---------------------------------------------------------------

template <typename T, bool kStored, int NQ>
__device__ __forceinline__ void softmax_warps(const KvopsAttend &a, const Plan &plan, Shared &sh, uint32_t smem,
                                              uint32_t begin, uint32_t end)
{
    using namespace tc;
    constexpr int NH = NQ / 2, kBlocks = NH / 8;  // a half's queries
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int quarter = warp & 3, half = warp >> 2;
    // The scores of 64 keys lie in lanes 0-15 of each quarter of tensor memory. A thread takes two keys,
    // key and key + 8, and of each eight columns of its half two: 8 b + pair, 8 b + pair + 1.
    const int key = quarter * 16 + (lane >> 2), pair = 2 * (lane & 3), dim = quarter * 32 + lane;
    // The column whose reference the thread keeps (the four warps of a half, and more than one thread
    // where a half has fewer than 32 columns, keep the same).
    const int slot_of = (lane >> 2) & (2 * kBlocks - 1), column = 8 * (slot_of >> 1) + pair + (slot_of & 1);
    const uint32_t lanes = static_cast<uint32_t>(quarter) << 21;
    const uint32_t s_at = sh.tmem + lanes + half * NH, o_at = s_at + 2 * NQ;
    const float factor = a.scale * 1.4426950408889634f;  // scores as powers of two
    float *mine = sh.per_warp[warp];
    const auto spread = [&](float x) {  // x of the thread's column, to be read by every lane
        __syncwarp();
        mine[column] = x;
        __syncwarp();
    };
    const auto spread2 = [&](int b) {  // of columns 8 b + pair and the next
        float2 f;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(f.x), "=f"(f.y) : "r"(smem_addr(mine + 8 * b + pair)) : "memory");
        return f;
    };
    const auto spread4 = [&](int i) {  // of columns i .. i + 3
        float4 f;
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(smem_addr(mine + i)) : "memory");
        return f;
    };
    const auto ended = [&](uint32_t n) {  // waits until the second product of the n-th tile (with a key) has ended
        mbar_wait(smem_addr(&sh.done[n & 1]), (n >> 1) & 1, &sh.stop);
    };
    uint32_t done = 0, unit = begin / plan.tiles, tile = begin - unit * plan.tiles, start_tile = tile;
    bool fresh = true, started = false, open = false;
    uint32_t word = 0;
    Unit u{};
    float ref = -INFINITY;   // of `column`
    float sum[2 * kBlocks];  // of this thread's keys, by its columns
    for (uint32_t at = begin, meta = 0; at < end; ++at, ++meta) {
        if (fresh) {
            fresh = started = false;
            start_tile = tile;
            u = unit_at<NQ>(plan, unit);
            ref = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2 * kBlocks; ++i) sum[i] = 0.f;
            if (a.drafts > 0) {
                group_barrier(3, kSoftmaxWarps * 32);
                if (threadIdx.x < NQ && threadIdx.x < u.rows) {
                    const uint32_t t = token_of(a, plan, u, u.row0 + threadIdx.x);
                    sh.tree[threadIdx.x] = a.tree != 0 ? reinterpret_cast<const uint64_t *>(a.tree)[u.req * a.tokens + t]
                                                       : (2ull << t) - 1;
                }
                group_barrier(3, kSoftmaxWarps * 32);
            }
        }
        // (to its end also after a wait has given up, since the warps meet at barriers; the warps of a half must agree)
        if (word != kOver) word = tile_word(sh, meta);
        const bool any = group_any(1 + half, 128, (word & kKeys) != 0);
        if (any) {
            mbar_wait(smem_addr(&sh.s_full[done & 1]), (done >> 1) & 1, &sh.stop);
            fence_after_sync();
        }
        const uint8_t kind[2] = {*const_cast<volatile uint8_t *>(&sh.kind[meta % kAhead][key]),
                                 *const_cast<volatile uint8_t *>(&sh.kind[meta % kAhead][key + 8])};
        if (any) {
            // The scores in powers of two, then less their references, then probabilities.
            float y[4 * kBlocks];
            const auto scores = [&]() {
                tmem_load_spread<kBlocks>(s_at + (done & 1) * NQ, y);
#pragma unroll
                for (int i = 0; i < 4 * kBlocks; ++i) y[i] = kind[i >> 1 & 1] == kNone ? -INFINITY : y[i] * factor;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    if (kind[r] < kDraft) continue;
                    const uint32_t j = tile * kTile + key + 8 * r - plan.list_end;
#pragma unroll
                    for (int i = 0; i < 2 * kBlocks; ++i) {
                        float &x = y[4 * (i >> 1) + 2 * r + (i & 1)];
                        if (!(sh.tree[half * NH + 8 * (i >> 1) + pair + (i & 1)] >> j & 1)) x = -INFINITY;
                        else if (kind[r] == kBadDraft) x = NAN;
                    }
                }
            };
            const auto lower = [&]() {  // by the references, which the warp keeps spread; their largest excess
                float excess = -INFINITY;
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    const float2 r = spread2(b);
                    y[4 * b] -= r.x, y[4 * b + 1] -= r.y, y[4 * b + 2] -= r.x, y[4 * b + 3] -= r.y;
                    excess = fmaxf(excess, fmaxf(fmaxf(y[4 * b], y[4 * b + 1]), fmaxf(y[4 * b + 2], y[4 * b + 3])));
                }
                return excess;
            };
            // The probabilities, to where the second product reads them: rounded to the rows' type, since the
            // matrix unit takes both its operands in one type, and the rows in 32 bits would take twice the
            // shared memory that bounds the products. The sums stay fp32, as lse is. (Errors against 64 bits:
            // fp16 2.4e-4 to 2.6e-4 where probabilities in fp32 leave 2.1e-4, the output's own rounding; bf16
            // 1.9e-3 to 2.1e-3 and 1.7e-3.)
            const auto write = [&]() {
                const uint32_t to = smem + Layout<NQ, kStored>::rope + (done & 1) * kChunkBytes + key * 128 + pair * 2;
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                    for (int i = 4 * b; i < 4 * b + 4; ++i) y[i] = exp2_fast(y[i]);
                    const uint32_t at = to + (((half * kBlocks + b) ^ (key & 7)) << 4);
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(T::pack(y[4 * b], y[4 * b + 1])) : "memory");
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + 1024), "r"(T::pack(y[4 * b + 2], y[4 * b + 3])) : "memory");
                }
            };
            scores();
            bool move_all = !started;
            if (started) {
                // The references only have to move when a score passes one by kMost, which each thread's largest excess tells. The probabilities are worked out as if none had, so that
                // the warps need not wait for one another before, and again in the rare tile where one has.
                const float excess = lower();
                write();
                move_all = group_any(1 + half, 128, excess > kMost || (open && excess > -INFINITY));
                if (move_all) scores();
            }
            if (move_all) {
                float m[2 * kBlocks];
#pragma unroll
                for (int i = 0; i < 2 * kBlocks; ++i) m[i] = fmaxf(y[4 * (i >> 1) + (i & 1)], y[4 * (i >> 1) + 2 + (i & 1)]);
                float top = join_columns<true>(m, slot_of);
                sh.top[half][quarter][column] = top;
                group_barrier(1 + half, 128);
                // the same decision in the four warps of this half
                top = fmaxf(fmaxf(sh.top[half][0][column], sh.top[half][1][column]),
                            fmaxf(sh.top[half][2][column], sh.top[half][3][column]));
                const bool move = top > ref + kMost || (ref == -INFINITY && top > -INFINITY);
                const float was = ref;
                if (move) ref = top - plan.lift;
                if (started && __any_sync(0xFFFFFFFFu, move)) {
                    spread(move ? exp2_fast(was - ref) : 1.f);
                    ended(done - 1);
                    fence_after_sync();
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) {
                        const float2 f = spread2(b);
                        sum[2 * b] *= f.x, sum[2 * b + 1] *= f.y;
                    }
#pragma unroll 1
                    for (int b = 0; b < 4 * NH / 8; ++b) {
                        const int i = b % (NH / 8) * 8;
                        const uint32_t o = o_at + b / (NH / 8) * NQ + i;
                        float v[8];
                        tmem_load<8>(o, v);
                        const float4 f = spread4(i), g = spread4(i + 4);
                        v[0] *= f.x, v[1] *= f.y, v[2] *= f.z, v[3] *= f.w;
                        v[4] *= g.x, v[5] *= g.y, v[6] *= g.z, v[7] *= g.w;
                        tmem_store<8>(o, v);
                    }
                }
                spread(ref == -INFINITY ? 0.f : ref);
                // a column without any key so far: its first finite score moves its reference
                open = __any_sync(0xFFFFFFFFu, ref == -INFINITY);
                lower();
                write();
            }
            fence_async_shared();
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&sh.p_full[done & 1]));
            // Off the way to the second product: the sums, and the wait for the end of the tile before. Every
            // tile's is waited for in its turn, since a parity only tells a phase from its neighbours, and
            // before the next tile of the same parity can end, which needs this warp's next arrival.
#pragma unroll
            for (int i = 0; i < 2 * kBlocks; ++i) sum[i] += y[4 * (i >> 1) + (i & 1)] + y[4 * (i >> 1) + 2 + (i & 1)];
            if (done > 0) ended(done - 1);
            started = true;
            ++done;
        }
        tile_done(sh, meta, lane);
        const bool ends = tile + 1 == plan.tiles;
        if (ends || at + 1 == end) {
            const bool complete = ends && start_tile == 0;
            const uint32_t slot = 2 * blockIdx.x + (at - tile + start_tile > begin ? 1 : 0);
            const float part = join_columns<false>(sum, slot_of);
            group_barrier(1 + half, 128);
            sh.top[half][quarter][column] = part;
            group_barrier(1 + half, 128);
            // From here on lane l has column l. Every warp adds the quarters in the same order.
            const int c = lane & (NH - 1);
            const float total = (sh.top[half][0][c] + sh.top[half][1][c]) + (sh.top[half][2][c] + sh.top[half][3][c]);
            const float at_ref = started ? mine[c] : 0.f;
            __syncwarp();
            const uint32_t col = half * NH + lane;
            if (lane < NH && quarter == 0 && col < u.rows) {
                if (!complete)
                    plan.part_ml[static_cast<uint64_t>(slot) * NQ + col] = make_float2(total == 0.f ? -INFINITY : at_ref, total);
                else if (a.lse != 0)
                    reinterpret_cast<float *>(a.lse)[u.out_row + col] =
                        total == 0.f ? -INFINITY : (at_ref + log2f(total)) * 0.6931471805599453f;
            }
            if (lane < NH) mine[lane] = total == 0.f ? 0.f : 1.f / total;
            __syncwarp();
            if (started) {
                ended(done - 1);
                fence_after_sync();
            }
            // 16 queries of 128 dimensions at a time (8, where a half has no more).
            constexpr int kRows = NH < 16 ? NH : 16;
#pragma unroll 1
            for (int b = 0; b < 4 * NH / kRows; ++b) {
                const uint32_t block = b / (NH / kRows), first = b % (NH / kRows) * kRows;  // of the half's queries
                float v[kRows];
#pragma unroll
                for (int i = 0; i < kRows; ++i) v[i] = 0.f;
                if (started) tmem_load<kRows>(o_at + block * NQ + first, v);
                if (!complete) {
                    float4 *to = reinterpret_cast<float4 *>(plan.part_o);
#pragma unroll
                    for (int i = 0; i < kRows; i += 4)
                        to[part_at<NQ>(slot, block, quarter, half, (first + i) / 4, lane)] =
                            make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    continue;
                }
                const uint32_t r0 = half * NH + first;
                if (!started) {  // no keys at all
                    for (int i = 0; i < kRows; ++i)
                        if (r0 + i < u.rows)
                            reinterpret_cast<uint16_t *>(a.out)[(u.out_row + r0 + i) * kValueDim + block * 128 + dim] = 0;
                    continue;
                }
                // A thread has one dimension of kRows queries. Four lanes exchange theirs, so that each has
                // four dimensions of a quarter of the queries and eight lanes write 64 bytes of a row.
                uint32_t two[kRows / 2];  // of an even lane rows 0, 2, .. with the next dimension, of an odd one rows 1, 3, ..
                const bool odd = lane & 1, upper = lane & 2;
#pragma unroll
                for (int i = 0; i < kRows; i += 4) {
                    const float4 f = spread4(first + i);
                    v[i] *= f.x, v[i + 1] *= f.y, v[i + 2] *= f.z, v[i + 3] *= f.w;
#pragma unroll
                    for (int c = i; c < i + 4; c += 2) {
                        const float other = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[c] : v[c + 1], 1);
                        two[c / 2] = odd ? T::pack(other, v[c + 1]) : T::pack(v[c], other);
                    }
                    const uint32_t keep = upper ? two[i / 2 + 1] : two[i / 2], give = upper ? two[i / 2] : two[i / 2 + 1];
                    const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, give, 2);
                    const uint32_t r = r0 + i + (upper ? 2 : 0) + odd;
                    if (r < u.rows)
                        reinterpret_cast<uint2 *>(a.out)[(u.out_row + r) * (kValueDim / 4) + block * 32 + (dim >> 2)] =
                            upper ? make_uint2(got, keep) : make_uint2(keep, got);
                }
            }
            fence_before_sync();  // ahead of the next unit's first product, which its probabilities release
            __syncwarp();
            fresh = true;
        }
        if (++tile == plan.tiles) {
            tile = 0;
            ++unit;
        }
    }
}

// The roles' code is long and each warp goes through its own once a tile, which is slow where it does not stay in
// the instruction caches: unrolled, the products' 36 + 16 instructions with their descriptors and the
// conversion of a row's 128 codes had warps waiting for instructions more than a quarter of the time
// (then, 64 requests x 128 heads took 80 us unrolled and 72 in loops; x 16 heads 42 and 37; 8-bit rows 58 and 48).
// So these are loops of short bodies, and the waits' slow halves are a function.
template <typename T, typename Code, bool kStored, int NQ>
__global__ void __launch_bounds__(kThreads, 1)
    attend_kernel(const KvopsAttend a, const Plan plan)
{
    using namespace tc;
    extern __shared__ uint8_t dynamic[];
    __shared__ Shared sh;
    const uint32_t smem = (smem_addr(dynamic) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5;
    // join_kernel, or the kernel behind, may take its seats and wait. (This grid has all of its own by then, and
    // two of its CTAs never share an SM, whose shared memory and tensor memory one fills.)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        sh.stop = 0;
        mbar_init(smem_addr(&sh.q_full), kLoadWarps * 32);
        for (int g = 0; g < kMostPlaces; ++g) {
            mbar_init(smem_addr(&sh.full[g]), 2 * 32);
            mbar_init(smem_addr(&sh.empty[g]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_addr(&sh.rope_full[b]), kLoadWarps * 32);
            mbar_init(smem_addr(&sh.rope_empty[b]), 1);
            mbar_init(smem_addr(&sh.s_full[b]), 1);
            mbar_init(smem_addr(&sh.done[b]), 1);
            mbar_init(smem_addr(&sh.p_full[b]), kSoftmaxWarps);
            mbar_init(smem_addr(&sh.drained[b]), 1);
        }
        for (uint32_t b = 0; b < kAhead; ++b) {
            mbar_init(smem_addr(&sh.meta_full[b]), 1);
            mbar_init(smem_addr(&sh.meta_empty[b]), kSoftmaxWarps + kLoadWarps + 2);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kScoreWarp) tmem_alloc<512>(&sh.tmem);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    // Launched as a programmatic dependent: what is above may run before the kernel ahead has ended.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t units = real_units(a, plan);
    const uint32_t run = run_length(plan, units), pairs = units * plan.tiles;
    const uint32_t begin = min(blockIdx.x * run, pairs), end = min(begin + run, pairs);
    // A wait that gives up sets sh.stop and every role goes on to its end without waiting for a tile
    // again, so that no thread is left at a barrier. What is under way by then still ends before the memory
    // that it uses is given back: the load warps wait for their copies, the product warps for their products.
    if (warp < kSoftmaxWarps) {
        softmax_warps<T, kStored, NQ>(a, plan, sh, smem, begin, end);
    } else if (warp < kSoftmaxWarps + kLoadWarps) {
        load_warps<T, Code, kStored, NQ>(a, plan, sh, smem, begin, end);
    } else if (warp == kScoreWarp) {
        score_warp<T, kStored, NQ>(plan, sh, smem, begin, end);
    } else if (warp == kWeighWarp) {
        weigh_warp<T, kStored, NQ>(plan, sh, smem, begin, end);
    } else {
        find_warp<NQ, kStored>(a, plan, sh, begin, end);
    }
    __syncwarp();
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (warp == kScoreWarp) tmem_free<512>(sh.tmem);
    if (threadIdx.x == 0 && sh.stop != 0 && a.err_word != 0)
        atomicCAS_system(reinterpret_cast<uint32_t *>(a.err_word), 0u, KVOPS_ERR_ATTEND_TIMEOUT);
}

static_assert(sizeof(Shared) <= 6 * 1024, "as Layout counts it");
static_assert(offsetof(Shared, per_warp) % 16 == 0 && alignof(Shared) % 16 == 0, "read as float4");

// Joins the parts of the units that the ends of runs cut. Block x is the cut behind CTA x's run, and does
// its unit if it is the first cut in it; block y takes four query rows, and block z kBlocks of the
// four blocks of 128 dimensions, a thread one of each. The parts are added in their order. Every warp works
// the weights out for itself and the first parts are fetched meanwhile, so that a block is one chain of
// two loads and the blocks, which have little to do, are few.
constexpr int kJoinThreads = 128;
template <typename T, int NQ, int kBlocks>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const KvopsAttend a, const Plan plan)
{
    constexpr uint32_t kFirst = 16 / kBlocks;  // parts fetched ahead
    __shared__ float4 weight[kJoinThreads / 32][32];  // of a part, by row
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t units = real_units(a, plan), run = run_length(plan, units), cut = (blockIdx.x + 1) * run;
    if (cut >= units * plan.tiles || cut % plan.tiles == 0) return;
    const uint32_t unit = cut / plan.tiles, begin = unit * plan.tiles, end = begin + plan.tiles;
    const uint32_t first = begin / run, parts = (end - 1) / run - first + 1;
    if (first != blockIdx.x) return;
    const Unit u = unit_at<NQ>(plan, unit);
    const uint32_t row = blockIdx.y * 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (row >= u.rows) return;
    const uint32_t half = row / (NQ / 2), i = row % (NQ / 2) / 4, block0 = blockIdx.z * kBlocks;
    // the part of CTA c: slot 2 c, or 2 c + 1 where its run started in an earlier unit (the first's may have)
    const auto slot_of = [&](uint32_t n) { return 2 * (first + n) + (n == 0 && first * run < begin ? 1 : 0); };
    const float4 *o = reinterpret_cast<const float4 *>(plan.part_o);
    float4 ahead[kFirst][kBlocks];
#pragma unroll
    for (uint32_t n = 0; n < kFirst; ++n)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
            if (n < parts) ahead[n][b] = o[part_at<NQ>(slot_of(n), block0 + b, warp, half, i, lane)];
    struct Stats {
        float top[4], sum[4];  // reference and sum of a part, by row
    };
    const auto stats = [&](uint32_t n) {  // of part n; of none, and in rows behind the last, nothing
        Stats x;
        const float2 *ml = plan.part_ml + static_cast<uint64_t>(slot_of(n)) * NQ + row;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool some = n < parts && row + k < u.rows;
            const float2 v = some ? ml[k] : make_float2(-INFINITY, 0.f);
            x.top[k] = v.x, x.sum[k] = v.y;
        }
        return x;
    };
    Stats x = stats(lane);
    float top[4], total[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) top[k] = x.top[k];
    for (uint32_t n = 32 + lane; n < parts; n += 32) {
        const Stats y = stats(n);
#pragma unroll
        for (int k = 0; k < 4; ++k) top[k] = fmaxf(top[k], y.top[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int w = 16; w > 0; w /= 2) top[k] = fmaxf(top[k], __shfl_xor_sync(0xFFFFFFFFu, top[k], w));
    float4 acc[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) acc[b] = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto add = [&](int b, const float4 &v, const float4 &w) {
        acc[b].x += v.x * w.x, acc[b].y += v.y * w.y, acc[b].z += v.z * w.z, acc[b].w += v.w * w.w;
    };
    for (uint32_t n0 = 0; n0 < parts; n0 += 32) {
        if (n0 > 0) x = stats(n0 + lane);
        float w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // (a part without any key has reference -inf and sum 0, or NaN)
            w[k] = x.top[k] != -INFINITY || x.sum[k] != 0.f ? exp2_fast(x.top[k] - top[k]) : 0.f;
            total[k] += x.sum[k] * w[k];
        }
        __syncwarp();
        weight[warp][lane] = make_float4(w[0], w[1], w[2], w[3]);
        __syncwarp();
        const uint32_t some = min(parts - n0, 32u);
        if (n0 == 0) {
#pragma unroll
            for (uint32_t n = 0; n < kFirst; ++n)
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
                    if (n < parts) add(b, ahead[n][b], weight[warp][n]);
        }
#pragma unroll 8
        for (uint32_t n = n0 == 0 ? kFirst : 0; n < some; ++n)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
                add(b, o[part_at<NQ>(slot_of(n0 + n), block0 + b, warp, half, i, lane)], weight[warp][n]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int w = 16; w > 0; w /= 2) total[k] += __shfl_xor_sync(0xFFFFFFFFu, total[k], w);
    float f[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = total[k] == 0.f ? 0.f : 1.f / total[k];
    const bool odd = lane & 1;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        const float v[4] = {total[0] == 0.f ? 0.f : acc[b].x * f[0], total[1] == 0.f ? 0.f : acc[b].y * f[1],
                            total[2] == 0.f ? 0.f : acc[b].z * f[2], total[3] == 0.f ? 0.f : acc[b].w * f[3]};
#pragma unroll
        for (int c = 0; c < 4; c += 2) {  // an even lane takes row c of its dimension and the next, an odd one c + 1
            const float other = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[c] : v[c + 1], 1);
            const uint32_t two = odd ? T::pack(other, v[c + 1]) : T::pack(v[c], other), k = row + c + odd;
            if (k < u.rows)
                reinterpret_cast<uint32_t *>(a.out)[((u.out_row + k) * kValueDim + (block0 + b) * 128 + warp * 32 + (lane & ~1u)) / 2] = two;
        }
    }
    if (threadIdx.x == 0 && block0 == 0 && a.lse != 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (row + k < u.rows)
                reinterpret_cast<float *>(a.lse)[u.out_row + row + k] =
                    total[k] == 0.f ? -INFINITY : (top[k] + log2f(total[k])) * 0.6931471805599453f;
    }
}

// ---- the host ----------------------------------------------------------------------------------

int invalid(const char *msg) { return set_last_error(KVOPS_E_INVALID, msg); }

// The argument checks that both entry points share.
int check_shape(const KvopsAttend *a)
{
    if (!is_inited()) return set_last_error(KVOPS_E_NOT_INITED, "kvops not inited");
    if (a == nullptr) return invalid("attend_hot: the arguments are NULL");
    if (a->tokens == 0 || a->tokens > 64) return invalid("attend_hot: tokens must be in [1, 64]");
    if (a->heads == 0 || a->heads > 128) return invalid("attend_hot: heads must be in [1, 128]");
    if (a->drafts > 64) return invalid("attend_hot: drafts must be <= 64");
    if (a->top_k > (1u << 24) || a->max_num_reqs > (1u << 16))
        return invalid("attend_hot: top_k / max_num_reqs out of range");
    if (a->row_format > KVOPS_ROW_INT8) return invalid("attend_hot: row_format must be 0, 1 or 2");
    if (a->row_dtype > KVOPS_DTYPE_BF16) return invalid("attend_hot: row_dtype must be 0 or 1");
    if (a->report_slots > 1) return invalid("attend_hot: report_slots must be 0 or 1");
    return KVOPS_OK;
}

int sm_count()
{
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return n;
}

// Queries per tile. A pair costs about the same for any number up to 64 (the rows' way into shared
// memory), so a tile takes as many as there are, unless there is little to do: then smaller tiles, whose
// queries and outputs are fewer, are sooner done, up to four pairs an SM. Queries a tile, in us, for 128
// heads x 2048 keys: one request 16: 13.2, 32: 17.5, 64: 18.6; two requests 16.3, 16.7, 24.1; four requests 22.5, 20.1,
// 23.3; one request's four tokens 24.1, 22.2, 27.6; eight requests 30.5, 28.0, 28.0.
uint32_t queries_per_tile(const KvopsAttend &a, uint32_t lists, int sms)
{
    const uint32_t rows = a.heads * (lists > 1 ? 1 : a.tokens);
    uint32_t nq = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    const uint64_t lists_all = static_cast<uint64_t>(a.max_num_reqs) * lists;
    const uint64_t tiles = (a.top_k + a.drafts + kTile - 1) / kTile;
    while (nq > 16 && lists_all * ((rows + nq / 2 - 1) / (nq / 2)) * tiles <= 4 * static_cast<uint64_t>(sms)) nq /= 2;
    return nq;
}

Plan make_plan(const KvopsAttend &a, uint32_t lists, uint32_t nq, int sms)
{
    Plan p{};
    p.lists = lists;
    p.group_rows = a.heads * (lists > 1 ? 1 : a.tokens);
    p.qtiles = (p.group_rows + nq - 1) / nq;
    p.list_end = (a.top_k + 3) & ~3u;
    p.tiles = (p.list_end + a.drafts + kTile - 1) / kTile;
    if (p.tiles == 0) p.tiles = 1;  // no keys at all: outputs of zero
    const uint64_t units = static_cast<uint64_t>(a.max_num_reqs) * lists * p.qtiles, pairs = units * p.tiles;
    // Whole units need no joining, equal runs of pairs leave no SM idle. In tiles' times: a unit costs its
    // tiles and about two more for its queries and outputs, a cut unit these for each part; the joining
    // costs six; and runs that cut a list's query tiles in different places read its rows at different
    // times, which costs an eighth. Whole units against runs, in us: 64 requests x 128 heads x 2048 keys 65, 79
    // (8-bit 90, 97); 100 requests x 128 heads x 1024 keys 72, 75; 130 requests x 16 heads 57, 64 (8-bit 84,
    // 84); but 40 requests x 128 heads 66, 56; 80 requests 130, 97; 100 requests x 16 heads 54, 51 (8-bit 84,
    // 65); 64 requests x 16 heads 52, 37 (8-bit 83, 45). For few short lists the joining is counted too dear:
    // 7 x 3 lists x 24 heads x 333 keys take whole units here, 13.6, where runs take 12.4 (8-bit 20.0, 14.5).
    const uint64_t whole = (units + sms - 1) / sms;
    const uint64_t run = (pairs + sms - 1) / sms;
    p.run_at_most = static_cast<uint32_t>(run);
    const uint64_t cost_runs = run + (p.qtiles > 1 ? run / 8 : 0) + 2 * (run / p.tiles + 2) + 6;
    if (p.tiles == 1 || whole * (p.tiles + 2) <= cost_runs) {
        p.whole = static_cast<uint32_t>(whole);
        p.ctas = static_cast<uint32_t>((units + whole - 1) / whole);
    } else {
        p.ctas = static_cast<uint32_t>(pairs < static_cast<uint64_t>(sms) ? pairs : sms);
    }
    const uint64_t part = p.whole > 0 || run > p.tiles ? p.tiles : run;  // tiles of a list that one CTA takes at the most
    p.lift = a.row_dtype == KVOPS_DTYPE_BF16 ? kLiftBf16 : part * kTile <= kLongPart ? kLiftFp16 : kLiftFp16Long;
    return p;
}

uint64_t workspace_of(const Plan &p, uint32_t nq)
{
    return p.whole > 0 ? 0 : 2ull * p.ctas * nq * (sizeof(float2) + kValueDim * sizeof(float));
}

template <typename T, typename Code, bool kStored, int NQ>
cudaError_t launch_as(const KvopsAttend &a, const Plan &p, cudaStream_t s)
{
    const auto kernel = attend_kernel<T, Code, kStored, NQ>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<NQ, kStored>::bytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.stream = s;
    cfg.gridDim = dim3(p.ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Layout<NQ, kStored>::bytes;
    e = cudaLaunchKernelEx(&cfg, kernel, a, p);
    if (e != cudaSuccess || p.whole > 0 || p.ctas < 2) return e;
    cfg.dynamicSmemBytes = 0;
    // All the dimensions of a row to a block where a unit has few parts, else four blocks for them.
    const bool few = p.run_at_most * 3 >= p.tiles;
    cfg.gridDim = dim3(p.ctas - 1, (p.group_rows < NQ ? p.group_rows + 3 : NQ) / 4, few ? 1 : 4);
    cfg.blockDim = dim3(kJoinThreads);
    return few ? cudaLaunchKernelEx(&cfg, join_kernel<T, NQ, 4>, a, p) : cudaLaunchKernelEx(&cfg, join_kernel<T, NQ, 1>, a, p);
}

template <typename T, int NQ>
cudaError_t launch_format(const KvopsAttend &a, const Plan &p, cudaStream_t s)
{
    switch (a.row_format) {
        case KVOPS_ROW_RAW: return launch_as<T, Int8, false, NQ>(a, p, s);
        case KVOPS_ROW_E4M3: return launch_as<T, E4m3, true, NQ>(a, p, s);
        default: return launch_as<T, Int8, true, NQ>(a, p, s);
    }
}

template <typename T>
cudaError_t launch_queries(const KvopsAttend &a, const Plan &p, uint32_t nq, cudaStream_t s)
{
    switch (nq) {
        case 16: return launch_format<T, 16>(a, p, s);
        case 32: return launch_format<T, 32>(a, p, s);
        default: return launch_format<T, 64>(a, p, s);
    }
}

}  // namespace
}  // namespace kvb

extern "C" int kvops_attend_workspace(const KvopsAttend *a, uint64_t *out_bytes)
{
    const int rc = kvb::check_shape(a);
    if (rc != KVOPS_OK) return rc;
    if (out_bytes == nullptr) return kvb::invalid("attend_workspace: out_bytes is NULL");
    const int sms = kvb::sm_count();
    if (sms <= 0) return kvb::set_last_error(KVOPS_E_CUDA, "attend_workspace: no current device");
    // enough for one list per request and for one per token
    uint64_t most = 0;
    for (uint32_t lists : {1u, a->tokens}) {
        const uint32_t nq = kvb::queries_per_tile(*a, lists, sms);
        const uint64_t n = a->max_num_reqs == 0 ? 0 : kvb::workspace_of(kvb::make_plan(*a, lists, nq, sms), nq);
        most = n > most ? n : most;
    }
    *out_bytes = most;
    return KVOPS_OK;
}

extern "C" int kvops_attend_hot(const KvopsAttend *a, uint64_t stream)
{
    using kvb::invalid;
    int rc = kvb::check_shape(a);
    if (rc != KVOPS_OK) return rc;
    if (a->max_num_reqs == 0) return KVOPS_OK;
    if (a->q == 0 || a->out == 0 || a->num_real == 0) return invalid("attend_hot: a tensor address is 0");
    if (a->top_k > 0 && (a->hot_row_base == 0 || a->req_pool_indices == 0 || a->topk_device_slots == 0))
        return invalid("attend_hot: a tensor address is 0");
    if (a->drafts > 0 && a->draft_rows == 0) return invalid("attend_hot: a tensor address is 0");
    if ((a->q | a->out | a->workspace | (a->top_k > 0 ? a->hot_row_base : 0) | (a->drafts > 0 ? a->draft_rows : 0)) % 16 != 0)
        return invalid("attend_hot: q, out, hot rows, draft rows and workspace must be 16-byte aligned");
    if ((a->q_stride_req | a->q_stride_token | a->q_stride_head) % 8 != 0 ||
        (a->drafts > 0 && (a->draft_stride_req | a->draft_stride_row) % 8 != 0))
        return invalid("attend_hot: strides of q and draft rows must be multiples of 8 values");
    if (a->lse % 4 != 0 || a->num_real % 4 != 0 || a->topk_device_slots % 4 != 0 || a->req_pool_indices % 8 != 0 ||
        a->tree % 8 != 0 || a->err_word % 4 != 0)
        return invalid("attend_hot: lse, num_real, slots, pool indices, tree and err_word must have their types' alignment");
    const int sms = kvb::sm_count();
    if (sms <= 0) return kvb::set_last_error(KVOPS_E_CUDA, "attend_hot: no current device");
    const uint32_t lists = a->tokens > 1 && a->slots_stride_token != 0 && a->top_k > 0 ? a->tokens : 1;
    const uint32_t nq = kvb::queries_per_tile(*a, lists, sms);
    kvb::Plan p = kvb::make_plan(*a, lists, nq, sms);
    // (the end of a CTA's run is a 32-bit number, rounded up to a whole run for each CTA)
    if (static_cast<uint64_t>(a->max_num_reqs) * lists * p.qtiles * p.tiles >= (1ull << 31))
        return invalid("attend_hot: requests x lists x keys out of range");
    const uint64_t need = kvb::workspace_of(p, nq);
    if (need > 0) {
        if (a->workspace == 0 || a->workspace_bytes < need)
            return invalid("attend_hot: the workspace is smaller than kvops_attend_workspace says");
        p.part_o = reinterpret_cast<float *>(a->workspace);
        p.part_ml = reinterpret_cast<float2 *>(p.part_o + 2ull * p.ctas * nq * kvb::kValueDim);
    }
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = a->row_dtype == KVOPS_DTYPE_FP16 ? kvb::launch_queries<kvb::Fp16>(*a, p, nq, s)
                                                           : kvb::launch_queries<kvb::Bf16>(*a, p, nq, s);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return kvb::set_last_error(KVOPS_E_CUDA, (std::string("launch attend_hot: ") + cudaGetErrorString(e)).c_str());
    }
    return KVOPS_OK;
}
