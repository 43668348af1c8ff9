// attend.cu — kvops_attend_hot: attention of drafted tokens over the hot rows that their top-K
// lists name and over one another's drafted rows along a tree (the formulas are in
// include/kvops_b200.h).
//
// A key row is read once for its score and its value, and every head and drafted token of a
// request shares it, so both products are matrix products over tiles of 128 keys:
//   S^T [128 keys x NQ queries] = K [128 x 576] Q^T,   O^T [512 x NQ] += V^T [512 x 128] P^T,
// with V the first 512 columns of K: one copy of the rows in shared memory serves both, K-major for
// the first and MN-major for the second. The transposed form keeps the matrix unit's 128 rows full
// (keys, then value dimensions) for any number of queries: with the queries as rows a tile of 64
// would run at half rate, and 128 rows of 512 fp32 outputs would fill tensor memory and leave no
// room for the scores. Measured on one SM: M = 64 takes 64 cycles for N = 128, 16 deep; M = 128, N = 64
// takes 48 (the operands' 6 KB at 128 bytes a cycle).
//
// One CTA per SM takes a run of (query tile, key tile) pairs. Warps 0-7: the softmax, a thread per
// key and half of the queries, and the outputs. Warps 8-15: the rows, by asynchronous 16-byte copies
// or, from stored rows, through registers. Warp 16: one thread issues the matrix instructions.
// Shared memory holds one key tile in five groups (four of 128 dimensions, one of the 64 rotary
// ones) that are refilled one by one as the second product passes them.
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
constexpr int kTile = 128;              // keys per tile
constexpr int kChunks = kKeyDim / 64;   // 128-byte columns of a tile
constexpr uint32_t kChunkBytes = kTile * 128;
constexpr int kGroups = 5;              // chunks 0-1, 2-3, 4-5, 6-7, 8
constexpr int kSoftmaxWarps = 8, kLoadWarps = 8;
constexpr int kThreads = (kSoftmaxWarps + kLoadWarps + 1) * 32;

// A running reference is kept this far (in powers of two) below the largest score seen, so that
// the probabilities, up to 2^kLift, lose none of their small neighbours to fp16's subnormals, and it is
// only moved when a score passes it by kLift + kSlack (2^15 still is an fp16 number): moving it means
// scaling the outputs in tensor memory.
constexpr float kLift = 11.f, kSlack = 4.f;

// How the (query tile, key tile) pairs are dealt out. Units are query tiles: group (a request, or a
// request's token where every token has its own list) by group.
struct Plan {
    uint32_t lists;       // lists per request: 1, or tokens
    uint32_t group_rows;  // query rows that share a list
    uint32_t qtiles;      // query tiles per group
    uint32_t tiles;       // key tiles per unit
    uint32_t ctas;
    uint32_t whole;       // > 0: every CTA takes this many whole units; 0: an equal run of pairs
    float2 *part_ml;      // [2 * ctas][NQ] reference and sum of a unit's part
    float *part_o;        // [2 * ctas][NQ][512] its weighted sums
};

__device__ __forceinline__ uint32_t real_units(const KvopsAttend &a, const Plan &p)
{
    const int32_t n = *reinterpret_cast<const int32_t *>(a.num_real);
    const uint32_t reqs = n < 0 ? 0u : min(static_cast<uint32_t>(n), a.max_num_reqs);
    return reqs * p.lists * p.qtiles;
}

// The first pair of CTA c.
__device__ __forceinline__ uint32_t run_start(const Plan &p, uint32_t units, uint32_t c)
{
    if (p.whole > 0) return min(c * p.whole, units) * p.tiles;
    return static_cast<uint32_t>(static_cast<uint64_t>(units) * p.tiles * c / p.ctas);
}

struct Unit {
    uint32_t req;       // batch row
    uint32_t token;     // its token, where every token has its own list
    uint32_t row0;      // first query row within the group
    uint32_t rows;      // query rows (at most NQ)
    uint64_t out_row;   // output row of query row row0
};

template <int NQ>
__device__ __forceinline__ Unit unit_at(const KvopsAttend &a, const Plan &p, uint32_t unit)
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

template <int NQ>
struct Layout {
    static constexpr uint32_t q = kChunks * kChunkBytes;
    // The probabilities [128 keys][64 x 16 bit] take the place of the rotary columns, which only the
    // scores need, where the queries leave no room for them elsewhere.
    static constexpr uint32_t p = NQ == 64 ? 8 * kChunkBytes : q + NQ * 2 * kKeyDim;
    static constexpr uint32_t bytes = (NQ == 64 ? q + NQ * 2 * kKeyDim : p + kChunkBytes) + 1024;
};

struct Shared {
    alignas(8) uint64_t q_full, full[kGroups], empty[kGroups], s_full, p_full, meta_full[2], meta_empty[2];
    uint64_t tree[64];         // of the unit's query rows
    float top[2][4][32];       // a tile's maxima by column, by half and lane quarter
    alignas(16) float per_warp[kSoftmaxWarps][32];  // read four at a time
    uint8_t kind[2][kTile];    // of the tile's keys: kNone, kList, kDraft or kBadDraft
    uint32_t any[2];           // whether the tile has a key
    uint32_t tmem, stop;
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
__device__ __forceinline__ float warp_max(float x)
{
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

// Lane l's sum over the warp of column l % kN.
template <int kN>
__device__ __forceinline__ float column_sum(float (&v)[kN], int lane)
{
#pragma unroll
    for (int w = kN / 2; w > 0; w /= 2) {
#pragma unroll
        for (int i = 0; i < w; ++i) {
            const bool up = (lane & w) != 0;
            const float give = up ? v[i] : v[i + w], keep = up ? v[i + w] : v[i];
            v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, w);
        }
    }
    float s = v[0];
#pragma unroll
    for (int w = kN; w < 32; w *= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, w);
    return s;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool some)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(some ? 16u : 0u) : "memory");
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

// This thread's share of a tile: unit `unit` (16 bytes) of the 128-byte columns of rows first + 32 j.
template <typename T, typename Code, bool kStored, int NQ>
__device__ __forceinline__ void load_warps(const KvopsAttend &a, const Plan &plan, Shared &sh, uint32_t smem,
                                           uint32_t begin, uint32_t end)
{
    using namespace tc;
    const int tid = threadIdx.x - kSoftmaxWarps * 32, lane = tid & 31;
    const uint32_t unit16 = tid & 7, first = tid >> 3;
    const uint64_t row_bytes = kStored ? kStoredBytes : 2 * kKeyDim;
    const uint32_t dst0 = smem + first * 128 + ((unit16 ^ (first & 7)) << 4);  // rows 32 apart swizzle alike
    uint32_t done = 0, meta = 0;  // tiles with a key, tiles
    uint32_t unit = begin / plan.tiles, tile = begin - unit * plan.tiles;
    Unit u = unit_at<NQ>(a, plan, unit);

    int32_t slot[4];
    const uint8_t *hot = nullptr;
    const auto fetch = [&]() {  // the slots of (u, tile), and where the request's hot rows are
        const int32_t *list = reinterpret_cast<const int32_t *>(a.topk_device_slots) + u.req * a.slots_stride_req +
                              u.token * a.slots_stride_token;
        hot = nullptr;
        if (a.top_k > 0) {
            const int64_t pool = reinterpret_cast<const int64_t *>(a.req_pool_indices)[u.req];
            if (pool >= 0 && pool < static_cast<int64_t>(a.pool_size))
                hot = reinterpret_cast<const uint8_t *>(a.hot_row_base) + pool * a.hot_req_stride_rows * row_bytes;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t k = tile * kTile + first + 32 * j;
            slot[j] = k < a.top_k ? list[k] : -1;
        }
    };
    if (begin < end) fetch();
    bool q_loaded = false;
    for (uint32_t at = begin; at < end; ++at) {
        const Unit now = u;
        const uint32_t now_tile = tile;
        const uint8_t *row[4];
        uint8_t kind[4];
        bool mine = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t k = now_tile * kTile + first + 32 * j;
            row[j] = nullptr;
            kind[j] = kNone;
            if (k < a.top_k) {
                if (hot != nullptr && slot[j] >= 0 && static_cast<uint32_t>(slot[j]) < a.hot_rows) {
                    row[j] = hot + static_cast<uint32_t>(slot[j]) * row_bytes;
                    kind[j] = kList;
                }
            } else if (k < a.top_k + a.drafts) {
                row[j] = reinterpret_cast<const uint8_t *>(a.draft_rows) +
                         2 * (now.req * a.draft_stride_req + (k - a.top_k) * a.draft_stride_row);
                kind[j] = kDraft;
            }
            mine |= kind[j] != kNone;
        }
        const uint32_t buf = meta & 1;
        if (meta >= 2) mbar_wait(smem_addr(&sh.meta_empty[buf]), ((meta >> 1) - 1) & 1, &sh.stop);
        if (unit16 == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) sh.kind[buf][first + 32 * j] = kind[j];
        }
        const bool any = group_any(4, kLoadWarps * 32, mine);
        if (tid == 0) {
            sh.any[buf] = any;
            mbar_arrive(smem_addr(&sh.meta_full[buf]));
        }
        ++meta;
        // the next tile's slots travel while this tile's rows do
        const bool last = at + 1 == end || tile + 1 == plan.tiles;
        if (++tile == plan.tiles) {
            tile = 0;
            ++unit;
            if (at + 1 < end) u = unit_at<NQ>(a, plan, unit);
        }
        if (at + 1 < end) fetch();
        if (any) {
            // Codes wait in registers for their place in shared memory: three groups of the four (a
            // fourth would not fit), the last one following the first.
            uint4 code[kStored ? 3 : 1][4];
            float scale[kStored ? 3 : 1][4];
            const auto stage = [&](int g) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    scale[g % 3][j] = 0.f;
                    code[g % 3][j] = make_uint4(0u, 0u, 0u, 0u);
                    if (kind[j] == kList) {
                        scale[g % 3][j] = __ldg(reinterpret_cast<const float *>(row[j] + kValueDim) + g);
                        code[g % 3][j] = __ldcs(reinterpret_cast<const uint4 *>(row[j] + g * 128) + unit16);
                    }
                }
            };
            if constexpr (kStored) {
                stage(0);
                stage(1);
                stage(2);
            }
            const uint32_t freed = (done - 1) & 1;
            if (!q_loaded) {
                // the queries' place is free once the last unit's products are done
                if (done > 0) mbar_wait(smem_addr(&sh.empty[kGroups - 1]), freed, &sh.stop);
                for (uint32_t i = tid; i < NQ * 72; i += kLoadWarps * 32) {
                    const uint32_t r = i / 72, c = i - r * 72;
                    const uint32_t q_row = now.row0 + r;
                    const uint32_t t = token_of(a, plan, now, q_row);
                    const uint32_t h = plan.lists > 1 ? q_row : q_row - t * a.heads;
                    const bool some = r < now.rows;
                    const uint8_t *src = reinterpret_cast<const uint8_t *>(a.q);
                    if (some)
                        src += 2 * (now.req * a.q_stride_req + t * a.q_stride_token + h * a.q_stride_head) + c * 16;
                    copy16(smem + Layout<NQ>::q + (c >> 3) * (NQ * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4), src, some);
                }
            }
            copy_close();
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                if (done > 0) mbar_wait(smem_addr(&sh.empty[g]), freed, &sh.stop);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t dst = dst0 + 2 * g * kChunkBytes + j * 32 * 128;
                    if (kind[j] == kDraft) {
                        // Rows that not every query sees: a value that is not finite would turn
                        // their zero probability into NaN, so it is left out and the row marked.
#pragma unroll
                        for (int c = 0; c < (g < 4 ? 2 : 1); ++c) {
                            uint4 v = *reinterpret_cast<const uint4 *>(row[j] + (2 * g + c) * 128 + unit16 * 16);
                            if (not_finite<T>(v)) {
                                v = make_uint4(0u, 0u, 0u, 0u);
                                sh.kind[buf][first + 32 * j] = kBadDraft;
                            }
                            store16(dst + c * kChunkBytes, v);
                        }
                    } else if (!kStored || g == 4) {
                        const uint8_t *src = kind[j] == kList ? row[j] : reinterpret_cast<const uint8_t *>(a.q);
                        if (kind[j] == kList)
                            src += (kStored ? kStoredPlain : 2 * g * 128) + unit16 * 16;
                        copy16(dst, src, kind[j] == kList);
                        if (g < 4) copy16(dst + kChunkBytes, src + (kind[j] == kList ? 128 : 0), kind[j] == kList);
                    } else if constexpr (kStored) {
                        // 16 codes: units 2 u and 2 u + 1 of the group's 16 (u = unit16)
                        const float s = scale[g % 3][j];
                        const uint4 c = code[g % 3][j];
                        const uint32_t r = first + 32 * j, to = smem + (2 * g + (unit16 >> 2)) * kChunkBytes + r * 128;
                        const uint32_t n = (unit16 & 3) * 2;
                        store16(to + ((n ^ (r & 7)) << 4), decode_unit<T, Code>(make_uint2(c.x, c.y), s));
                        store16(to + (((n + 1) ^ (r & 7)) << 4), decode_unit<T, Code>(make_uint2(c.z, c.w), s));
                    }
                }
                copy_close();
                if constexpr (kStored) {
                    if (g == 0) stage(3);
                }
            }
            const auto hand_over = [&](uint64_t *bar) {
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(bar));
            };
            copy_wait<5>();
            if (!q_loaded) hand_over(&sh.q_full);
            q_loaded = true;
            copy_wait<4>();
            hand_over(&sh.full[0]);
            copy_wait<3>();
            hand_over(&sh.full[1]);
            copy_wait<2>();
            hand_over(&sh.full[2]);
            copy_wait<1>();
            hand_over(&sh.full[3]);
            copy_wait<0>();
            hand_over(&sh.full[4]);
            ++done;
        }
        if (last) q_loaded = false;
    }
}

// ---- the products ------------------------------------------------------------------------------

template <typename T, int NQ>
__device__ __forceinline__ void product_thread(const Plan &plan, Shared &sh, uint32_t smem, uint32_t begin, uint32_t end)
{
    using namespace tc;
    constexpr uint32_t type = std::is_same<T, Bf16>::value ? 1u : 0u;
    constexpr uint32_t score = instruction(type, false, 128, NQ), weigh = instruction(type, true, 128, NQ);
    const uint32_t s_at = sh.tmem, o_at = sh.tmem + NQ;
    uint32_t done = 0, units = 0, tile = begin % plan.tiles;
    bool started = false;  // this unit's part has outputs in tensor memory
    for (uint32_t at = begin, meta = 0; at < end; ++at, ++meta) {
        const uint32_t buf = meta & 1;
        mbar_wait(smem_addr(&sh.meta_full[buf]), (meta >> 1) & 1, &sh.stop);
        const bool any = *const_cast<volatile uint32_t *>(&sh.any[buf]) != 0;
        mbar_arrive(smem_addr(&sh.meta_empty[buf]));
        if (any) {
            if (!started) mbar_wait(smem_addr(&sh.q_full), units++ & 1, &sh.stop);
#pragma unroll 1
            for (int g = 0; g < kGroups; ++g) {
                mbar_wait(smem_addr(&sh.full[g]), done & 1, &sh.stop);
                fence_after_sync();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (g == 4 && i >= 4) break;
                    const int c = 2 * g + i / 4;
                    mma(s_at, operand(smem + c * kChunkBytes + (i & 3) * 32, 16, 1024),
                        operand(smem + Layout<NQ>::q + c * (NQ * 128) + (i & 3) * 32, 16, 1024), score, g > 0 || i > 0);
                }
            }
            commit(smem_addr(&sh.s_full));
            mbar_wait(smem_addr(&sh.p_full), done & 1, &sh.stop);
            fence_after_sync();
#pragma unroll 1
            for (int b = 0; b < 4; ++b) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    mma(o_at + b * NQ, operand(smem + 2 * b * kChunkBytes + i * 2048, kChunkBytes, 1024),
                        operand(smem + Layout<NQ>::p + i * 2048, 16, 1024), weigh, started || i > 0);
                commit(smem_addr(&sh.empty[b]));
            }
            commit(smem_addr(&sh.empty[kGroups - 1]));
            started = true;
            ++done;
        }
        if (++tile == plan.tiles) {
            tile = 0;
            started = false;
        }
    }
}

// ---- the softmax and the outputs ---------------------------------------------------------------

template <typename T, int NQ>
__device__ __forceinline__ void softmax_warps(const KvopsAttend &a, const Plan &plan, Shared &sh, uint32_t smem,
                                              uint32_t begin, uint32_t end)
{
    using namespace tc;
    constexpr int NH = NQ / 2;  // queries of a thread
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int quarter = warp & 3, half = warp >> 2;
    const int key = quarter * 32 + lane;  // this thread's row of the tile
    const uint32_t lanes = static_cast<uint32_t>(quarter) << 21;
    const uint32_t s_at = sh.tmem + lanes + half * NH, o_at = sh.tmem + lanes + NQ + half * NH;
    const float factor = a.scale * 1.4426950408889634f;  // scores as powers of two
    float *mine = sh.per_warp[warp];
    const auto spread = [&](float x) {  // column c's x, held by lane c, to be read by every lane
        __syncwarp();
        mine[lane] = x;
        __syncwarp();
    };
    // of columns i .. i + 3; volatile: read where it is used, not kept in registers
    const auto spread4 = [&](int i) {
        float4 f;
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(smem_addr(mine + i)) : "memory");
        return f;
    };
    uint32_t done = 0, unit = begin / plan.tiles, tile = begin - unit * plan.tiles, start_tile = tile;
    bool fresh = true, started = false;
    Unit u{};
    float ref = -INFINITY;  // of column `lane` of this half
    float sum[NH];          // of this thread's keys, by column
    for (uint32_t at = begin, meta = 0; at < end; ++at, ++meta) {
        if (fresh) {
            fresh = started = false;
            start_tile = tile;
            u = unit_at<NQ>(a, plan, unit);
            ref = -INFINITY;
#pragma unroll
            for (int i = 0; i < NH; ++i) sum[i] = 0.f;
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
        const uint32_t buf = meta & 1;
        mbar_wait(smem_addr(&sh.meta_full[buf]), (meta >> 1) & 1, &sh.stop);
        // (through a barrier: after a wait has given up, too, the warps of a half must agree)
        const bool any = group_any(1 + half, 128, *const_cast<volatile uint32_t *>(&sh.any[buf]) != 0);
        if (any) {
            mbar_wait(smem_addr(&sh.s_full), done & 1, &sh.stop);
            fence_after_sync();
        }
        const uint8_t kind = *const_cast<volatile uint8_t *>(&sh.kind[buf][key]);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&sh.meta_empty[buf]));
        if (any) {
            float x[NH];
            tmem_load<NH>(s_at, x);
#pragma unroll
            for (int i = 0; i < NH; ++i) x[i] = kind == kNone ? -INFINITY : x[i] * factor;
            if (kind >= kDraft) {
                const uint32_t j = tile * kTile + key - a.top_k;
#pragma unroll
                for (int i = 0; i < NH; ++i) {
                    const bool sees = (sh.tree[half * NH + i] >> j) & 1;
                    if (!sees) x[i] = -INFINITY;
                    else if (kind == kBadDraft) x[i] = NAN;
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < NH; ++i) {
                const float m = warp_max(x[i]);
                if (lane == i) top = m;
            }
            sh.top[half][quarter][lane] = top;
            group_barrier(1 + half, 128);
            top = fmaxf(fmaxf(sh.top[half][0][lane], sh.top[half][1][lane]),
                        fmaxf(sh.top[half][2][lane], sh.top[half][3][lane]));
            // the same decision in the four warps of this half
            const bool move = top > ref + (kLift + kSlack) || (ref == -INFINITY && top > -INFINITY);
            if (__any_sync(0xFFFFFFFFu, move)) {
                const float was = ref;
                if (move) ref = top - kLift;
                if (started) {
                    spread(move ? exp2_fast(was - ref) : 1.f);
                    mbar_wait(smem_addr(&sh.empty[kGroups - 1]), (done - 1) & 1, &sh.stop);
                    fence_after_sync();
#pragma unroll
                    for (int i = 0; i < NH; i += 4) {
                        const float4 f = spread4(i);
                        sum[i] *= f.x, sum[i + 1] *= f.y, sum[i + 2] *= f.z, sum[i + 3] *= f.w;
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
            }
            spread(ref == -INFINITY ? 0.f : ref);
            const uint32_t to = smem + Layout<NQ>::p + key * 128;
#pragma unroll
            for (int i = 0; i < NH; i += 8) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    const int c = i + 2 * k;
                    const float4 r = spread4(c);
                    const float p0 = exp2_fast(x[c] - r.x), p1 = exp2_fast(x[c + 1] - r.y);
                    const float p2 = exp2_fast(x[c + 2] - r.z), p3 = exp2_fast(x[c + 3] - r.w);
                    sum[c] += p0, sum[c + 1] += p1, sum[c + 2] += p2, sum[c + 3] += p3;
                    w[k] = T::pack(p0, p1);
                    w[k + 1] = T::pack(p2, p3);
                }
                store16(to + ((((half * NH + i) >> 3) ^ (key & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
            }
            fence_async_shared();
            fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&sh.p_full));
            started = true;
            ++done;
        }
        const bool ends = tile + 1 == plan.tiles;
        if (ends || at + 1 == end) {
            const bool complete = ends && start_tile == 0;
            const uint32_t slot = 2 * blockIdx.x + (at - tile + start_tile > begin ? 1 : 0);
            float total = column_sum<NH>(sum, lane);
            group_barrier(1 + half, 128);
            sh.top[half][quarter][lane] = total;
            group_barrier(1 + half, 128);
            // every warp adds the quarters in the same order
            total = (sh.top[half][0][lane & (NH - 1)] + sh.top[half][1][lane & (NH - 1)]) +
                    (sh.top[half][2][lane & (NH - 1)] + sh.top[half][3][lane & (NH - 1)]);
            group_barrier(1 + half, 128);
            const uint32_t col = half * NH + lane;
            if (lane < NH && quarter == 0 && col < u.rows) {
                if (!complete)
                    plan.part_ml[static_cast<uint64_t>(slot) * NQ + col] = make_float2(ref, total);
                else if (a.lse != 0)
                    reinterpret_cast<float *>(a.lse)[u.out_row + col] =
                        total == 0.f ? -INFINITY : (ref + log2f(total)) * 0.6931471805599453f;
            }
            spread(complete ? (total == 0.f ? 0.f : 1.f / total) : 1.f);
            if (started) {
                mbar_wait(smem_addr(&sh.empty[kGroups - 1]), (done - 1) & 1, &sh.stop);
                fence_after_sync();
            }
#pragma unroll 1
            for (int b = 0; b < 4 * NH / 8; ++b) {
                const int i = b % (NH / 8) * 8;
                const uint32_t dim = b / (NH / 8) * 128 + key, c = half * NH + i;
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (started) tmem_load<8>(o_at + b / (NH / 8) * NQ + i, v);
                const float4 f = spread4(i), g = spread4(i + 4);
                v[0] *= f.x, v[1] *= f.y, v[2] *= f.z, v[3] *= f.w;
                v[4] *= g.x, v[5] *= g.y, v[6] *= g.z, v[7] *= g.w;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (c + k >= u.rows) break;
                    if (complete)
                        reinterpret_cast<uint16_t *>(a.out)[(u.out_row + c + k) * kValueDim + dim] =
                            static_cast<uint16_t>(T::pack(v[k], 0.f));
                    else
                        plan.part_o[(static_cast<uint64_t>(slot) * NQ + c + k) * kValueDim + dim] = v[k];
                }
            }
            fence_before_sync();
            fresh = true;
        }
        if (++tile == plan.tiles) {
            tile = 0;
            ++unit;
        }
    }
}

template <typename T, typename Code, bool kStored, int NQ>
__global__ void __launch_bounds__(kThreads, 1) attend_kernel(const KvopsAttend a, const Plan plan)
{
    using namespace tc;
    extern __shared__ uint8_t dynamic[];
    __shared__ Shared sh;
    const uint32_t smem = (smem_addr(dynamic) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        sh.stop = 0;
        mbar_init(smem_addr(&sh.q_full), kLoadWarps);
        for (int g = 0; g < kGroups; ++g) {
            mbar_init(smem_addr(&sh.full[g]), kLoadWarps);
            mbar_init(smem_addr(&sh.empty[g]), 1);
        }
        mbar_init(smem_addr(&sh.s_full), 1);
        mbar_init(smem_addr(&sh.p_full), kSoftmaxWarps);
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_addr(&sh.meta_full[b]), 1);
            mbar_init(smem_addr(&sh.meta_empty[b]), kSoftmaxWarps + 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kSoftmaxWarps + kLoadWarps) tmem_alloc<512>(&sh.tmem);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t units = real_units(a, plan);
    const uint32_t begin = run_start(plan, units, blockIdx.x), end = run_start(plan, units, blockIdx.x + 1);
    // A wait that gives up sets sh.stop and every role goes on to its end without waiting again, so
    // that no thread is left at a barrier.
    if (warp < kSoftmaxWarps) {
        softmax_warps<T, NQ>(a, plan, sh, smem, begin, end);
    } else if (warp < kSoftmaxWarps + kLoadWarps) {
        load_warps<T, Code, kStored, NQ>(a, plan, sh, smem, begin, end);
    } else if ((threadIdx.x & 31) == 0) {
        product_thread<T, NQ>(plan, sh, smem, begin, end);
    }
    __syncwarp();
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (warp == kSoftmaxWarps + kLoadWarps) tmem_free<512>(sh.tmem);
    if (threadIdx.x == 0 && sh.stop != 0 && a.err_word != 0)
        atomicCAS_system(reinterpret_cast<uint32_t *>(a.err_word), 0u, KVOPS_ERR_ATTEND_TIMEOUT);
}

static_assert(offsetof(Shared, per_warp) % 16 == 0 && alignof(Shared) % 16 == 0, "read as float4");

// Joins the parts of the units that a CTA's run cuts. Block x is the cut between CTAs x and x + 1, and
// does its unit if it is the first cut in it; eight query rows per block, one per warp. The parts are
// added in their order.
template <typename T, int NQ>
__global__ void __launch_bounds__(256) join_kernel(const KvopsAttend a, const Plan plan)
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t units = real_units(a, plan);
    const uint32_t cut = run_start(plan, units, blockIdx.x + 1);
    if (cut % plan.tiles == 0) return;
    const uint32_t unit = cut / plan.tiles, begin = unit * plan.tiles, end = begin + plan.tiles;
    if (run_start(plan, units, blockIdx.x) > begin) return;
    const Unit u = unit_at<NQ>(a, plan, unit);
    const uint32_t row = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= u.rows) return;
    float top = -INFINITY;
    for (uint32_t c = blockIdx.x; c < plan.ctas && run_start(plan, units, c) < end; ++c) {
        const uint32_t from = run_start(plan, units, c);
        if (run_start(plan, units, c + 1) == from) continue;
        top = fmaxf(top, plan.part_ml[static_cast<uint64_t>(2 * c + (from < begin ? 1 : 0)) * NQ + row].x);
    }
    float total = 0.f;
    float4 acc[4];
    for (int i = 0; i < 4; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t c = blockIdx.x; c < plan.ctas && run_start(plan, units, c) < end; ++c) {
        const uint32_t from = run_start(plan, units, c);
        if (run_start(plan, units, c + 1) == from) continue;
        const uint64_t part = static_cast<uint64_t>(2 * c + (from < begin ? 1 : 0)) * NQ + row;
        const float2 ml = plan.part_ml[part];
        if (ml.x == -INFINITY && ml.y == 0.f) continue;
        const float w = exp2_fast(ml.x - top);
        total += ml.y * w;
        const float4 *o = reinterpret_cast<const float4 *>(plan.part_o + part * kValueDim);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = o[i * 32 + lane];
            acc[i].x += v.x * w, acc[i].y += v.y * w, acc[i].z += v.z * w, acc[i].w += v.w * w;
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    uint2 *out = reinterpret_cast<uint2 *>(a.out) + (u.out_row + row) * (kValueDim / 4);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        out[i * 32 + lane] = make_uint2(T::pack(acc[i].x * inv, acc[i].y * inv), T::pack(acc[i].z * inv, acc[i].w * inv));
    if (lane == 0 && a.lse != 0)
        reinterpret_cast<float *>(a.lse)[u.out_row + row] =
            total == 0.f ? -INFINITY : (top + log2f(total)) * 0.6931471805599453f;
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

// Queries per tile and how the work is dealt out, for `lists` lists per request. The number of
// pairs must stay below 2^32 (check_pairs).
uint32_t queries_per_tile(uint32_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

Plan make_plan(const KvopsAttend &a, uint32_t lists, uint32_t nq, int sms)
{
    Plan p{};
    p.lists = lists;
    p.group_rows = a.heads * (lists > 1 ? 1 : a.tokens);
    p.qtiles = (p.group_rows + nq - 1) / nq;
    p.tiles = (a.top_k + a.drafts + kTile - 1) / kTile;
    if (p.tiles == 0) p.tiles = 1;  // no keys at all: outputs of zero
    const uint64_t units = static_cast<uint64_t>(a.max_num_reqs) * lists * p.qtiles, pairs = units * p.tiles;
    // Whole units need no joining, equal runs of pairs leave no SM idle. In tiles' times: a unit costs
    // its tiles and about one more for its queries and outputs, a cut unit its parts and the joining.
    const uint64_t whole = (units + sms - 1) / sms;
    const uint64_t run = (pairs + sms - 1) / sms;
    const uint64_t cuts = run / p.tiles + 2;
    if (p.tiles == 1 || whole * (p.tiles + 1) <= run + cuts + 3) {
        p.whole = static_cast<uint32_t>(whole);
        p.ctas = static_cast<uint32_t>((units + whole - 1) / whole);
    } else {
        p.ctas = static_cast<uint32_t>(pairs < static_cast<uint64_t>(sms) ? pairs : sms);
    }
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
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<NQ>::bytes);
    if (e != cudaSuccess) return e;
    kernel<<<p.ctas, kThreads, Layout<NQ>::bytes, s>>>(a, p);
    e = cudaGetLastError();
    if (e != cudaSuccess || p.whole > 0 || p.ctas < 2) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.ctas - 1, NQ / 8);
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<T, NQ>, a, p);
}

template <typename T, int NQ>
cudaError_t launch_format(const KvopsAttend &a, const Plan &p, cudaStream_t s)
{
    switch (a.row_format) {
        case KVOPS_ROW_E4M3: return launch_as<T, E4m3, true, NQ>(a, p, s);
        case KVOPS_ROW_INT8: return launch_as<T, Int8, true, NQ>(a, p, s);
        default: return launch_as<T, Int8, false, NQ>(a, p, s);
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
        const uint32_t nq = kvb::queries_per_tile(a->heads * (lists > 1 ? 1 : a->tokens));
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
    const uint32_t nq = kvb::queries_per_tile(a->heads * (lists > 1 ? 1 : a->tokens));
    kvb::Plan p = kvb::make_plan(*a, lists, nq, sms);
    if (static_cast<uint64_t>(a->max_num_reqs) * lists * p.qtiles * p.tiles >= (1ull << 32))
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
