// tcgen05.cuh — the inline PTX of the fifth-generation tensor core that attend.cu issues: shared
// memory descriptors, matrix instructions, tensor memory loads and stores, and mbarriers whose
// waits are bounded.
#pragma once

#include <stdint.h>

namespace kvb {
namespace tc {

__device__ __forceinline__ uint32_t smem_addr(const void *p)
{
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.b32 %0, 1, 0, p; }"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// The whole warp waits for the phase of this parity, or until another wait of the CTA has given up
// (*stop). Gives up itself, and says so in *stop, after kWaitClocks (half a second or more; the SM's own
// clock, since reading the global timer takes microseconds). The warp leaves together: a lane left
// behind could find the barrier two phases on, where the parity is its own again, and wait for good.
constexpr long long kWaitClocks = 1ll << 30;
__device__ __noinline__ void mbar_wait_on(uint32_t bar, uint32_t parity, volatile uint32_t *stop)
{
    const long long start = clock64();
    while (!mbar_try(bar, parity)) {
        if (*stop != 0) break;
        if (clock64() - start > kWaitClocks) {
            *stop = 1u;
            break;
        }
    }
}
__device__ __forceinline__ void mbar_wait(uint32_t bar, uint32_t parity, volatile uint32_t *stop)
{
    if (!mbar_try(bar, parity)) mbar_wait_on(bar, parity, stop);
    __syncwarp();
}

// What generic stores wrote to shared memory becomes visible to the matrix instructions.
__device__ __forceinline__ void fence_async_shared()
{
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Descriptor of an operand in 128-byte rows under the 128-byte swizzle (16-byte unit u of row i of
// each 1024-byte block lies at unit u ^ (i & 7)). Contraction along the row (K-major): sbo is the
// distance of 8 rows. Contraction across the rows (MN-major): lbo is the distance from 64 values
// of a row to the next 64, sbo that of 8 rows.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lbo, uint32_t sbo)
{
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lbo >> 4) << 16) |
           (static_cast<uint64_t>(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction word of kind::f16 with fp32 accumulators: type 0 is fp16, 1 bf16, for both operands;
// mn: both operands are MN-major.
__host__ __device__ constexpr uint32_t instruction(uint32_t type, bool mn, uint32_t m, uint32_t n)
{
    return (1u << 4) | (type << 7) | (type << 10) | (mn ? (1u << 15) | (1u << 16) : 0u) | ((n / 8) << 17) |
           ((m / 16) << 24);
}

// acc (in tensor memory) = a * b + (accumulate ? acc : 0), 16 deep. The whole warp comes here and the
// one lane with `elected` issues: the operands are then uniform over the warp and stay in uniform
// registers (issued from a branch of one lane, each took some 90 cycles to move there).
__device__ __forceinline__ void mma(uint32_t elected, uint32_t acc, uint64_t a, uint64_t b, uint32_t inst, bool accumulate)
{
    asm volatile(
        "{ .reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0; "
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(acc),
        "l"(a), "l"(b), "r"(inst), "r"(accumulate ? 1u : 0u), "r"(elected) : "memory");
}
// The barrier gets an arrival once every matrix instruction that the lane issued so far has ended.
__device__ __forceinline__ void commit(uint32_t elected, uint32_t bar)
{
    asm volatile(
        "{ .reg .pred q; setp.ne.b32 q, %1, 0; "
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(bar), "r"(elected)
        : "memory");
}
// Waits until every matrix instruction that the elected lane issued has ended, and every arrival that it
// committed has been made, whether or not another wait has given up: `bar` is a barrier of one arrival that nothing
// else uses. Issued instructions always end; the limit only keeps the wait bounded.
__device__ __forceinline__ void drain(uint32_t elected, uint32_t bar)
{
    commit(elected, bar);
    const long long start = clock64();
    while (!mbar_try(bar, 0))
        if (clock64() - start > kWaitClocks) break;
    __syncwarp();
}
// 1 in one lane of the converged warp.
__device__ __forceinline__ uint32_t elect()
{
    uint32_t e;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(e));
    return e;
}

template <uint32_t kCols>
__device__ __forceinline__ void tmem_alloc(uint32_t *where)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(where)), "n"(kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <uint32_t kCols>
__device__ __forceinline__ void tmem_free(uint32_t at)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "n"(kCols));
}

// The calling warp's 32 lanes (one per thread) of kN columns from `at`; at names the warp's lanes.
// The load and its wait are one statement: nothing may use the values between them.
template <int kN>
__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[kN])
{
    static_assert(kN == 8 || kN == 16 || kN == 32, "columns");
    uint32_t r[kN];
    if constexpr (kN == 8) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x8.b32 {"
            "%0,%1,%2,%3,%4,%5,%6,%7"
            "}, [%8]; tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
            : "r"(at) : "memory");
    } else if constexpr (kN == 16) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
            "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15"
            "}, [%16]; tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
              "=r"(r[15])
            : "r"(at) : "memory");
    } else {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
            "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%2"
            "2,%23,%24,%25,%26,%27,%28,%29,%30,%31"
            "}, [%32]; tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
              "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
              "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
              "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
            : "r"(at) : "memory");
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = __uint_as_float(r[i]);
}
// Lanes 0-15 of the calling warp's quarter, 8 kBlocks columns from `at`, spread over all its threads:
// v[4 b + 2 r + e] of thread t is lane t / 4 + 8 r, column 8 b + 2 (t % 4) + e.
template <int kBlocks>
__device__ __forceinline__ void tmem_load_spread(uint32_t at, float (&v)[4 * kBlocks])
{
    static_assert(kBlocks == 1 || kBlocks == 2 || kBlocks == 4, "blocks");
    uint32_t r[4 * kBlocks];
    if constexpr (kBlocks == 1) {
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4]; "
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
            : "r"(at) : "memory");
    } else if constexpr (kBlocks == 2) {
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8]; "
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
            : "r"(at) : "memory");
    } else {
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16]; "
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
              "=r"(r[15])
            : "r"(at) : "memory");
    }
#pragma unroll
    for (int i = 0; i < 4 * kBlocks; ++i) v[i] = __uint_as_float(r[i]);
}
template <int kN>
__device__ __forceinline__ void tmem_store(uint32_t at, const float (&v)[kN])
{
    static_assert(kN == 8 || kN == 16 || kN == 32, "columns");
#pragma unroll
    for (int c = 0; c < kN; c += 8)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at + c),
                     "r"(__float_as_uint(v[c])), "r"(__float_as_uint(v[c + 1])), "r"(__float_as_uint(v[c + 2])),
                     "r"(__float_as_uint(v[c + 3])), "r"(__float_as_uint(v[c + 4])), "r"(__float_as_uint(v[c + 5])),
                     "r"(__float_as_uint(v[c + 6])), "r"(__float_as_uint(v[c + 7])) : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

}  // namespace tc
}  // namespace kvb
