// tcgen05_utils.cuh — wrappers of the tensor-memory and mbarrier instructions the attention kernels use, and waits
// that give up after a second or so.
#pragma once

#include "device_utils.cuh"

namespace ds4b200 {
namespace tc {

constexpr int kWaitPolls = 1 << 22;               // with a sleep of 20 to 300 ns (NS) ahead of each: a tenth of a second to one or two

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operands: 128-byte rows, 128-byte swizzle, groups of eight rows 1024 bytes apart.  The low word of the
// descriptor holds the address and, where the operand lies with its long side contiguous, `lbo`, the distance between
// blocks of 64 elements of that side; the high word is the same for all.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return ((lbo >> 4) << 16) | ((saddr & 0x3FFFFu) >> 4); }
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// f16 x f16 -> f32, both operands in shared memory; bit 15: A lies with M contiguous.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool a_m_major) {
    return (1u << 4) | (a_m_major ? 1u << 15 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// One lane of a converged warp (always the same one).
__device__ __forceinline__ uint32_t elect() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e;
}
// Issued by the lane with `one` set, as a predicate of the instruction.  The whole warp runs the loop around it, on values the
// compiler knows to be uniform (a shuffle from lane 0): the operands then live in uniform registers, and an MMA of M 64, N 64, K 16
// takes the 32 cycles its 4 KiB of operands need of shared memory.  Issued from a branch that one lane takes, each operand moves
// to a uniform register for every MMA, and the same MMA took 48 to 150 cycles, depending on the code around it.
__device__ __forceinline__ void mma_f16(uint32_t one, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "setp.ne.b32 q, %6, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHi), "r"(one) : "memory");
}
// One arrival on the barrier when every MMA the electing lane has issued so far has finished.
__device__ __forceinline__ void commit(uint32_t one, uint32_t bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                 ::"r"(bar), "r"(one) : "memory");
}
template <int N> __device__ __forceinline__ void set_max_registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void set_max_registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// 16 lanes x 64 columns: register 4 i + k of lane t is row t / 4 + 8 (k / 2), column 8 i + 2 (t % 4) + k % 2.
__device__ __forceinline__ void ld_16x64(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
// The same for 32 columns.
__device__ __forceinline__ void ld_16x32(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ float exp2_approx(float x) {     // ex2.approx.ftz: relative error 2^-22, 0 below 2^-126
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
                 : "memory");
}

// Barriers go by their shared-memory address, held in a register: from a pointer the compiler works the address out again, three
// instructions, at every poll.
__device__ __forceinline__ uint32_t held(uint32_t x) {
    asm volatile("mov.u32 %0, %0;" : "+r"(x));
    return x;
}
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool try_phase(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A box of a two-dimensional tensor map into this CTA's shared memory.
__device__ __forceinline__ void load_box(uint32_t dst, const void *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
// A wait on an mbarrier phase.  It polls at most kWaitPolls times; the first that runs out raises the status bit and a
// CTA-wide flag with which every later wait returns soon, so the kernel always ends (its results are invalid then).  Returns whether the
// phase was found: if not, what the wait was for may not be used.  A poll takes
// issue slots and shared-memory bandwidth from the warps that work: with polls every 40 ns the waiting warps issued a third of
// all instructions.
template <int NS = 100>
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int *status, int polls = kWaitPolls) {
    if (try_phase(bar, parity)) return true;
#pragma unroll 1
    for (int i = 1; i <= polls; ++i) {
        __nanosleep(NS);
        if (try_phase(bar, parity)) return true;
        if ((i & 63) == 0 && *abort_flag) return false;
    }
    *abort_flag = 1;
    if (status) atomicOr(status, kStatusBulkCopyTimeout);
    return false;
}

// For what is still in flight when a kernel gives up.
__device__ __forceinline__ void settle(uint32_t bar, uint32_t parity) {
#pragma unroll 1
    for (int i = 0; i < (1 << 16) && !try_phase(bar, parity); ++i) __nanosleep(100);
}

}  // namespace tc
}  // namespace ds4b200
