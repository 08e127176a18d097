// The sm_100a pieces that a tensor-core tile pipeline is made of: mbarriers
// with bounded waits, TMA tile copies, tensor memory and tcgen05 products, and
// the host's tensor maps.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace mg {

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}

// ------------------------------------------------------------------ mbarriers

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
// The copying and the issuing warp run their loops with all lanes, so that
// addresses and descriptors stay in uniform registers, and one lane (`on`)
// executes the instruction. A product's operands come from uniform registers:
// moving them there from a lane's takes 50 to 210 cycles a product, where 64
// columns keep the tensor core for 32 (measured, 128 x n x 16).
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t on;
    asm volatile(
        "{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}"
        : "=r"(on));
    return on;
}
// v, the same in all lanes, as a uniform register.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_or_sync(0xffffffffu, v); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes, uint32_t on) {
    asm volatile(
        "{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\n"
        "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}" ::"r"(bar),
        "r"(bytes), "r"(on)
        : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// Every wait ends: after `rounds` rounds (kMbarRounds outside the self-test, some
// 4 s at the 3.7 us that one takes when nothing arrives) it gives up, records
// `code` in the device error word and raises the block's stop flag, which ends
// the block's other waits too. A round is one try_wait, which the hardware may
// suspend. Nothing that is not valid is read before the flag is up, so who stores
// results looks at it after the last read: NaN if it is.
constexpr int kMbarRounds = 1 << 20;
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, int rounds, volatile int* stop,
                                          int32_t* error_word, int32_t code) {
    if (mbar_try(bar, parity)) return true;
    for (int i = 1; i < rounds; ++i) {
        if (*stop) return false;
        if (mbar_try(bar, parity)) return true;
    }
    if (*stop) return false;
    *stop = 1;
    record_device_error(error_word, code);
    return false;
}

// The same for a whole warp, which agrees on the answer (and stays in step).
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, int rounds, volatile int* stop,
                                               int32_t* error_word, int32_t code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, rounds, stop, error_word, code));
}

// ------------------------------------------------------------------------ TMA

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                         uint32_t bar, uint32_t on) {
    asm volatile(
        "{\n.reg .pred q;\nsetp.ne.u32 q, %6, 0;\n"
        "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];\n}" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(on)
        : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, int x, int y, int z, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(src)
                 : "memory");
}
__device__ __forceinline__ void tma_store_commit() {
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_store_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void tma_store_wait_all() {
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ void fence_async_shared() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void named_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// --------------------------------------------------------- tensor memory, MMA

__device__ __forceinline__ void tmem_alloc(uint32_t dst_smem, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
// A block that asks for all 512 columns has them from address 0 on.
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kTmemBase = 0;
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns)
                 : "memory");
}
__device__ __forceinline__ void tmem_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// 32 lanes x 32 columns of fp32: lane i of the warp gets row i's columns.
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// D (fp32, tensor memory) = or += A B, one step of 16 along the contraction;
// A and B are bf16 tiles in shared memory behind their descriptors, given as
// the low word (address and block stride) and the constant high word.
template <uint32_t A_HI, uint32_t B_HI>
__device__ __forceinline__ void mma_bf16(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                         bool add, uint32_t on) {
    asm volatile(
        "{\n.reg .pred p, q;\n.reg .b64 da, db;\nsetp.ne.u32 p, %4, 0;\nsetp.ne.u32 q, %5, 0;\n"
        "mov.b64 da, {%1, %6};\nmov.b64 db, {%2, %7};\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(on), "n"(A_HI), "n"(B_HI)
        : "memory");
}
// The same with A in tensor memory: row i in lane i, two contraction entries
// to a 32-bit column.
template <uint32_t B_HI>
__device__ __forceinline__ void mma_bf16_ta(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                            bool add, uint32_t on) {
    asm volatile(
        "{\n.reg .pred p, q;\n.reg .b64 db;\nsetp.ne.u32 p, %4, 0;\nsetp.ne.u32 q, %5, 0;\n"
        "mov.b64 db, {%2, %6};\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(on), "n"(B_HI)
        : "memory");
}
// The barrier gets an arrival when every product issued so far is done.
__device__ __forceinline__ void mma_commit(uint32_t bar, uint32_t on) {
    asm volatile(
        "{\n.reg .pred q;\nsetp.ne.u32 q, %1, 0;\n"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar),
        "r"(on)
        : "memory");
}

// bf16 x bf16 -> fp32, 128 rows by n columns; *_mn: the operand is stored with
// its row (not its contraction) index running fastest.
__device__ __forceinline__ uint32_t mma_idesc(int n, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

// Descriptors. A tile whose contraction index runs fastest, `bytes` (128 or
// 64) to a row: groups of 8 rows follow one another.
__host__ __device__ constexpr uint32_t k_major_hi(int bytes) {
    return (uint32_t)(8 * bytes / 16) | 1u << 14 | (bytes == 128 ? 2u : 4u) << 29;
}
__device__ __forceinline__ uint32_t k_major_lo(uint32_t addr) {
    return ((addr & 0x3ffffu) >> 4) | 1u << 16;
}
// A tile whose row index runs fastest: blocks of 64 rows (128 bytes) by the
// contraction, block_bytes from one block of rows to the next.
constexpr uint32_t kMnMajorHi = (1024u / 16) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t mn_major_lo(uint32_t addr, int block_bytes) {
    return ((addr & 0x3ffffu) >> 4) | (uint32_t)(block_bytes / 16) << 16;
}

// ----------------------------------------------------------------------- host

// A (columns, rows, parts) bf16 tensor and the tile copied from it; strides in
// bytes, multiples of 16. Reads past an edge give zeros, writes are dropped.
mg_status make_tensor_map(CUtensorMap* map, const void* base, int64_t columns, int64_t rows,
                          int64_t parts, int64_t row_bytes, int64_t part_bytes, int box_columns,
                          int box_rows, bool swizzle128, const char* what);

}  // namespace mg
