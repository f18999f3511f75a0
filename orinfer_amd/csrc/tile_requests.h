// Requests from memory to LDS for the products by tiles, in asm statements, waited for by hand.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace orx {
namespace tile_requests {

// Requests to LDS where `wanted` is above 0, by a branch inside the statement: the K loop stays one block.  16 or 4 bytes a lane, one lane behind the other.
#define ORX_WANTED(BODY) "s_cmp_gt_i32 %2, 0\n\ts_cbranch_scc0 .Lskipped%=\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t" BODY "\n.Lskipped%=:"
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is reserved: it holds nothing of the compiler's from one statement to the next)
__device__ __forceinline__ void request_16_from(const uint8_t* lane_address, uint32_t lds_wave_base, int wanted) {
    asm volatile(ORX_WANTED("global_load_lds_dwordx4 %0, off") ::"v"(lane_address), "s"(lds_wave_base), "s"(wanted) : "memory", "m0", "scc");
}
__device__ __forceinline__ const uint8_t* uniform_pointer(const uint8_t* pointer) {
    const uint64_t bits = reinterpret_cast<uint64_t>(pointer);
    const uint32_t low = __builtin_amdgcn_readfirstlane((uint32_t)bits), high = __builtin_amdgcn_readfirstlane((uint32_t)(bits >> 32));
    return reinterpret_cast<const uint8_t*>(((uint64_t)high << 32) | low);
}
__device__ __forceinline__ void request_4_from(const uint8_t* lane_address, uint32_t lds_wave_base, int wanted) {
    asm volatile(ORX_WANTED("global_load_lds_dword %0, off") ::"v"(lane_address), "s"(lds_wave_base), "s"(wanted) : "memory", "m0", "scc");
}
// one kilobyte
__device__ __forceinline__ void request_half_tile(uint32_t lane_offset, const uint8_t* uniform_base, uint32_t lds_wave_base, int wanted) {
    asm volatile(ORX_WANTED("global_load_lds_dwordx4 %0, %3") ::"v"(lane_offset), "s"(lds_wave_base), "s"(wanted), "s"(uniform_base) : "memory", "m0", "scc");
}
// two kilobytes that lie together on both sides
__device__ __forceinline__ void request_tile(uint32_t lane_offset, const uint8_t* uniform_base, uint32_t lds_wave_base, int wanted) {
    asm volatile(ORX_WANTED("global_load_lds_dwordx4 %0, %3\n\tglobal_load_lds_dwordx4 %0, %3 offset:1024") ::"v"(lane_offset), "s"(lds_wave_base), "s"(wanted), "s"(uniform_base)
                 : "memory", "m0", "scc");
}
#pragma clang diagnostic pop
#undef ORX_WANTED
// All requests and LDS reads of this wave have ended, and those of the others.  (The builtin, not a statement: the compiler then knows that its reads are there.)
__device__ __forceinline__ void everybody_arrived() {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The same, but the newest PENDING of this wave's requests may be on their way where `all` is above 0.
template <int PENDING>
__device__ __forceinline__ void everybody_arrived_but(int all) {
    static_assert(PENDING > 0 && PENDING < 64, "vmcnt has six bits");
    asm volatile("s_cmp_gt_i32 %0, 0\n\ts_cbranch_scc0 .Lnone%=\n\ts_waitcnt vmcnt(%1)\n\ts_branch .Ldone%=\n.Lnone%=:\n\ts_waitcnt vmcnt(0)\n.Ldone%=:" ::"s"(all), "n"(PENDING) : "memory", "scc");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

}  // namespace tile_requests
}  // namespace orx
