// Buffer-to-LDS copies (buffer_load .. lds): the data goes from memory into LDS without passing through
// registers, offsets past the buffer copy zeros, and a wave's copies land in the order of their issue.
#pragma once

#include "tsa_common.h"

namespace tsa {
namespace {

typedef int buf_v4i __attribute__((ext_vector_type(4)));

__device__ __forceinline__ buf_v4i buf_desc(const void* p, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return buf_v4i{__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)),
                  __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}

// Lane l's 16 (or 4) bytes at buffer offset voff + soff land at LDS byte lds + 16 l (or 4 l).
__device__ __forceinline__ void lds_copy16(const buf_v4i& r, uint32_t voff, uint32_t soff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\t" TSA_COPY_WAIT "buffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(r), "s"(soff),
                 "s"(__builtin_amdgcn_readfirstlane((int)lds))
                 : "memory", "m0");
}
__device__ __forceinline__ void lds_copy4(const buf_v4i& r, uint32_t voff, uint32_t soff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\t" TSA_COPY_WAIT "buffer_load_dword %0, %1, %2 offen lds" ::"v"(voff), "s"(r), "s"(soff),
                 "s"(__builtin_amdgcn_readfirstlane((int)lds))
                 : "memory", "m0");
}

// This wave's copies have landed but for the newest N, and its LDS reads are done; then the barrier.
template <int N>
__device__ __forceinline__ void wait_copies_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

}  // namespace
}  // namespace tsa
