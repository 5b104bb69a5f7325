/*
 * 32 bytes of memory at a time: the unit that the L2 fetches and that memory
 * is written whole in.
 */
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace noel {

struct Sector {
    uint32_t u[8];
};
__device__ __forceinline__ Sector sector_load(const void *p) {
    Sector s;
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(s.u[0]), "=r"(s.u[1]), "=r"(s.u[2]), "=r"(s.u[3]), "=r"(s.u[4]), "=r"(s.u[5]), "=r"(s.u[6]),
                   "=r"(s.u[7])
                 : "l"(p));
    return s;
}
__device__ __forceinline__ void sector_store(void *p, const Sector &s) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(s.u[0]), "r"(s.u[1]),
                 "r"(s.u[2]), "r"(s.u[3]), "r"(s.u[4]), "r"(s.u[5]), "r"(s.u[6]), "r"(s.u[7])
                 : "memory");
}
/* the same on 16-byte aligned memory */
__device__ __forceinline__ void sector_store16(void *p, const Sector &s) {
    static_cast<uint4 *>(p)[0] = make_uint4(s.u[0], s.u[1], s.u[2], s.u[3]);
    static_cast<uint4 *>(p)[1] = make_uint4(s.u[4], s.u[5], s.u[6], s.u[7]);
}

}  // namespace noel
