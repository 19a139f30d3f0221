// Fragments of key blocks in LDS, as the attention kernels that fill it with
// direct-to-LDS copies read them.
#pragma once

#include "common.h"

namespace parrot {

// N fragments from LDS at addr + B + S i, landed on return.  By inline asm,
// because the compiler would otherwise wait for the direct-to-LDS copies in
// flight (the next stages) before every read; loads and wait are one block,
// so no register is named before its data is there.
template <int B, int S>
__device__ __forceinline__ void lds_frags(uint32_t addr, bf16x8 (&f)[4]) {
  asm volatile(
      "ds_read_b128 %0, %4 offset:%5\n\tds_read_b128 %1, %4 offset:%6\n\t"
      "ds_read_b128 %2, %4 offset:%7\n\tds_read_b128 %3, %4 offset:%8\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3])
      : "v"(addr), "i"(B), "i"(B + S), "i"(B + 2 * S), "i"(B + 3 * S));
}

template <int B, int S>
__device__ __forceinline__ void lds_frags(uint32_t addr, bf16x8 (&f)[6]) {
  asm volatile(
      "ds_read_b128 %0, %6 offset:%7\n\tds_read_b128 %1, %6 offset:%8\n\t"
      "ds_read_b128 %2, %6 offset:%9\n\tds_read_b128 %3, %6 offset:%10\n\t"
      "ds_read_b128 %4, %6 offset:%11\n\tds_read_b128 %5, %6 offset:%12\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5])
      : "v"(addr), "i"(B), "i"(B + S), "i"(B + 2 * S), "i"(B + 3 * S), "i"(B + 4 * S),
        "i"(B + 5 * S));
}

template <int B, int S>
__device__ __forceinline__ void lds_frags(uint32_t addr, bf16x8 (&f)[8]) {
  asm volatile(
      "ds_read_b128 %0, %8 offset:%9\n\tds_read_b128 %1, %8 offset:%10\n\t"
      "ds_read_b128 %2, %8 offset:%11\n\tds_read_b128 %3, %8 offset:%12\n\t"
      "ds_read_b128 %4, %8 offset:%13\n\tds_read_b128 %5, %8 offset:%14\n\t"
      "ds_read_b128 %6, %8 offset:%15\n\tds_read_b128 %7, %8 offset:%16\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]),
        "=&v"(f[6]), "=&v"(f[7])
      : "v"(addr), "i"(B), "i"(B + S), "i"(B + 2 * S), "i"(B + 3 * S), "i"(B + 4 * S),
        "i"(B + 5 * S), "i"(B + 6 * S), "i"(B + 7 * S));
}

// The V fragments of one key block, vf[2 i + s] = 32-dim tile i, 16-key step s
// (bytes 2048 i + 512 s from the lane's piece).
template <int B, int N>
__device__ __forceinline__ void read_values(uint32_t addr, bf16x8 (&vf)[N]) {
  static_assert(N == 4 || N == 6 || N == 8, "two to four 32-dim tiles");
  if constexpr (N == 4)
    asm volatile(
        "ds_read_b128 %0, %4 offset:%5\n\tds_read_b128 %1, %4 offset:%6\n\t"
        "ds_read_b128 %2, %4 offset:%7\n\tds_read_b128 %3, %4 offset:%8\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(vf[0]), "=&v"(vf[1]), "=&v"(vf[2]), "=&v"(vf[3])
        : "v"(addr), "i"(B), "i"(B + 512), "i"(B + 2048), "i"(B + 2560));
  else if constexpr (N == 6)
    asm volatile(
        "ds_read_b128 %0, %6 offset:%7\n\tds_read_b128 %1, %6 offset:%8\n\t"
        "ds_read_b128 %2, %6 offset:%9\n\tds_read_b128 %3, %6 offset:%10\n\t"
        "ds_read_b128 %4, %6 offset:%11\n\tds_read_b128 %5, %6 offset:%12\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(vf[0]), "=&v"(vf[1]), "=&v"(vf[2]), "=&v"(vf[3]), "=&v"(vf[4]), "=&v"(vf[5])
        : "v"(addr), "i"(B), "i"(B + 512), "i"(B + 2048), "i"(B + 2560), "i"(B + 4096),
          "i"(B + 4608));
  else
    asm volatile(
        "ds_read_b128 %0, %8 offset:%9\n\tds_read_b128 %1, %8 offset:%10\n\t"
        "ds_read_b128 %2, %8 offset:%11\n\tds_read_b128 %3, %8 offset:%12\n\t"
        "ds_read_b128 %4, %8 offset:%13\n\tds_read_b128 %5, %8 offset:%14\n\t"
        "ds_read_b128 %6, %8 offset:%15\n\tds_read_b128 %7, %8 offset:%16\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(vf[0]), "=&v"(vf[1]), "=&v"(vf[2]), "=&v"(vf[3]), "=&v"(vf[4]), "=&v"(vf[5]),
          "=&v"(vf[6]), "=&v"(vf[7])
        : "v"(addr), "i"(B), "i"(B + 512), "i"(B + 2048), "i"(B + 2560), "i"(B + 4096),
          "i"(B + 4608), "i"(B + 6144), "i"(B + 6656));
}

}  // namespace parrot
