// Device-side pieces shared by the decode kernels: the operator's widths, UMMA instruction
// descriptors, the swizzled operand layout and the bounded mbarrier wait.
#pragma once
#include <stdint.h>

#include "dsa_b200.h"
#include "sm100_ptx.cuh"

namespace dsa {

constexpr int kDCkv = 512;            // latent (value) width
constexpr int kDKpe = 64;             // rope key width
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint64_t kWaitCycles = 4000000000ull;  // default wait bound: ~2 s at ~2 GHz

constexpr uint32_t kSw128 = 2, kSw64 = 4;  // UMMA descriptor layout types

// UMMA shared-memory descriptor (sm_100, version 1): start, leading and stride byte offsets.
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo, uint32_t sbo,
                                         uint32_t layout) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)layout << 61);
}

// Instruction descriptor, kind::f16: bf16 A/B, fp32 D; A and B K-major unless flagged.
__host__ __device__ constexpr uint32_t idesc_bf16(int M, int N, bool a_mn_major,
                                                  bool b_mn_major = false) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn_major ? 1u : 0u) << 15) |
         ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Byte offset of element (row h, column k) in a [rows x 64] bf16 tile stored
// K-major with the 128-byte swizzle (the UMMA canonical SW128 K-major layout).
__device__ __forceinline__ uint32_t sw128_off(int h, int k) {
  return (uint32_t)((h >> 3) * 1024 + (h & 7) * 128 + ((((k >> 3) ^ (h & 7))) << 4) + (k & 7) * 2);
}

// Bounded mbarrier wait.  `spin` polls without letting the hardware suspend the thread
// (for the latency-critical MMA issuer); otherwise try_wait may suspend it briefly.
struct Waiter {
  volatile uint32_t* abort_flag;
  uint32_t* err;
  uint64_t limit;  // cycles
  bool spin = false;
  __device__ __forceinline__ bool poll(uint32_t bar, uint32_t parity) const {
    return spin ? ptx::mbar_test_wait(bar, parity) : ptx::mbar_try_wait(bar, parity);
  }
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
    if (poll(bar, parity)) return true;
    const uint64_t t0 = ptx::cycles();
    for (uint32_t it = 1;; ++it) {
      if (poll(bar, parity)) return true;
      if ((it & 63u) == 0) {
        if (*abort_flag) return false;
        if (ptx::cycles() - t0 > limit) {
          *abort_flag = 1;
          atomicOr(err, (uint32_t)DSA_DEVERR_TIMEOUT);
          return false;
        }
      }
    }
  }
};

}  // namespace dsa
