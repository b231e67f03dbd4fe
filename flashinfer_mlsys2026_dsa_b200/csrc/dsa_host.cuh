// Host-side pieces shared by the C ABI's translation units: argument checks and tensor-map
// encoding with a per-thread cache.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <mutex>

#include "dsa_b200.h"

namespace dsa {

// The bound of every wait in the kernels, in SM cycles (set by dsa_set_wait_limit).
uint64_t wait_limit_cycles();

namespace {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn get_encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, []() {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

bool heads_supported(int heads) {
  return heads == 16 || heads == 32 || heads == 64 || heads == 128;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Encoded tensor maps of recent calls (per host thread): a decode loop reuses its pools and
// usually its query buffers, and encoding costs microseconds of host time per map.
struct MapKey {
  const void* base;
  int dtype;
  int rank;
  cuuint64_t dims[3], strides[2];
  cuuint32_t box[3];
  int swz;
  bool operator==(const MapKey& o) const { return memcmp(this, &o, sizeof(MapKey)) == 0; }
};
struct MapCache {
  static constexpr int kWays = 16;
  MapKey key[kWays];
  CUtensorMap map[kWays];
  bool used[kWays] = {};
  int next = 0;
};
thread_local MapCache t_maps;

int encode(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims,
           const cuuint64_t* strides_bytes, const cuuint32_t* box, CUtensorMapSwizzle swz,
           CUtensorMapDataType dtype = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16) {
  MapKey k;
  memset(&k, 0, sizeof(k));  // padding bytes take part in the comparison
  k.base = base;
  k.dtype = (int)dtype;
  k.rank = rank;
  for (int i = 0; i < rank; ++i) {
    k.dims[i] = dims[i];
    k.box[i] = box[i];
  }
  for (int i = 0; i + 1 < rank; ++i) k.strides[i] = strides_bytes[i];
  k.swz = (int)swz;
  MapCache& c = t_maps;
  for (int w = 0; w < MapCache::kWays; ++w)
    if (c.used[w] && c.key[w] == k) {
      *m = c.map[w];
      return DSA_OK;
    }
  EncodeTiledFn fn = get_encode_fn();
  if (!fn) return DSA_ERR_DRIVER;
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(m, dtype, (cuuint32_t)rank, const_cast<void*>(base),
                  dims, strides_bytes, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return DSA_ERR_DRIVER;
  const int w = c.next;
  c.next = (c.next + 1) % MapCache::kWays;
  c.key[w] = k;
  c.map[w] = *m;
  c.used[w] = true;
  return DSA_OK;
}

}  // namespace
}  // namespace dsa
