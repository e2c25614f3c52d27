// Shared by the kernels of the paged 4-bit cache and of beam search.
#pragma once
#include "common.cuh"
#include "kv4_layout.h"

namespace cb {

// Kernel-side refusal of an index that came from device memory: the access is skipped and the next synchronising call reports it.
__device__ __forceinline__ void report_bad_index(int *status, int site, int detail) {
  if (atomicCAS(status, 0, DEV_BAD_INDEX) == 0) { status[1] = site; status[2] = detail; }
}

int kv4_check(caten_b200_ctx *ctx, const char *who, const caten_b200_kv4_desc *c, Kv4Shape *s);

}  // namespace cb
