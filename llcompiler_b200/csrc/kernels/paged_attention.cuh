// What the paged-attention kernels share: the parameters on the device, the description of one sequence of the batch and
// the keys that its tokens see.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace llc {

struct PagedArgs {
  const void* q; const void* k; const void* v; void* out;
  const int* table; const int* qStart; const int* kvLen; int* badPages;
  long long qSt, qSh, oSt, oSh, kcSp, kcSn, kcSh, vcSp, vcSn, vcSh, tableS0;
  long long tokens, numPages, pageSize, reach, maxQ;
  long long window, sinks;             // window: past the longest sequence where the caller has none
  int batch, heads, kvHeads, group, d, dtype;
  float scaleLog2;                     // scale * log2(e): the softmax is taken to base 2
};

// One sequence: rows begin .. begin + n - 1 of q, the i-th of them at place len - n + i.
struct Sequence { long long begin, n, len; };
__device__ __forceinline__ Sequence sequenceOf(const PagedArgs& p, int b) {
  Sequence s;
  const long long lo = p.qStart[b], hi = p.qStart[b + 1];
  s.begin = lo < 0 ? 0 : lo;
  s.n = (hi > p.tokens ? p.tokens : hi) - s.begin;
  if (s.n < 0 || s.n > p.maxQ) s.n = 0;
  const long long len = p.kvLen[b];
  s.len = len < 0 ? 0 : len > p.reach ? p.reach : len;
  return s;
}

// Page of slot j of sequence b, -1 where its number is not one of the pool's.
__device__ __forceinline__ long long pageOf(const PagedArgs& p, int b, long long index) {
  const long long page = p.table[b * p.tableS0 + index];
  return page >= 0 && page < p.numPages ? page : -1;
}

__device__ __forceinline__ float exp2Fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

}  // namespace llc
