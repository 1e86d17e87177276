// What the paged-attention kernels share: the parameters on the device, the description of one sequence of the batch and
// the keys that its tokens see.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace llc {

struct PagedArgs {
  const void* q; const void* k; const void* v; void* out;
  const int* table; const int* qStart; const int* kvLen; int* badPages;
  long long qSt, qSh, oSt, oSh, kcSp, kcSn, kcSh, vcSp, vcSn, vcSh, tableS0;
  long long tokens, numPages, pageSize, maxQ;
  int reach, window, sinks;            // slots that a row of the page table names, below 2^31 - 256; window: reach + 1 where the caller has none
  int batch, heads, kvHeads, group, d, dtype;
  float scaleLog2;                     // scale * log2(e): the softmax is taken to base 2
};

// One sequence: rows begin .. begin + n - 1 of q, the i-th of them at place len - n + i.
struct Sequence { long long begin; int n, len; };
__device__ __forceinline__ Sequence sequenceOf(const PagedArgs& p, int b) {
  Sequence s;
  const long long lo = p.qStart[b], hi = p.qStart[b + 1];
  s.begin = lo < 0 ? 0 : lo;
  const long long n = (hi > p.tokens ? p.tokens : hi) - s.begin;
  s.n = n < 0 || n > p.maxQ ? 0 : (int)n;
  const int len = p.kvLen[b];
  s.len = len < 0 ? 0 : len > p.reach ? p.reach : len;
  return s;
}

// Page of slot j of sequence b, -1 where its number is not one of the pool's.
__device__ __forceinline__ long long pageOf(const PagedArgs& p, int b, long long index) {
  const long long page = p.table[b * p.tableS0 + index];
  return page >= 0 && page < p.numPages ? page : -1;
}

// What a row's sums are divided by.  A token at place 0 or later sees at least the key at its own place; one before place 0 sees none and gets
// zeros.  `top` is the maximum of its scores: -inf where all that it sees score -inf, and then the softmax is 0 / 0, whatever the weights were taken
// to be relative to a stand-in for that maximum.
__device__ __forceinline__ float divisorOf(float sum, float top, bool sees) { return !sees ? INFINITY : top == -INFINITY ? NAN : sum; }

// The keys that tokens at places first .. last of a sequence see, some of them at least: [0, sinkEnd) and [lo, hi).  Places below 0
// (more new tokens than the length says) see nothing; they are clipped to -1, so that all of this fits 32 bits.
struct Seen { int sinkEnd, lo, hi; };
__device__ __forceinline__ int clipPlace(long long place) { return place < 0 ? -1 : (int)place; }
__device__ __forceinline__ Seen seenBy(const PagedArgs& p, int first, int last) {
  Seen s;
  s.hi = last + 1;
  s.lo = first + 1 - p.window > 0 ? first + 1 - p.window : 0;
  if (s.lo > s.hi) s.lo = s.hi;
  s.sinkEnd = p.sinks < s.lo ? p.sinks : s.lo;
  return s;
}
// The same in blocks of keys: `sink` blocks from the start, then the blocks from `first` on, `count` in all.
struct Blocks { int sink, first, count; };
__device__ __forceinline__ Blocks blocksOf(const Seen& s, int keys) {
  Blocks b;
  b.first = s.lo / keys;
  b.sink = (s.sinkEnd + keys - 1) / keys;
  if (b.sink > b.first) b.sink = b.first;
  b.count = b.sink + (s.hi + keys - 1) / keys - b.first;
  return b;
}
__device__ __forceinline__ int keyOf(const Blocks& b, int unit, int keys) { return (unit < b.sink ? unit : unit - b.sink + b.first) * keys; }

// Two numbers rounded to T, and whether one of two packed numbers is NaN or infinite.
template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) { __nv_bfloat162 v = __floats2bfloat162_rn(x, y); return *reinterpret_cast<uint32_t*>(&v); }
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) { __half2 v = __floats2half2_rn(x, y); return *reinterpret_cast<uint32_t*>(&v); }
template <typename T> __device__ __forceinline__ bool notFinite(uint32_t x) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (x & e) == e || (x & (e << 16)) == (e << 16);
}
// Weights are rounded to the tensors' type for the second product: the tensor core multiplies two operands of one 16-bit type, and a second product
// with what the rounding left would cost as much again.  bf16 results are then 2.3e-3 from 64 bits, where rounding the result alone leaves 1.6e-3, f16
// 2.9e-4 and 2.1e-4; f32 tensors keep all bits.  f16 weights are kept 2^7 times larger, so that a weight loses
// bits to f16's subnormals only below 2^-21 of the largest (2^7 x 2^8 of lag stays below 65504).
template <typename T> constexpr float weightShift() { return std::is_same<T, __half>::value ? 7.f : 0.f; }
constexpr float kRescaleStep = 8.f;    // the running maximum follows in steps larger than 2^8 only: the weights stay below 2^8

__device__ __forceinline__ float exp2Fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

}  // namespace llc
