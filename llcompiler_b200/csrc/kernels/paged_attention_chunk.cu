// Paged attention for chunks of new tokens, on the 5th-generation tensor cores.
// Mathematics: as in the decode kernel, out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m) with a running m.  The rows of a tile are
// (token, query head) pairs of one key head, token-major, so that all query heads of a group read the keys once and a tile's rows
// differ little in what they see.
// A CTA takes two tiles of 128 rows and walks the blocks of 128 keys that either sees:
//   16 softmax warps  eight a tile, two threads a row: a thread's 64 scores come out of tensor memory into registers once; maximum,
//                     2^x, sum, weights back into tensor memory as 16-bit numbers over the scores' own columns, from where the
//                     second product takes them as its A operand (they never cross shared memory).  (One thread a row, eight
//                     warps: the schedulers found a warp to issue from in 31 % of the cycles.)
//   loader warp       one lane a page box: TMA loads of K and V blocks into a ring of slots
//   issuer warp       S_A, S_B, then for every block: O_A += P_A V, S_A of the next block, O_B += P_B V, S_B of the next block, so that
//                     one tile's softmax runs under the other tile's products
// Tensor memory: S_A, S_B (128 columns each), O_A, O_B (d columns each).  The issuer's products run in the order of issue, so the next
// S_A may overwrite P_A as soon as O_A += P_A V has been issued.
// Bound: at d = 128 a block of two tiles costs 2048 cycles of products and as many of exponentials (16 a cycle and SM); it takes 3460, a
// tile's chain score -> weight -> sum -> next score, of which the other tile's fills a part.  Measured: 1.8 - 2.0 us a block (1250 to 1390
// TFLOP/s in the steady state), 4096 tokens over 16384 keys of 32 heads of 128 0.86 ms (1120 TFLOP/s) after a pause and 0.94 - 0.97 ms (1000 TFLOP/s) call
// after call, under the power cap; d = 64 1.5 - 1.6 us a block.
#include "page_map.h"
#include "paged_attention.cuh"
#include "tc_common.cuh"

namespace llc {
__device__ int g_pagedChunkStatus = 0;    // non-zero after a bounded wait gave up: 10 loader, 11 issuer, 12 softmax

namespace {
using namespace tc;

constexpr int kSoftmaxWarps = 16, kLoaderWarp = 16, kIssuerWarp = 17;
constexpr int kThreads = 20 * 32;          // the last two warps are idle: they fill the warpgroup that gives registers away
constexpr int kTileRows = 128, kCtaRows = 256, kKeys = 128;
// Least blocks of a part.  Nine sequences of up to 2048 keys: 59 us with 2, 35 with 12; 40 tokens of 32 heads over 500 keys: 48 us in parts of one
// block, 17 whole.
constexpr int kCutBlocks = 12;
constexpr int kMaxSplits = 32;

template <int D> struct Config {
  static constexpr int kAtom = 128 * 128;             // bytes of 128 rows x 64 elements
  static constexpr int kTile = kAtom * (D / 64);      // Q of a tile, K or V of a block
  static constexpr int kSlots = D == 128 ? 5 : 10;
  static constexpr int kMisc = 3072;                  // barriers, then the row statistics that a row's two threads exchange
  static constexpr int kSmem = 2 * kTile + kSlots * kTile + kMisc;
  static constexpr int kPart = kTileRows * (D + 2);   // floats of a tile's partial sums: O as [D / 4][128 rows] vectors, then m, then l
  static_assert(kSmem <= 227 * 1024, "one CTA an SM");
};
// Columns of tensor memory.
constexpr uint32_t kColS = 0, kColO = 256;

struct ChunkArgs {
  PagedArgs p;
  int doneRows;                // sequences of at most so many rows are the decode kernel's
  int pageShift, boxRows;
  int maxCut, maxSplits;       // CTAs that cut keys may fill, one and a half times the SMs (0: no key is cut), most parts of a pair's keys
  float scaleAbs, signQ;       // the scale's size; its sign goes into Q, so that the largest product is the largest score
  int4* records;               // [0]: pairs of tiles of the call, CTAs of each; then of each pair its sequence, its tile and the parts of its keys
  float* parts;                // [pairs][2][CTAs of a pair][kPart]
};

// What a tile's rows see.
struct Tile {
  int first, last;             // places of its first and last token
  Seen seen;
};
__device__ __forceinline__ Tile tileOf(const PagedArgs& p, const Sequence& s, int row0, int rows) {
  Tile t;
  const int rowEnd = rows - row0 > kTileRows ? row0 + kTileRows : rows;
  if (row0 >= rowEnd) { t.first = 0; t.last = -1; t.seen = Seen{0, 0, 0}; return t; }
  t.first = clipPlace((long long)s.len - s.n + (uint32_t)row0 / (uint32_t)p.group);
  t.last = clipPlace((long long)s.len - s.n + (uint32_t)(rowEnd - 1) / (uint32_t)p.group);
  t.seen = seenBy(p, t.first, t.last);
  return t;
}
// The same in units (positions in the CTA's list of blocks): a tile takes part in units u < sink and lo <= u < hi, and every row of it sees
// all keys of the units u < wholeSink and wholeLo <= u < wholeHi.
struct Units { int sink, lo, hi, wholeSink, wholeLo, wholeHi; };
__device__ __forceinline__ Units unitsOf(const PagedArgs& p, const Tile& t, const Blocks& bl) {
  Units n;
  const int shift = bl.sink - bl.first;               // unit of a block of the second part; 0 where the two parts meet
  n.sink = (t.seen.sinkEnd + kKeys - 1) / kKeys;
  n.lo = t.seen.lo / kKeys + shift;
  if (n.lo < n.sink) n.lo = n.sink;
  n.hi = (t.seen.hi + kKeys - 1) / kKeys + shift;
  if (t.seen.hi == 0) n.sink = n.lo = n.hi = 0;
  const int before = t.first + 1;                     // keys that lie before every row's own place or on it
  n.wholeSink = (p.sinks < before ? p.sinks : before) / kKeys;
  n.wholeHi = before / kKeys + shift;
  n.wholeLo = (t.last - p.window >= 0 ? (t.last - p.window) / kKeys + 1 : 0) + shift;
  return n;
}

// The same value in every lane, known as such to the compiler.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ Units uniform(const Units& n) { return Units{uniform(n.sink), uniform(n.lo), uniform(n.hi), uniform(n.wholeSink), uniform(n.wholeLo), uniform(n.wholeHi)}; }
__device__ __forceinline__ bool electOne() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}

// What a CTA does, worked out by one thread and read from shared memory where it is needed: kept in registers it would displace scores.
struct Plan {
  Units units[2];              // of the two tiles
  Blocks bl;
  Seen seen;                   // by the rows of both
  int begin, end;              // units of this CTA's part of the keys
  int seq, tile;               // sequence (-1: nothing to do) and pair of tiles
  int pair, split, splits;     // (pair of tiles, key head), which part of its keys of how many
  int ctas;                    // of each pair of the call
  int n, len;                  // of the sequence
  int row0, rows, qBegin;      // rows (token, query head) of the sequence: the host keeps tokens x query heads below 2^31
};

// Barriers by their shared-memory address (a generic pointer costs two registers and a conversion at every use).
__device__ __forceinline__ bool waitAt(uint32_t bar, uint32_t parity, uint32_t abortAt) {
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
    if ((i & 255) == 255) {
      uint32_t gone;
      asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(gone) : "r"(abortAt) : "memory");
      if (gone) return false;
    }
  }
  asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(abortAt), "r"(1) : "memory");
  return false;
}
__device__ __forceinline__ void arriveAt(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void commitAt(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ int tilesOf(const PagedArgs& p, const Sequence& s, int doneRows) {
  const int rows = s.n * p.group;
  return rows <= doneRows ? 0 : (rows + kCtaRows - 1) / kCtaRows;
}

__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
// 2^x of two numbers without the special-function unit, which computes 16 a cycle and SM and would be what a block waits for: x = n + r with
// n the nearest whole number and |r| <= 1/2, 2^r by a polynomial (the least maximal relative error of its degree: 2^-13.7 for bf16, whose
// weights are rounded to 2^-9 right after, 2^-18.5 for f16), 2^n by its exponent bits.  Below -126 the result is 2^-126, NaN stays NaN.
constexpr int kPolyOf4 = 1;               // of 4 pairs, in blocks that every row sees whole
template <typename T> __device__ __forceinline__ void exp2Poly2(float& x0, float& x1) {
  constexpr float kRound = 12582912.f + 127.f;        // 1.5 x 2^23: the sum's last bits are n + 127
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x0) : "f"(-126.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x1) : "f"(-126.f));
  float t0 = x0, t1 = x1;
  add2(t0, t1, kRound, kRound);
  float n0 = t0, n1 = t1;
  add2(n0, n1, -kRound, -kRound);
  fma2(n0, n1, -1.f, -1.f, x0, x1);                   // r = x - n
  float p0, p1;
  if constexpr (std::is_same<T, __half>::value) {
    p0 = p1 = 0.009570102207362652f;
    horner2(p0, p1, n0, n1, 0.05591785907745361f);
    horner2(p0, p1, n0, n1, 0.240247443318367f);
    horner2(p0, p1, n0, n1, 0.6931217908859253f);
    horner2(p0, p1, n0, n1, 0.9999992847442627f);
  } else {
    p0 = p1 = 0.0551716685295105f;
    horner2(p0, p1, n0, n1, 0.2426111251115799f);
    horner2(p0, p1, n0, n1, 0.6932609677314758f);
    horner2(p0, p1, n0, n1, 0.9999280571937561f);
  }
  x0 = p0 * __uint_as_float(__float_as_uint(t0) << 23);
  x1 = p1 * __uint_as_float(__float_as_uint(t1) << 23);
}

// Barriers of the two warps that share 32 rows; the first also tells whether any of the 64 threads said yes.
__device__ __forceinline__ void pairBarrier(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool barrierOr(int id, bool yes) {
  int any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.s32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"(id), "r"((int)yes) : "memory");
  return any != 0;
}
__device__ __forceinline__ void storeShared(uint32_t at, float x) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(x) : "memory"); }
__device__ __forceinline__ float loadShared(uint32_t at) { float x; asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory"); return x; }
__device__ __forceinline__ uint32_t bitsBelow(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// A lane's elements of a row of D: kEach neighbours.
template <int D> struct LaneOf { static constexpr int kEach = D / 32; using Pack = typename std::conditional<D == 128, uint2, uint32_t>::type; };
template <typename T> __device__ __forceinline__ float2 twoFloats(uint32_t x);
template <> __device__ __forceinline__ float2 twoFloats<__nv_bfloat16>(uint32_t x) { return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 twoFloats<__half>(uint32_t x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }
template <typename T, int D> __device__ __forceinline__ void unpack(const typename LaneOf<D>::Pack& x, float* f) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) { const float2 two = twoFloats<T>(w[i]); f[2 * i] = two.x; f[2 * i + 1] = two.y; }
}
__device__ __forceinline__ bool seesKey(const PagedArgs& p, int pos, int j) { return j <= pos && (pos - j < p.window || j < p.sinks); }

// Values that are not finite, and the rows whose sums they spoil.  The products multiply every value of a block by every row's weight, the weights
// that are 0 because the row does not see the key too, and 0 x NaN is NaN.  Only blocks that some row of the tile does not see whole have such
// weights.  `Taint` holds, of each of a lane's columns, the last and the first such key (the sinks, which every later row sees, are not asked for
// the first) and the first and last key with a NaN, over the blocks [begin, end) that the tile does not see whole.
template <int D> struct Taint { int last[D / 32], first[D / 32], nan0[D / 32], nan1[D / 32]; };
template <typename T, int D> __device__ __forceinline__ void findTaint(const ChunkArgs& a, const Plan* plan, int t, int h, Taint<D>& x) {
  using L = LaneOf<D>;
  const PagedArgs& p = a.p;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int e = 0; e < L::kEach; ++e) { x.last[e] = x.nan0[e] = x.nan1[e] = -1; x.first[e] = 0x7fffffff; }
  const Units n = plan->units[t];
  const Seen seen = plan->seen;
  for (int u = plan->begin; u < plan->end; ++u) {
    if (!(u < n.sink || (u >= n.lo && u < n.hi)) || u < n.wholeSink || (u >= n.wholeLo && u < n.wholeHi)) continue;
    const int j0 = keyOf(plan->bl, u, kKeys);
#pragma unroll 8
    for (int j = j0; j < j0 + kKeys; ++j) {
      if (!(j < seen.sinkEnd || (j >= seen.lo && j < seen.hi))) continue;      // zeroed before the products
      const long long page = pageOf(p, plan->seq, j >> a.pageShift);
      if (page < 0) continue;
      const T* v = reinterpret_cast<const T*>(p.v) + page * p.vcSp + (j & ((1 << a.pageShift) - 1)) * p.vcSn + h * p.vcSh;
      float f[L::kEach];
      unpack<T, D>(reinterpret_cast<const typename L::Pack*>(v)[lane], f);
#pragma unroll
      for (int e = 0; e < L::kEach; ++e) {
        if (fabsf(f[e]) <= 3.402823466e38f) continue;
        x.last[e] = j;                                // u and j only grow
        if (j >= p.sinks && j < x.first[e]) x.first[e] = j;
        if (f[e] != f[e]) { if (x.nan0[e] < 0) x.nan0[e] = j; x.nan1[e] = j; }
      }
    }
  }
}
// Whether the sum of a row at `pos` may be spoilt: in some column a key that it does not see is not finite, and no NaN that it sees makes the column
// NaN in any case.
template <int D> __device__ __forceinline__ bool spoils(const PagedArgs& p, const Taint<D>& x, int pos) {
  bool any = false;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
    any = any || ((x.last[e] > pos || x.first[e] <= pos - p.window) && !(x.nan0[e] >= 0 && (seesKey(p, pos, x.nan0[e]) || seesKey(p, pos, x.nan1[e]))));
  return __any_sync(0xffffffffu, any);
}

// Sums the rows of `redo` again that may be spoilt, by multiply-adds over the keys that they see: the two warps that share 32 rows call it with their
// `side` and take every other such row, four rows and four keys at a time, lane l the kEach elements l of a row.  What lane i knows of row i: its place,
// its query's offset, what its weights are relative to, its factor.  The sums go to `part` of cut keys, else divided and rounded to the tile's
// outputs in shared memory.
template <typename T, int D>
__device__ __noinline__ void mendRows(const ChunkArgs& a, const Plan* plan, int t, int side, int row0, int h, unsigned redo, int pos, long long qOff, float base, float inv,
                                      uint8_t* tileQ, float* part) {
  using L = LaneOf<D>;
  using Pack = typename L::Pack;
  constexpr int kRows = 4, kBatch = 4, kEach = L::kEach;
  const PagedArgs& p = a.p;
  const int lane = threadIdx.x & 31;
  unsigned mine = 0;
  {
    Taint<D> taint;
    findTaint<T, D>(a, plan, t, h, taint);
    for (int count = 0; redo; redo &= redo - 1) {
      const int src = __ffs(redo) - 1;
      if (spoils<D>(p, taint, __shfl_sync(0xffffffffu, pos, src)) && (count++ & 1) == side) mine |= 1u << src;
    }
  }
  while (mine) {
    int src[kRows], at[kRows], low = 0x7fffffff, high = -1;
    float q[kRows][kEach], o[kRows][kEach], minus[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      src[r] = mine ? __ffs(mine) - 1 : src[r > 0 ? r - 1 : 0];   // fewer than four are left: the last one again
      mine &= mine - 1;
      at[r] = __shfl_sync(0xffffffffu, pos, src[r]);
      low = min(low, at[r]);
      high = max(high, at[r]);
      minus[r] = -__shfl_sync(0xffffffffu, base, src[r]);
      unpack<T, D>(reinterpret_cast<const Pack*>(reinterpret_cast<const T*>(p.q) + __shfl_sync(0xffffffffu, qOff, src[r]))[lane], q[r]);
#pragma unroll
      for (int e = 0; e < kEach; ++e) { q[r][e] *= a.signQ; o[r][e] = 0.f; }
    }
    for (int u = plan->begin; u < plan->end; ++u) {
      const int j0 = keyOf(plan->bl, u, kKeys);
      const bool whole = j0 + kKeys - 1 <= low && (j0 > high - p.window || j0 + kKeys <= p.sinks);   // every row sees all keys
      for (int j = j0; j < j0 + kKeys; j += kBatch) {
        int page[kBatch];
        Pack k[kBatch], v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) page[i] = j + i <= high ? (int)pageOf(p, plan->seq, (j + i) >> a.pageShift) : -1;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {              // without branches, so that all are under way: what has no page, from page 0
          const long long from = page[i] < 0 ? 0 : page[i], slot = (j + i) & ((1 << a.pageShift) - 1);
          k[i] = reinterpret_cast<const Pack*>(reinterpret_cast<const T*>(p.k) + from * p.kcSp + slot * p.kcSn + h * p.kcSh)[lane];
          v[i] = reinterpret_cast<const Pack*>(reinterpret_cast<const T*>(p.v) + from * p.vcSp + slot * p.vcSn + h * p.vcSh)[lane];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          float x[kEach], y[kEach], w[kRows];
          unpack<T, D>(k[i], x);
          unpack<T, D>(v[i], y);
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            w[r] = 0.f;
#pragma unroll
            for (int e = 0; e < kEach; ++e) w[r] = fmaf(x[e], q[r][e], w[r]);
          }
#pragma unroll
          for (int r = 0; r < kRows; ++r) w[r] = exp2Fast(fmaf(warpSum(w[r]), a.scaleAbs, minus[r]));
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            if (page[i] < 0 || !(whole || seesKey(p, at[r], j + i))) continue;
#pragma unroll
            for (int e = 0; e < kEach; ++e) o[r][e] = fmaf(w[r], y[e], o[r][e]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float f = __shfl_sync(0xffffffffu, inv, src[r]);
      const int row = row0 + src[r];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int e = lane * kEach + i;
        if (part) part[((long long)(e / 4) * kTileRows + row) * 4 + (e & 3)] = o[r][i];
        else {
          T* dst = reinterpret_cast<T*>(tileQ + (e >> 6) * Config<D>::kAtom + row * 128 + ((((e >> 3) & 7) ^ (row & 7)) << 4)) + (e & 7);
          if constexpr (std::is_same<T, __half>::value) *dst = __float2half_rn(o[r][i] * f);
          else *dst = __float2bfloat16_rn(o[r][i] * f);
        }
      }
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV, const __grid_constant__ ChunkArgs a) {
  using C = Config<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;                                 // [2] tiles; the outputs pass through here at the end
  uint8_t* ring = smem + 2 * C::kTile;
  uint8_t* misc = ring + C::kSlots * C::kTile;
  uint64_t* kvFull = reinterpret_cast<uint64_t*>(misc);
  uint64_t* kvEmpty = kvFull + C::kSlots;
  uint64_t* sFull = kvEmpty + C::kSlots;              // [2] scores of a tile complete, and every product issued before them
  uint64_t* pReady = sFull + 2;                       // [2] weights of a tile written, its sums rescaled
  uint64_t* oFull = pReady + 2;                       // [2] all products of a tile complete
  uint64_t* qReady = oFull + 2;                       // both tiles of Q written
  uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(misc + 256);
  volatile int* abortWord = reinterpret_cast<volatile int*>(misc + 260);
  int* sScan = reinterpret_cast<int*>(misc + 272);               // [20]
  Plan* plan = reinterpret_cast<Plan*>(misc + 512);
  float* sRow = reinterpret_cast<float*>(misc + 1024);           // [2 tiles][2 halves][128]
  const PagedArgs& p = a.p;
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (smemAddr(smem) & 1023) {                        // the swizzled tiles need it; no static shared memory lies before them
    if (threadIdx.x == 0) {
      atomicExch(&g_pagedChunkStatus, 10);
      if (a.maxCut && blockIdx.x == 0) a.records[0] = make_int4(0, 1, 0, 0);
    }
    return;
  }

  asm volatile("griddepcontrol.launch_dependents;");
  // Which sequence and tiles.  The pairs of tiles, heads of one pair side by side, are taken from the last, which sees the most keys of its
  // sequence.  Where they leave SMs idle (known here, from the lengths), each has several CTAs and is cut into as many parts of its keys, if they
  // have kCutBlocks blocks each: a table's width says nothing of a sequence's length.  The other CTAs of a short pair leave.
  int h;
  {
    // a thread keeps its (last) sequence: with up to kThreads of them nothing is read twice
    const int per = (p.batch + kThreads - 1) / kThreads, first = threadIdx.x * per;
    int mine = 0;
    Sequence s{};
    for (int i = first; i < first + per && i < p.batch; ++i) { s = sequenceOf(p, i); mine += tilesOf(p, s, a.doneRows); }
    int run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += x; }
    if (lane == 31) sScan[warp] = run;
    if (warp == kLoaderWarp) {                        // not the warp that will work out the plan of a lone sequence
      if (lane == 0) { plan->seq = -1; *abortWord = 0; prefetchTensorMap(&mapK); prefetchTensorMap(&mapV); }
      const int per = 2 * C::kSlots;                  // then sFull, pReady, oFull of two tiles, qReady
      if (lane < per + 7) mbarInit(&kvFull[lane], lane == per + 2 || lane == per + 3 ? kSoftmaxWarps / 2 : lane == per + 6 ? kSoftmaxWarps : 1);
      fenceBarrierInit();
    }
    static_assert(2 * C::kSlots + 7 <= 32, "a lane a barrier");
    __syncthreads();
    int before = run - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) { const int x = sScan[w]; if (w < warp) before += x; all += x; }
    const long long pairs = (long long)all * p.kvHeads;
    int ctas = 1;
    if (pairs > 0 && 2 * pairs <= a.maxCut) ctas = min((2 * a.maxCut / 3 + (int)pairs / 2) / (int)pairs, a.maxSplits);   // nearest to the SMs
    if (a.maxCut && blockIdx.x == 0 && threadIdx.x == 0) a.records[0] = make_int4((int)min(pairs, 0x7fffffffLL), ctas, 0, 0);
    const int pair = blockIdx.x / (unsigned)ctas, split = blockIdx.x - pair * ctas, tile = pair / p.kvHeads;
    h = pair - tile * p.kvHeads;
    const int want = all - 1 - tile;
    if (want >= before && want < before + mine) {
      int i = first;
      if (per > 1) {
        for (; i < first + per; ++i) {
          s = sequenceOf(p, i);
          const int c = tilesOf(p, s, a.doneRows);
          if (want < before + c) break;
          before += c;
        }
      }
      const int rows = s.n * p.group, row0 = (want - before) * kCtaRows;
      const Tile tile0 = tileOf(p, s, row0, rows), tile1 = tileOf(p, s, row0 + kTileRows, rows);
      plan->seen = seenBy(p, tile0.first, tile1.last >= 0 ? tile1.last : tile0.last);
      const Blocks bl = blocksOf(plan->seen, kKeys);
      const int splits = max(1, min(ctas, bl.count / kCutBlocks));
      plan->units[0] = unitsOf(p, tile0, bl);
      plan->units[1] = unitsOf(p, tile1, bl);
      plan->bl = bl;
      // at most 2^24 blocks and kMaxSplits parts; the last, whose blocks have masks, is never the longest
      plan->begin = (bl.count * split + splits - 1) / splits;
      plan->end = (bl.count * (split + 1) + splits - 1) / splits;
      plan->seq = split < splits ? i : -1; plan->tile = want - before; plan->n = s.n; plan->len = s.len;
      plan->row0 = row0; plan->rows = rows; plan->qBegin = (int)s.begin;
      plan->pair = pair; plan->split = split; plan->splits = splits; plan->ctas = ctas;
      if (ctas > 1 && split == 0) a.records[1 + pair] = make_int4(i, want - before, splits, 0);
    }
    if (warp == kIssuerWarp) tmemAlloc(tmemSlot, 512);
    tcFenceBefore();
    __syncthreads();
    tcFenceAfter();
  }
  if (plan->seq < 0) {                                // fewer tiles, or parts of this one's keys, than the grid has room for
    if (warp == kIssuerWarp) tmemDealloc(*tmemSlot, 512);
    return;
  }
  const uint32_t tmem = *tmemSlot;

  // Registers: 96 a thread at launch, 640 threads; 104 for the 512 softmax threads and 64 for the other 128 make the same sum.
  if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == kLoaderWarp) {
      // ---------------------------------------------------------------- loader: items K, V, K, V, ...
      const int boxes = kKeys / a.boxRows, loads = boxes * (D / 64), box = lane % boxes, half = lane / boxes;
      bool ok = true;
      uint32_t item = 0;
      const int b = plan->seq, begin = plan->begin, end = plan->end;
      const Blocks bl = plan->bl;
      const Seen seen = plan->seen;
      auto lookUp = [&](int u) -> long long {
        const int j = keyOf(bl, u, kKeys) + box * a.boxRows;
        // a box that no row sees any key of is not looked up: it reads as zeros, as does one with a bad page number
        if (lane >= loads || !(j < seen.sinkEnd || (j < seen.hi && j + a.boxRows > seen.lo))) return -1;
        const long long page = pageOf(p, b, j >> a.pageShift);
        if (page < 0 && half == 0 && p.badPages) atomicAdd(p.badPages, 1);
        return page;
      };
      long long next = begin < end ? lookUp(begin) : -1;
      for (int u = begin; u < end && ok; ++u) {
        const long long page = next;
        if (u + 1 < end) next = lookUp(u + 1);
        const int slotIn = (int)((keyOf(bl, u, kKeys) + box * a.boxRows) & ((1 << a.pageShift) - 1));
        for (int kv = 0; kv < 2 && ok; ++kv, ++item) {
          const int st = item % C::kSlots;
          if (item >= C::kSlots) ok = __all_sync(0xffffffffu, mbarWait(&kvEmpty[st], (item / C::kSlots - 1) & 1u, abortWord));
          if (!ok) break;
          if (lane == 0) mbarExpectTx(&kvFull[st], C::kTile);
          __syncwarp();
          if (lane < loads)
            tmaLoad4d(ring + st * C::kTile + half * C::kAtom + box * a.boxRows * 128, kv ? &mapV : &mapK, &kvFull[st], half * 64, slotIn, h,
                      page < 0 ? (int)p.numPages : (int)page);
        }
      }
      if (!ok) {
        if (lane == 0) atomicExch(&g_pagedChunkStatus, 10);
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);   // copies in flight land before the CTA gives its memory back
      }
    } else if (warp == kIssuerWarp) {
      // ---------------------------------------------------------------- issuer
      // The whole warp walks the loop, one elected thread issues: what the products are given then stays in uniform registers (a loop
      // run by one thread alone moved every descriptor there anew, 90 cycles a product of 64).  Descriptors are built once, a slot only
      // adds its offset, and the loop has no division.
      constexpr int fmt = std::is_same<T, __half>::value ? 0 : 1;
      constexpr uint32_t idescS = instrDesc(fmt, kTileRows, kKeys, 0, 0), idescO = instrDesc(fmt, kTileRows, D, 0, 1);
      const Units n0 = uniform(plan->units[0]), n1 = uniform(plan->units[1]);
      const int begin = uniform(plan->begin), end = uniform(plan->end);
      const uint32_t tm = uniform((int)tmem);
      const bool leader = electOne();
      const uint64_t descQ = smemDescKMajorSw128(smemAddr(sQ)), descK = smemDescKMajorSw128(smemAddr(ring)), descV = smemDescMnMajorSw128(smemAddr(ring), C::kAtom);
      const uint32_t full = smemAddr(kvFull), empty = smemAddr(kvEmpty), sf = smemAddr(sFull), pr = smemAddr(pReady), gone = smemAddr((const void*)abortWord);
      constexpr uint32_t kAtom16 = C::kAtom >> 4, kTile16 = C::kTile >> 4;
      bool ok = waitAt(smemAddr(qReady), 0, gone);
      auto active = [&](const Units& n, int u) { return u < n.sink || (u >= n.lo && u < n.hi); };
      auto issueS = [&](int t, uint32_t slot) {
        const uint64_t q = descQ + t * kTile16, k = descK + slot * kTile16;
        if (!leader) return;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          mmaSS<false>(tm + kColS + t * kKeys, q + (ks / 4) * kAtom16 + 2 * (ks % 4), k + (ks / 4) * kAtom16 + 2 * (ks % 4), idescS, ks > 0 ? 1u : 0u);
        commitAt(sf + 8 * t);
      };
      auto issueO = [&](int t, uint32_t slot, bool more) {
        const uint64_t v = descV + slot * kTile16;
        if (!leader) return;
#pragma unroll
        for (int ks = 0; ks < kKeys / 16; ++ks) mmaTS(tm + kColO + t * D, tm + kColS + t * kKeys + 8 * ks, v + ks * (16 * 128 >> 4), idescO, ks > 0 || more ? 1u : 0u);
      };
      uint32_t slot = 0, phase = 0;                   // the next item's slot, and the parity of its load
      auto step = [&]() { if (++slot == C::kSlots) { slot = 0; phase ^= 1u; } };
      uint32_t ph0 = 0, ph1 = 0;                      // parities of the tiles' weights
      bool more0 = false, more1 = false;              // a tile's sums have been started
      if (begin < end) {
        ok = ok && waitAt(full, 0, gone);
        tcFenceAfter();
        if (active(n0, begin)) issueS(0, 0);
        if (active(n1, begin)) issueS(1, 0);
        if (leader) commitAt(empty);
        step();
      }
      for (int u = begin; u < end; ++u) {
        const uint32_t vSlot = slot;
        ok = ok && waitAt(full + 8 * slot, phase, gone);
        step();
        const uint32_t kSlot = slot, kPhase = phase;
        const bool next = u + 1 < end;
        bool haveK = false;
        if (active(n0, u)) {
          ok = ok && waitAt(pr, ph0, gone);
          ph0 ^= 1u;
          tcFenceAfter();
          issueO(0, vSlot, more0);
          more0 = true;
        }
        if (next && active(n0, u + 1)) {
          ok = ok && waitAt(full + 8 * kSlot, kPhase, gone);
          haveK = true;
          tcFenceAfter();
          issueS(0, kSlot);
        }
        if (active(n1, u)) {
          ok = ok && waitAt(pr + 8, ph1, gone);
          ph1 ^= 1u;
          tcFenceAfter();
          issueO(1, vSlot, more1);
          more1 = true;
        }
        if (leader) commitAt(empty + 8 * vSlot);
        if (next) {
          if (!haveK) { ok = ok && waitAt(full + 8 * kSlot, kPhase, gone); tcFenceAfter(); }   // a slot is given back only after its load has landed
          if (active(n1, u + 1)) issueS(1, kSlot);
          if (leader) commitAt(empty + 8 * kSlot);
          step();
        }
      }
      if (leader) { commitAt(smemAddr(&oFull[0])); commitAt(smemAddr(&oFull[1])); }
      if (!ok && leader) atomicExch(&g_pagedChunkStatus, 11);
    }
  } else {
    // ------------------------------------------------------------------ softmax
    const int t = warp >> 3, side = (warp >> 2) & 1, q4 = warp & 3, r = q4 * 32 + lane;   // tile, half of the columns, row
    // this thread's row: its place, and where it lies in q and out (worked out again after the loop)
    auto liveRow = [&]() { return plan->row0 + t * kTileRows + r < plan->rows; };
    auto tokenOf = [&](int& head) {
      const uint32_t row = plan->row0 + t * kTileRows + r, x = min(row, (uint32_t)plan->rows - 1u), tok = x / (uint32_t)p.group;
      head = h * p.group + (int)(x - tok * p.group);
      return (int)tok;
    };
    int head;
    const int tok = tokenOf(head), pos = clipPlace((long long)plan->len - plan->n + tok);
    uint8_t* tileQ = sQ + t * C::kTile;
    const uint32_t mineAt = smemAddr(sRow + (t * 2 + side) * kTileRows + r), otherAt = smemAddr(sRow + (t * 2 + (side ^ 1)) * kTileRows + r);
    const int bar = 1 + t * 4 + q4;                   // the two warps that share 32 rows
    constexpr int kChunks = D / 8;                    // 16-byte chunks of a row
    constexpr int kRowsAtOnce = 32 / kChunks;         // rows that a warp's 16-byte accesses cover
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const long long qOff = (long long)(plan->qBegin + tok) * p.qSt + head * p.qSh;
    const bool inQ = liveRow();
    {
    // Q, a warp 16 of its 32 rows: neighbouring lanes take neighbouring chunks of a row
    uint4 x[16 / kRowsAtOnce];
#pragma unroll
    for (int i = 0; i < 16 / kRowsAtOnce; ++i) {
      const int src = side * 16 + i * kRowsAtOnce + lane / kChunks;
      const long long off = __shfl_sync(0xffffffffu, qOff, src);
      const bool in = __shfl_sync(0xffffffffu, (int)inQ, src);
      x[i] = make_uint4(0, 0, 0, 0);
      if (in) x[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + off + lane % kChunks * 8);
    }
#pragma unroll
    for (int i = 0; i < 16 / kRowsAtOnce; ++i) {
      const int c = lane % kChunks, rr = q4 * 32 + side * 16 + i * kRowsAtOnce + lane / kChunks;
      if (a.signQ < 0.f) { x[i].x ^= 0x80008000u; x[i].y ^= 0x80008000u; x[i].z ^= 0x80008000u; x[i].w ^= 0x80008000u; }
      *reinterpret_cast<uint4*>(tileQ + (c >> 3) * C::kAtom + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = x[i];
    }
    }
    fenceProxyAsync();
    __syncwarp();
    if (lane == 0) mbarArrive(qReady);

    const uint32_t lanes = (uint32_t)(q4 * 32) << 16;
    const uint32_t colS = tmem + lanes + kColS + t * kKeys, colO = tmem + lanes + kColO + t * D + side * (D / 2);
    constexpr float kShift = weightShift<T>();
    float m = -INFINITY, l = 0.f;                     // the row's running maximum (the same in both threads), this thread's share of the sum
    uint32_t done = 0;                                // blocks of this tile so far
    bool ok = true;
    const int end = plan->end;
    const uint32_t fullAt = smemAddr(&sFull[t]), readyAt = smemAddr(&pReady[t]), gone = smemAddr((const void*)abortWord);
    for (int u = plan->begin; u < end; ++u) {
      const Units n = plan->units[t];
      if (u >= n.sink && u < n.lo) { u = n.lo - 1; continue; }
      if (u >= n.hi && u >= n.sink) break;
      if (ok && !waitAt(fullAt, done & 1u, gone)) { ok = false; atomicExch(&g_pagedChunkStatus, 12); }
      tcFenceAfter();
      const bool whole = u < n.wholeSink || (u >= n.wholeLo && u < n.wholeHi);
      uint32_t x[64], w[32];
      auto load = [&]() {
        __syncwarp();
        tmemIssue32(colS + side * 64, x);
        tmemIssue32(colS + side * 64 + 32, x + 32);
        tmemWait32(x);
        tmemWait32(x + 32);
        if (!whole) {
          // visible columns: c < hi and (c >= lo or c < sink), as bits (a branch a column costs 8 us a block)
          const int j1 = keyOf(plan->bl, u, kKeys) + side * 64, hi = pos + 1 - j1, lo = max(pos + 1 - p.window, 0) - j1, sink = p.sinks - j1;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t vis = bitsBelow(hi - 32 * c) & (~bitsBelow(lo - 32 * c) | bitsBelow(sink - 32 * c));
#pragma unroll
            for (int i = 0; i < 32; ++i) x[32 * c + i] = (vis >> i) & 1u ? x[32 * c + i] : 0xff800000u;   // -inf, whatever the score is
          }
        }
      };
      // The row's largest score of this block, from both its threads.
      auto exchange = [&](float mine) {
        storeShared(mineAt, mine);
        pairBarrier(bar);
        return fmaxf(mine, loadShared(otherAt));
      };
      if (done == 0) {                                // the first block sets the maximum before its weights are taken
        load();
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; ++i) mx[i & 3] = max3(mx[i & 3], __uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
        m = exchange(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scaleAbs);
      }
      // Weights relative to the maximum so far, and the block's own maximum beside them: no exponential waits for it.  If some row's grew by
      // more than the step, the block is taken again from tensor memory (the weights have not been stored over it yet).
      for (;;) {
        load();
        const float base = m == -INFINITY ? 0.f : m - kShift;
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, sum[4] = {0.f, 0.f, 0.f, 0.f};
        auto weights = [&](auto poly) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float y0 = __uint_as_float(x[2 * i]), y1 = __uint_as_float(x[2 * i + 1]);
            mx[i & 3] = max3(mx[i & 3], y0, y1);
            fma2(y0, y1, a.scaleAbs, a.scaleAbs, -base, -base);
            if (decltype(poly)::value && i % 4 >= 4 - kPolyOf4) exp2Poly2<T>(y0, y1);
            else { y0 = exp2Fast(y0); y1 = exp2Fast(y1); }
            add2(sum[(i & 1) * 2], sum[(i & 1) * 2 + 1], y0, y1);
            w[i] = pack2<T>(y0, y1);
          }
        };
        // two loops: with the choice inside, every pair of weights is a branch
        if (whole) weights(std::true_type{});
        else weights(std::false_type{});
        const float mine = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scaleAbs;
        // The row's two warps meet here in any case: both have taken their scores out before either stores weights over them.
        if (!barrierOr(bar, mine > m + kRescaleStep)) {
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          break;
        }
        const float top = exchange(mine);
        float keep = 1.f;
        if (top > m + kRescaleStep) { keep = exp2Fast(m - top); m = top; l *= keep; }
        if (done > 0 && __any_sync(0xffffffffu, keep != 1.f)) {
          // the scores' barrier says that all products into O are complete
#pragma unroll 1
          for (int c = 0; c < D / 2; c += 32) {
            float o[32];
            tmemLoad32x32(colO + c, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= keep;
            tmemStore32(colO + c, reinterpret_cast<uint32_t*>(o));
            tmemStoreWait();
          }
        }
      }
      __syncwarp();
      tmemStore32(colS + 32 * side, w);
      tmemStoreWait();
      if (!whole) {
        // Values of keys that no row sees may be NaN, and 0 x NaN is NaN: the tile that uses the block first zeroes them, row r key r.
        const Seen seen = plan->seen;
        const Units n0 = plan->units[0];
        const int j0 = keyOf(plan->bl, u, kKeys), j = j0 + r;
        const bool clean = j0 + kKeys <= seen.sinkEnd || (j0 + kKeys <= seen.hi && (j0 >= seen.lo || seen.sinkEnd == seen.lo));
        if (!clean && (t == 0 || !(u < n0.sink || (u >= n0.lo && u < n0.hi)))) {
          const uint32_t vItem = 2 * (u - plan->begin) + 1;
          if (ok && !waitAt(smemAddr(&kvFull[vItem % C::kSlots]), (vItem / C::kSlots) & 1u, gone)) { ok = false; atomicExch(&g_pagedChunkStatus, 12); }
          if (!(j < seen.sinkEnd || (j >= seen.lo && j < seen.hi))) {
#pragma unroll
            for (int i = 0; i < kChunks / 2; ++i) {
              const int c = side * (kChunks / 2) + ((i + r) & (kChunks / 2 - 1));   // neighbouring rows start at other banks
              *reinterpret_cast<uint4*>(ring + (vItem % C::kSlots) * C::kTile + (c >> 3) * C::kAtom + r * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
            }
          }
          fenceProxyAsync();
        }
      }
      tcFenceBefore();
      __syncwarp();
      if (lane == 0) arriveAt(readyAt);
      ++done;
    }
    // ---------------------------------------------------------------- output
    pairBarrier(bar);                                 // both have read the last maximum
    storeShared(mineAt, l);
    if (ok && !mbarWait(&oFull[t], 0, abortWord)) { ok = false; atomicExch(&g_pagedChunkStatus, 12); }
    tcFenceAfter();
    pairBarrier(bar);
    l += loadShared(otherAt);
    const float base = m == -INFINITY ? 0.f : m - kShift;
    const bool cut = plan->splits > 1;
    float* part = a.parts + (((long long)plan->pair * 2 + t) * plan->ctas + plan->split) * C::kPart;
    const float inv = 1.f / divisorOf(l, m, pos >= 0);
    bool odd = false;
    if (cut && side == 0) {
      part[kTileRows * D + r] = m;
      part[kTileRows * (D + 1) + r] = l;
    }
#pragma unroll 1
    for (int c = 0; c < D / 2; c += 32) {
      float o[32];
      __syncwarp();
      if (done) tmemLoad32x32(colO + c, o);
      else {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0.f;
      }
      float zero = 0.f;                               // stays 0 unless some element is NaN or infinite
#pragma unroll
      for (int i = 0; i < 32; ++i) zero = fmaf(o[i], 0.f, zero);
      odd = odd || zero != 0.f;
      const int col = side * (D / 2) + c;
      if (cut) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<float4*>(part + ((long long)(col / 4 + i) * kTileRows + r) * 4) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ch = col / 8 + i;
          *reinterpret_cast<uint4*>(tileQ + (ch >> 3) * C::kAtom + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) =
              make_uint4(pack2<T>(o[8 * i] * inv, o[8 * i + 1] * inv), pack2<T>(o[8 * i + 2] * inv, o[8 * i + 3] * inv), pack2<T>(o[8 * i + 4] * inv, o[8 * i + 5] * inv),
                         pack2<T>(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
        }
      }
    }
    const bool live = liveRow();
    int oHead;
    const int oTok = tokenOf(oHead);
    odd = odd && live && fabsf(l) <= 3.402823466e38f;
    if (barrierOr(bar, odd)) {
      // sums that are not finite though their weights are
      storeShared(mineAt, odd ? 1.f : 0.f);
      pairBarrier(bar);
      const unsigned redo = __ballot_sync(0xffffffffu, odd || loadShared(otherAt) != 0.f);
      mendRows<T, D>(a, plan, t, side, q4 * 32, h, redo, pos, (long long)(plan->qBegin + oTok) * p.qSt + oHead * p.qSh, base, inv, tileQ, cut ? part : nullptr);
      pairBarrier(bar);
    }
    if (!cut) {
      const long long oOff = (long long)(plan->qBegin + oTok) * p.oSt + oHead * p.oSh;
#pragma unroll
      for (int i = 0; i < 16; i += kRowsAtOnce) {
        const int src = side * 16 + i + lane / kChunks, c = lane % kChunks, rr = q4 * 32 + src;
        const long long off = __shfl_sync(0xffffffffu, oOff, src);
        const bool in = __shfl_sync(0xffffffffu, (int)live, src);
        const uint4 x = *reinterpret_cast<const uint4*>(tileQ + (c >> 3) * C::kAtom + rr * 128 + (((c & 7) ^ (rr & 7)) << 4));
        if (in) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + off + c * 8) = x;
      }
    }
  }
  tcFenceBefore();
  __syncthreads();
  if (warp == kIssuerWarp) { tcFenceAfter(); tmemDealloc(tmem, 512); }
}

// Joins the parts of a tile: block = one tile of 128 rows, thread = one row and every other vector of four elements.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_chunk_join_kernel(const ChunkArgs a) {
  using C = Config<D>;
  __shared__ float sF[kMaxSplits][kTileRows];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const PagedArgs& p = a.p;
  const int pair = blockIdx.x >> 1, t = blockIdx.x & 1, r = threadIdx.x & 127, side = threadIdx.x >> 7;
  const int4 call = a.records[0], rec = a.records[1 + pair];   // the second read before it is known to be one: the workspace holds it in any case
  const int splits = rec.z;
  if (call.y < 2 || pair >= call.x || splits < 2) return;      // no pair of the call, or not cut and written already
  const Sequence s = sequenceOf(p, rec.x);
  const long long rows = (long long)s.n * p.group, row = (long long)rec.y * kCtaRows + t * kTileRows + r;
  const float* part = a.parts + ((long long)pair * 2 + t) * call.y * C::kPart;
  float top = -INFINITY, sum = 0.f;
  for (int i = 0; i < splits; ++i) top = fmaxf(top, part[(long long)i * C::kPart + kTileRows * D + r]);
  for (int i = 0; i < splits; ++i) {
    const float m = part[(long long)i * C::kPart + kTileRows * D + r], l = part[(long long)i * C::kPart + kTileRows * (D + 1) + r];
    const float f = m == -INFINITY ? 0.f : exp2Fast(m - top);
    if (side == 0) sF[i][r] = f;
    sum += l * f;                                     // a part without a maximum weighs nothing, unless its scores are NaN: then l is
  }
  __syncthreads();
  if (row >= rows) return;
  const long long tok = row / p.group;
  const float inv = 1.f / divisorOf(sum, top, s.len - s.n + tok >= 0);
  const int head = (int)(pair % p.kvHeads) * p.group + (int)(row - tok * p.group);
  T* out = reinterpret_cast<T*>(p.out) + (s.begin + tok) * p.oSt + head * p.oSh;
  for (int c = side; c < D / 4; c += 2) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < splits; ++i) {
      const float f = sF[i][r];
      if (f != 0.f) {
        const float4 v = *reinterpret_cast<const float4*>(part + (long long)i * C::kPart + ((long long)c * kTileRows + r) * 4);
        x.x = fmaf(v.x, f, x.x); x.y = fmaf(v.y, f, x.y); x.z = fmaf(v.z, f, x.z); x.w = fmaf(v.w, f, x.w);
      }
    }
    *reinterpret_cast<uint2*>(out + 4 * c) = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
  }
}

// CTAs of the grid (a bound on the pairs of tiles times key heads from what the host knows), and whether keys may be cut: where the rows that
// the call names would fill less than three quarters of the SMs, and the table's reach or the window leaves room for two parts of
// kCutBlocks blocks (the device knows whether the sequences have them): a part costs a CTA's start and end and its sums' way through
// memory, what eight blocks cost.
struct Launch { long long ctas; int maxCut, maxSplits; };
Launch launchOf(const PagedArgs& p) {
  Launch l{};
  const long long each = (p.maxQ * p.group + kCtaRows - 1) / kCtaRows, tiles = p.tokens * p.group / kCtaRows + p.batch, sms = deviceSMs();
  l.ctas = (each * p.batch < tiles ? each * p.batch : tiles) * p.kvHeads;
  // blocks that a pair's rows see, at most: the rows of a pair belong to at most kCtaRows tokens; windows and sinks begin and end inside blocks
  long long most = ((long long)p.reach + kKeys - 1) / kKeys;
  const long long seen = ((long long)p.sinks + kKeys - 1) / kKeys + ((long long)p.window + kCtaRows + kKeys - 1) / kKeys + 1;
  if (seen < most) most = seen;
  const long long splits = most / kCutBlocks;
  l.maxSplits = (int)(splits < kMaxSplits ? splits : kMaxSplits);
  if (l.maxSplits > 1 && 4 * (p.tokens * p.group / kCtaRows) * p.kvHeads <= 3 * sms) l.maxCut = (int)(sms * 3 / 2);
  return l;
}
template <int D> long long bytesOf(const Launch& l) { return l.maxCut ? 16LL * (1 + l.maxCut) + 2LL * l.maxCut * Config<D>::kPart * 4 : 0; }

template <typename T, int D>
int launch(const PagedArgs& p, int doneRows, void* workspace, long long bytes, cudaStream_t st) {
  using C = Config<D>;
  CUtensorMap mk, mv;
  ChunkArgs a{};
  a.p = p;
  a.doneRows = doneRows;
  a.boxRows = p.pageSize < kKeys ? (int)p.pageSize : kKeys;
  while ((1LL << a.pageShift) < p.pageSize) ++a.pageShift;
  if (!makePageMap(&mk, p.k, p.dtype, p, p.kcSp, p.kcSn, p.kcSh, a.boxRows) || !makePageMap(&mv, p.v, p.dtype, p, p.vcSp, p.vcSn, p.vcSh, a.boxRows))
    return setError(LLC_ERR_CUDA, "llc cuda: cuTensorMapEncodeTiled rejected the cache");
  // a scale of 0 becomes one that no score survives: 0 times a masked score's -inf would be NaN
  a.scaleAbs = fabsf(p.scaleLog2) > 1e-37f || p.scaleLog2 != p.scaleLog2 ? fabsf(p.scaleLog2) : 1e-37f;
  a.signQ = p.scaleLog2 < 0.f ? -1.f : 1.f;
  Launch l = launchOf(p);
  if (!workspace || bytes < bytesOf<D>(l)) l.maxCut = 0;
  if (l.ctas < l.maxCut) l.ctas = l.maxCut;
  if (l.ctas > 0x7FFFFFFFLL) return setError(LLC_ERR_UNSUPPORTED, "llc argument: paged_attention too many tiles");
  a.maxCut = l.maxCut;
  a.maxSplits = l.maxSplits;
  a.records = static_cast<int4*>(workspace);
  a.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + 16LL * (1 + l.maxCut));
  static DeviceOnce configured;
  const int dev = currentDevice();
  if (!configured.test(dev)) {
    LLC_CUDA_CHECK(cudaFuncSetAttribute(paged_chunk_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    configured.set(dev);
  }
  paged_chunk_kernel<T, D><<<(unsigned)l.ctas, kThreads, C::kSmem, st>>>(mk, mv, a);
  LLC_LAUNCH_CHECK("paged_chunk_kernel");
  if (l.maxCut) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)l.maxCut);         // two tiles of each of at most maxCut / 2 pairs
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    LLC_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_chunk_join_kernel<T, D>, a));
  }
  return LLC_OK;
}

}  // namespace

// The sequences of more than doneRows rows (new tokens x query heads of a key head).
long long pagedChunkWorkspace(const PagedArgs& p) { return p.d == 64 ? bytesOf<64>(launchOf(p)) : bytesOf<128>(launchOf(p)); }
int pagedChunk(const PagedArgs& p, int doneRows, void* workspace, long long bytes, cudaStream_t st) {
  if (p.dtype == LLC_BFLOAT16)
    return p.d == 64 ? launch<__nv_bfloat16, 64>(p, doneRows, workspace, bytes, st) : launch<__nv_bfloat16, 128>(p, doneRows, workspace, bytes, st);
  return p.d == 64 ? launch<__half, 64>(p, doneRows, workspace, bytes, st) : launch<__half, 128>(p, doneRows, workspace, bytes, st);
}

int pagedChunkStatus() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_pagedChunkStatus, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_pagedChunkStatus, &zero, sizeof(int));
  return v;
}

}  // namespace llc
