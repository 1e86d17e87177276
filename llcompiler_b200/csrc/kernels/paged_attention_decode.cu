// Paged attention for sequences of few new tokens (decoding): rows = new tokens x query heads of one key head, at most 16 or
// 32 of them, so that the cache is read once for all of them.
// Mathematics: out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m), s_j = scale log2(e) q.k_j, m any number near the maximum of s; sums
// over parts of the keys with maxima m_i join as sum_i 2^(m_i - m) (...)_i.
// Bound: the cache's bytes.  16 keys and values of one head (8 KB at d = 128) have to leave memory every 340 cycles on every SM; the 32
// small matrix products that they take are a third of that, so plain mma.sync from swizzled shared memory serves (tcgen05 would
// compute 128 rows for the 4 to 16 that exist, with a longer chain from scores to values).
// Work: the blocks of 16 keys of all (sequence, key head) pairs form one line, cut into equal shares, one a WARP: ragged batches and
// single long sequences load every SM alike, and no warp waits for another.  A warp is its own producer: when a block has been
// used, its lanes start the TMA loads of the block that comes a ring's length later (boxes of 16 rows x 64 elements,
// eight warps an SM).  A pair that a share's end cuts leaves its parts' sums in the workspace, which a second kernel joins
// (launched early, it waits for this one on the device).  Few and short pairs (SPLIT false) take a CTA each instead, whose warps
// take the blocks in turn and meet in shared memory: the second launch costs more than it saves there.
// 17 to 32 rows at d = 128: two tiles of queries, scores and sums in a warp are more than 255 registers (176 bytes of a thread in memory in bf16 and f16,
// 32 at d = 64), 32 x 8192 keys for 4 tokens of 8 heads a key head 259 us with L2 flushed, floor 164.
// Before this, four warps shared blocks of 64 keys and met at the end of every pair: 10000 cycles from one pair to the next.
#include "page_map.h"
#include "paged_attention.cuh"
#include "tc_common.cuh"

namespace llc {
__device__ int g_pagedDecodeStatus = 0;   // non-zero after a bounded wait gave up: 8; 9: misplaced shared memory

namespace {
using namespace tc;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 16;                          // keys of a block
constexpr int kTail = 4;                           // floats behind a part's row of sums: its maximum, its sum of weights, two unused

template <int D, int MT> struct Config {
  static constexpr int kRows = 16 * MT;
  static constexpr int kCtas = 2;                  // of an SM
  static constexpr int kBox = kKeys * 128;         // bytes of 16 keys x 64 elements
  static constexpr int kTensor = kBox * (D / 64);  // K or V of a block
  static constexpr int kBlock = 2 * kTensor;
  // 16 KB in flight for a warp, 128 KB for an SM; with 24 KB everything an SM asks for stands in a longer line (32 x 8192 keys of 8 heads
  // of 128: 177 us, 189 with 24 KB; one sequence of 131072: 97 and 101)
  static constexpr int kStages = 16 * 1024 / kBlock;
  static constexpr int kRing = kWarps * kStages * kBlock;
  static constexpr int kMisc = 512 + 2 * kWarps * kRows * 4;   // barriers and the shares' starts, then m and l of every warp's rows
  static constexpr int kSmem = kRing + kMisc;
  static_assert(kWarps * kRows * D * 4 <= kRing, "the warps of a CTA meet where the ring was");
  static_assert(kCtas * (kSmem + 1024) <= 228 * 1024 && kWarps * kStages * 8 <= 256, "the CTAs of an SM share 228 KB");
};

struct DecodeArgs {
  PagedArgs p;
  int pageShift, minBlocks;    // page_size = 1 << pageShift; least share of a warp
  int slotRows;                // rows of a slot: the most that a sequence of this call has
  int joinRows;                // rows of a block of the joining kernel
  int2* records;               // [pairs]: first warp of the pair, number of warps that have a part of it
  float* slots;                // [2 x warps][slotRows][D + kTail]: a part's sums, see slotOf
  int warps;                   // of the grid
};
// A share's ends cut two pairs at most: the one that a warp before it has begun, and the last one that it begins itself.
constexpr int kCutsOfAShare = 2;
__device__ __forceinline__ long long slotOf(const DecodeArgs& a, int warp, bool begun) { return begun ? warp : (long long)a.warps + warp; }

// The blocks of keys of one key head of a sequence; one empty block where nothing is visible, which writes the zeros; none where the
// sequence has no rows, or more than this kernel takes.
__device__ __forceinline__ Blocks blocksOf(const PagedArgs& p, const Sequence& s, const Seen& seen, int maxRows) {
  if (s.n == 0 || (long long)s.n * p.group > maxRows) return Blocks{0, 0, 0};
  Blocks b = blocksOf(seen, kKeys);
  if (b.count < 1) b.count = 1;
  return b;
}
__device__ __forceinline__ int countOf(const PagedArgs& p, int b, int maxRows) {
  const Sequence s = sequenceOf(p, b);
  return blocksOf(p, s, seenBy(p, clipPlace((long long)s.len - s.n), s.len - 1), maxRows).count;
}

// A warp's way along its share: the segments (pair, blocks unit .. end - 1), in order.
struct Walk {
  int b, h, unit, end;
  long long left;              // blocks of the share behind this segment
  Sequence s;
  Seen seen;
  Blocks bl;
  // The segment that begins at (b, h, unit); false where the share is used up.  Called again only with b or left changed.
  __device__ __forceinline__ bool open(const PagedArgs& p, int maxRows) {
    while (left > 0) {
      s = sequenceOf(p, b);
      seen = seenBy(p, clipPlace((long long)s.len - s.n), s.len - 1);
      bl = blocksOf(p, s, seen, maxRows);
      if (bl.count == 0) { ++b; h = 0; continue; }
      end = bl.count - unit < left ? bl.count : unit + (int)left;
      left -= end - unit;
      return true;
    }
    return false;
  }
  // The next pair's first block.
  __device__ __forceinline__ bool next(const PagedArgs& p, int maxRows) {
    unit = 0;
    if (++h == p.kvHeads) { h = 0; ++b; }
    else if (left > 0) {                           // the same sequence: what is known of it holds
      end = bl.count < left ? bl.count : (int)left;
      left -= end;
      return true;
    }
    return open(p, maxRows);
  }
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T> __device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int D, int MT, bool SPLIT>
__global__ void __launch_bounds__(kThreads, Config<D, MT>::kCtas)
paged_decode_kernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV, const __grid_constant__ DecodeArgs a) {
  using C = Config<D, MT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* misc = smem + C::kRing;
  const PagedArgs& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(misc) + warp * C::kStages;   // one a stage of this warp
  volatile int* abortWord = reinterpret_cast<volatile int*>(misc + 256);
  long long* sScan = reinterpret_cast<long long*>(misc + 264);      // [4] sums of the warps' sequences
  int* sSeq = reinterpret_cast<int*>(misc + 296);                   // [4] the sequence that a warp's share begins in, -1: no share
  long long* sStart = reinterpret_cast<long long*>(misc + 312);     // [4] its first block there, counted over all key heads
  float* sM = reinterpret_cast<float*>(misc + 512);                 // [4][kRows]
  float* sL = sM + kWarps * C::kRows;
  if (smemAddr(smem) & 1023) {                     // the swizzled boxes need it; no static shared memory lies before them
    if (threadIdx.x == 0) atomicExch(&g_pagedDecodeStatus, 9);
    if (SPLIT) for (int i = threadIdx.x; i < p.batch * p.kvHeads; i += kThreads) a.records[i] = make_int2(0, 0);
    return;
  }
  if (threadIdx.x == 0) { prefetchTensorMap(&mapK); prefetchTensorMap(&mapV); *abortWord = 0; }
  if (lane == 0) {
    for (int i = 0; i < C::kStages; ++i) mbarInit(&full[i], 1);
    fenceBarrierInit();
  }
  asm volatile("griddepcontrol.launch_dependents;");

  Walk use;                                        // what is being computed
  constexpr int step = SPLIT ? 1 : kWarps;
  const long long me = (long long)blockIdx.x * kWarps + warp;
  long long share = 0;
  bool more;
  if (!SPLIT) {
    __syncthreads();
    use.b = blockIdx.x / p.kvHeads;
    use.h = blockIdx.x - use.b * p.kvHeads;
    use.unit = 0;
    use.left = countOf(p, use.b, C::kRows);
    if (use.left == 0) return;
    more = use.open(p, C::kRows);
    use.unit = warp;
  } else {
    const int per = (p.batch + kThreads - 1) / kThreads, first = threadIdx.x * per;
    long long mine = 0;
    for (int i = first; i < first + per && i < p.batch; ++i) mine += countOf(p, i, C::kRows);
    long long run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const long long x = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += x; }
    if (lane == 31) sScan[warp] = run;
    if (lane == 0) sSeq[warp] = -1;
    __syncthreads();
    long long before = run - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) { if (w < warp) before += sScan[w]; all += sScan[w]; }
    before *= p.kvHeads; mine *= p.kvHeads; all *= p.kvHeads;
    const long long workers = (long long)gridDim.x * kWarps;
    share = (all + workers - 1) / workers;
    if (share < a.minBlocks) share = a.minBlocks;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const long long start = ((long long)blockIdx.x * kWarps + w) * share;
      if (start < before || start >= before + mine) continue;
      long long at = before;
      int i = first;
      if (per > 1) {
        for (; i < first + per; ++i) {
          const long long c = (long long)countOf(p, i, C::kRows) * p.kvHeads;
          if (start < at + c) break;
          at += c;
        }
      }
      sSeq[w] = i;
      sStart[w] = start - at;
    }
    __syncthreads();
    use.b = sSeq[warp];
    if (use.b < 0) return;                         // more warps than shares
    use.left = all - me * share < share ? all - me * share : share;
    const int c = countOf(p, use.b, C::kRows);
    use.h = (int)(sStart[warp] / c);
    use.unit = (int)(sStart[warp] - (long long)use.h * c);
    more = use.open(p, C::kRows);
  }

  // ---- loads: a second walk, a ring's length ahead
  Walk load = use;
  bool loading = more && load.unit < load.end;
  int pages = 0, k = 32;                           // lane i: the page of the i-th block from here on; the next one's i
  uint32_t loaded = 0;
  uint8_t* ring = smem + warp * C::kStages * C::kBlock;
  auto issue = [&]() {
    if (!loading) return;
    if (k == 32) {
      const int u = load.unit + lane * step, j = keyOf(load.bl, u, kKeys);
      // a block that no token sees any key of is not looked up: it reads as zeros, as does one with a bad page number
      long long page = -1;
      if (u < load.end && (j < load.seen.sinkEnd || (j < load.seen.hi && j + kKeys > load.seen.lo))) {
        page = pageOf(p, load.b, j >> a.pageShift);
        if (page < 0 && p.badPages) atomicAdd(p.badPages, 1);
      }
      pages = page < 0 ? (int)p.numPages : (int)page;
      k = 0;
    }
    const int page = __shfl_sync(0xffffffffu, pages, k), st = loaded % C::kStages;
    if (lane == 0) mbarExpectTx(&full[st], C::kBlock);
    __syncwarp();
    constexpr int kLoads = 2 * (D / 64);
    if (lane < kLoads) {
      const int which = lane / (D / 64), half = lane % (D / 64);
      tmaLoad4d(ring + st * C::kBlock + lane * C::kBox, which ? &mapV : &mapK, &full[st], half * 64, keyOf(load.bl, load.unit, kKeys) & ((1 << a.pageShift) - 1), load.h, page);
    }
    ++loaded;
    ++k;
    load.unit += step;
    if (load.unit >= load.end) { loading = SPLIT && load.next(p, C::kRows); k = 32; }
  };
  const uint32_t ringAddr = smemAddr(ring);
  const int g4 = lane >> 2, c4 = lane & 3;         // a thread's row (and row + 8) of a tile, its pair of columns
  // K: matrices (keys 0-7, d 0-7), (keys 0-7, d 8-15), (keys 8-15, d 0-7), (keys 8-15, d 8-15) of a 16 x 16 step
  const int kRow = (lane & 7) + ((lane >> 4) << 3), kChunk = (lane >> 3) & 1;
  // V, transposed on the way: (keys 0-7, d 0-7), (keys 8-15, d 0-7), (keys 0-7, d 8-15), (keys 8-15, d 8-15)
  const int vRow = lane & 15, vChunk = lane >> 4;
  const uint32_t kBase = ringAddr + kRow * 128, vBase = ringAddr + C::kTensor + vRow * 128;
  constexpr float kShift = weightShift<T>();
  uint32_t used = 0;
  bool ok = true;
  for (; more; more = SPLIT && use.next(p, C::kRows)) {
    const Sequence& s = use.s;
    const Seen& seen = use.seen;
    const int begin = use.unit, rows = s.n * p.group;
    const T* q = reinterpret_cast<const T*>(p.q);
    uint32_t qf[MT][D / 16][4];
    int pos[MT][2];                                // places of this thread's rows
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = mt * 16 + r * 8 + g4;
        const int tok = row / p.group;
        pos[mt][r] = clipPlace((long long)s.len - s.n + tok);
        const T* src = q + (s.begin + tok) * p.qSt + (use.h * p.group + row - tok * p.group) * p.qSh + c4 * 2;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          qf[mt][ks][r] = row < rows ? *reinterpret_cast<const uint32_t*>(src + ks * 16) : 0u;
          qf[mt][ks][2 + r] = row < rows ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8) : 0u;
        }
      }
    // The first loads start behind the queries': what an SM asks for comes in about the order of asking.
    if (loaded == 0)
#pragma unroll 1
      for (int i = 0; i < C::kStages; ++i) issue();
    float o[MT][D / 8][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) { o[mt][i][0] = o[mt][i][1] = o[mt][i][2] = o[mt][i][3] = 0.f; }
      m[mt][0] = m[mt][1] = -INFINITY;
      l[mt][0] = l[mt][1] = 0.f;
    }
#pragma unroll 1
    for (; use.unit < use.end; use.unit += step, ++used) {
      const int st = used % C::kStages;
      const int j0 = keyOf(use.bl, use.unit, kKeys);
      if (ok && !mbarWait(&full[st], (used / C::kStages) & 1u, abortWord)) { ok = false; atomicExch(&g_pagedDecodeStatus, 8); }
      __syncwarp();
      const uint32_t kAddr = kBase + st * C::kBlock, vAddr = vBase + st * C::kBlock;
      float sc[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[mt][0][i] = sc[mt][1][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t bf[4];
        ldmatrix4(kAddr + (ks / 4) * C::kBox + ((((ks % 4) * 2 + kChunk) ^ (kRow & 7)) << 4), bf);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) { mma16816<T>(sc[mt][0], qf[mt][ks], bf[0], bf[1]); mma16816<T>(sc[mt][1], qf[mt][ks], bf[2], bf[3]); }
      }
      // every row sees all 16 keys: they lie before the first token, and inside the last one's window or among the sinks
      const bool whole = j0 + kKeys - 1 <= s.len - s.n && (j0 > s.len - 1 - p.window || j0 + kKeys <= p.sinks);
      uint32_t vMask[2] = {0xffffffffu, 0xffffffffu}, hidden = 0;   // bits of the scores that are not seen: mt, row, column
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {              // columns c4 * 2 + {0, 1} and 8 more
          const int j = j0 + c4 * 2 + (i & 1) + (i >> 1) * 8;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const bool sees = j <= pos[mt][r] && (pos[mt][r] - j < p.window || j < p.sinks);
              if (!sees) hidden |= 1u << (mt * 8 + r * 4 + i);
            }
          // a value that nobody sees may be NaN, and 0 x NaN is NaN: it is taken as 0
          if (!(j < seen.hi && (j >= seen.lo || j < seen.sinkEnd))) vMask[i >> 1] &= (i & 1) ? 0x0000ffffu : 0xffff0000u;
        }
      }
      uint32_t pf[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float keep[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float x0 = sc[mt][0][2 * r] * p.scaleLog2, x1 = sc[mt][0][2 * r + 1] * p.scaleLog2, x2 = sc[mt][1][2 * r] * p.scaleLog2, x3 = sc[mt][1][2 * r + 1] * p.scaleLog2;
          if (!whole) {                            // after the scale, and whatever the score is: NaN where the slot holds NaN
            const uint32_t hide = hidden >> (mt * 8 + r * 4);
            if (hide & 1u) x0 = -INFINITY;
            if (hide & 2u) x1 = -INFINITY;
            if (hide & 4u) x2 = -INFINITY;
            if (hide & 8u) x3 = -INFINITY;
          }
          float mx = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          keep[r] = 1.f;
          if (mx > m[mt][r] + kRescaleStep) { keep[r] = exp2Fast(m[mt][r] - mx); m[mt][r] = mx; }
          const float base = m[mt][r] == -INFINITY ? 0.f : m[mt][r] - kShift;
          x0 = exp2Fast(x0 - base); x1 = exp2Fast(x1 - base); x2 = exp2Fast(x2 - base); x3 = exp2Fast(x3 - base);
          l[mt][r] = l[mt][r] * keep[r] + ((x0 + x1) + (x2 + x3));
          pf[mt][r] = pack2<T>(x0, x1);
          pf[mt][2 + r] = pack2<T>(x2, x3);
        }
        if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i) { o[mt][i][0] *= keep[0]; o[mt][i][1] *= keep[0]; o[mt][i][2] *= keep[1]; o[mt][i][3] *= keep[1]; }
        }
      }
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        uint32_t bf[4];
        ldmatrix4t(vAddr + (c / 4) * C::kBox + ((((c % 4) * 2 + vChunk) ^ (vRow & 7)) << 4), bf);
        bf[0] &= vMask[0]; bf[1] &= vMask[1]; bf[2] &= vMask[0]; bf[3] &= vMask[1];
        if (!whole && s.n > 1 && __any_sync(0xffffffffu, notFinite<T>(bf[0]) || notFinite<T>(bf[1]) || notFinite<T>(bf[2]) || notFinite<T>(bf[3]))) {
          // a value that some tokens see and others do not is NaN or infinite: token by token, its rows take the product
          // with the values that it sees
          for (int tok = 0; tok < s.n; ++tok) {
            const int at = clipPlace((long long)s.len - s.n + tok);
            uint32_t tm[2] = {0u, 0u};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = j0 + c4 * 2 + (i & 1) + (i >> 1) * 8;
              if (j <= at && (at - j < p.window || j < p.sinks)) tm[i >> 1] |= (i & 1) ? 0xffff0000u : 0x0000ffffu;
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int nt = 0; nt < 2; ++nt) {
                float t[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816<T>(t, pf[mt], bf[2 * nt] & tm[0], bf[2 * nt + 1] & tm[1]);
#pragma unroll
                for (int r = 0; r < 2; ++r)
                  if (pos[mt][r] == at) { o[mt][2 * c + nt][2 * r] += t[2 * r]; o[mt][2 * c + nt][2 * r + 1] += t[2 * r + 1]; }
              }
          }
          continue;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) { mma16816<T>(o[mt][2 * c], pf[mt], bf[0], bf[1]); mma16816<T>(o[mt][2 * c + 1], pf[mt], bf[2], bf[3]); }
      }
      __syncwarp();                                // every lane is done with the block: its slot takes the one a ring's length on
      issue();
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[mt][r] += __shfl_xor_sync(0xffffffffu, l[mt][r], 1);
        l[mt][r] += __shfl_xor_sync(0xffffffffu, l[mt][r], 2);
      }
    if (SPLIT) {
      const bool whole = begin == 0 && use.end == use.bl.count;
      const long long pair = (long long)use.b * p.kvHeads + use.h;
      if (begin == 0 && lane == 0) a.records[pair] = make_int2((int)me, 1 + (int)((use.bl.count - use.end + share - 1) / share));
      float* slot = a.slots + slotOf(a, (int)me, begin != 0) * a.slotRows * (D + kTail);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = mt * 16 + r * 8 + g4;
          if (row >= rows) continue;
          if (whole) {
            const int tok = row / p.group;
            const float inv = 1.f / divisorOf(l[mt][r], m[mt][r], pos[mt][r] >= 0);
            T* dst = reinterpret_cast<T*>(p.out) + (s.begin + tok) * p.oSt + (use.h * p.group + row - tok * p.group) * p.oSh + c4 * 2;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) *reinterpret_cast<uint32_t*>(dst + 8 * i) = pack2<T>(o[mt][i][2 * r] * inv, o[mt][i][2 * r + 1] * inv);
          } else {
            float* dst = slot + row * (D + kTail);
#pragma unroll
            for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(dst + 8 * i + c4 * 2) = make_float2(o[mt][i][2 * r], o[mt][i][2 * r + 1]);
            if (c4 == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(m[mt][r], l[mt][r]);
          }
        }
    } else {
      // The warps meet where the ring was: every load has landed and been used.
      float* sO = reinterpret_cast<float*>(smem);  // [4][kRows][D], columns of 8 swapped by the row against bank conflicts
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (c4 == 0) { sM[warp * C::kRows + mt * 16 + r * 8 + g4] = m[mt][r]; sL[warp * C::kRows + mt * 16 + r * 8 + g4] = l[mt][r]; }
      __syncthreads();
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = mt * 16 + r * 8 + g4;
          if (mt * 16 + r * 8 >= rows) continue;
          float top = sM[row];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sM[w * C::kRows + row]);
          const float f = m[mt][r] == -INFINITY ? 0.f : exp2Fast(m[mt][r] - top);
          float* dst = sO + (warp * C::kRows + row) * D + c4 * 2;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(dst + ((i ^ g4) << 3)) = make_float2(o[mt][i][2 * r] * f, o[mt][i][2 * r + 1] * f);
        }
      __syncthreads();
      constexpr int kEach = D / 16;                // elements of a thread: 16 threads a row
      const int at = (threadIdx.x & 15) * kEach;
#pragma unroll 1
      for (int row = threadIdx.x >> 4; row < rows; row += kThreads / 16) {
        float x[kEach], top = sM[row], sum = 0.f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sM[w * C::kRows + row]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) { const float mw = sM[w * C::kRows + row]; sum += mw == -INFINITY ? 0.f : sL[w * C::kRows + row] * exp2Fast(mw - top); }
#pragma unroll
        for (int e = 0; e < kEach; ++e) x[e] = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float* src = sO + (w * C::kRows + row) * D + (((at >> 3) ^ (row & 7)) << 3) + (at & 7);
#pragma unroll
          for (int e = 0; e < kEach; e += 4) {
            const float4 v = *reinterpret_cast<const float4*>(src + e);
            x[e] += v.x; x[e + 1] += v.y; x[e + 2] += v.z; x[e + 3] += v.w;
          }
        }
        const int tok = row / p.group;
        const float inv = 1.f / divisorOf(sum, top, (long long)s.len - s.n + tok >= 0);
        T* dst = reinterpret_cast<T*>(p.out) + (s.begin + tok) * p.oSt + (use.h * p.group + row - tok * p.group) * p.oSh + at;
        uint32_t w[kEach / 2];
#pragma unroll
        for (int e = 0; e < kEach / 2; ++e) w[e] = pack2<T>(x[2 * e] * inv, x[2 * e + 1] * inv);
        if constexpr (kEach == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      }
    }
  }
  if (!ok)
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);   // copies in flight land before the CTA gives its memory back
}

// Joins the parts of a pair that was cut: block (pair, rows).  Few parts: a warp takes a row alone.  Many, or a block with a single row: all
// warps take every eighth part of the row and meet.  Eight loads of a lane are under way; the order depends on the shapes alone.
constexpr int kJoinWarps = 8;
template <typename T, int D, int MT>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_decode_join_kernel(const DecodeArgs a) {
  using C = Config<D, MT>;
  using V = typename std::conditional<D == 128, float4, float2>::type;   // a lane's elements
  constexpr int kEach = D / 32;
  extern __shared__ float sF[];                    // [parts]
  __shared__ float sTop[kJoinWarps], sSum[kJoinWarps], sO[kJoinWarps][D];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const PagedArgs& p = a.p;
  const int pair = blockIdx.x, b = pair / p.kvHeads, h = pair - b * p.kvHeads;
  const int2 rec = a.records[pair];                // read before it is known to be one: the workspace holds it in any case
  const Sequence s = sequenceOf(p, b);
  const int row0 = blockIdx.y * a.joinRows, rows = s.n * p.group;
  if (s.n == 0 || (long long)s.n * p.group > C::kRows || row0 >= rows || rec.y < 2) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, parts = rec.y;
  const long long stride = (long long)a.slotRows * (D + kTail);
  // A row's sums in part n: the first warp has begun the pair, the ones behind it go on with it.
  auto partAt = [&](int row, int n) { return a.slots + slotOf(a, rec.x + n, n > 0) * stride + row * (D + kTail); };
  // Sums the parts first, first + step, ... of a row with factors that `factor` knows.
  auto add = [&](int row, int first, int step, float* x, auto factor) {
#pragma unroll 1
    for (int i = first; i < parts; i += 8 * step) {
      V v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int n = i + u * step;
        if (n < parts) v[u] = reinterpret_cast<const V*>(partAt(row, n))[lane];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int n = i + u * step;
        const float f = factor(n < parts ? n : i);
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          if (n < parts) x[e] = fmaf(reinterpret_cast<const float*>(&v[u])[e], f, x[e]);
      }
    }
  };
  auto place = [&](int row) {
    const int tok = row / p.group;
    return reinterpret_cast<T*>(p.out) + (s.begin + tok) * p.oSt + (h * p.group + row - tok * p.group) * p.oSh;
  };
  auto sees = [&](int row) { return (long long)s.len - s.n + row / p.group >= 0; };
  if (a.joinRows > 1 && parts <= 32) {
    const int row = row0 + warp;
    if (row >= rows) return;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < parts) ml = *reinterpret_cast<const float2*>(partAt(row, lane) + D);
    const float top = warpMax(ml.x), f = ml.x == -INFINITY ? 0.f : exp2Fast(ml.x - top), total = warpSum(ml.y * f), inv = 1.f / divisorOf(total, top, sees(row));
    float x[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) x[e] = 0.f;
    add(row, 0, 1, x, [&](int n) { return __shfl_sync(0xffffffffu, f, n); });
    T* dst = place(row) + lane * kEach;
    if constexpr (kEach == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(x[0] * inv, x[1] * inv), pack2<T>(x[2] * inv, x[3] * inv));
    else *reinterpret_cast<uint32_t*>(dst) = pack2<T>(x[0] * inv, x[1] * inv);
    return;
  }
  for (int row = row0; row < row0 + a.joinRows && row < rows; ++row) {
    float top = -INFINITY, sum = 0.f;
    for (int i = threadIdx.x; i < parts; i += kJoinWarps * 32) top = fmaxf(top, partAt(row, i)[D]);
    top = warpMax(top);
    if (lane == 0) sTop[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, sTop[w]);
    for (int i = threadIdx.x; i < parts; i += kJoinWarps * 32) {
      const float2 ml = *reinterpret_cast<const float2*>(partAt(row, i) + D);
      const float f = ml.x == -INFINITY ? 0.f : exp2Fast(ml.x - top);
      sF[i] = f;
      sum += ml.y * f;
    }
    sum = warpSum(sum);
    if (lane == 0) sSum[warp] = sum;
    __syncthreads();
    float x[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) x[e] = 0.f;
    add(row, warp, kJoinWarps, x, [&](int n) { return sF[n]; });
#pragma unroll
    for (int e = 0; e < kEach; ++e) sO[warp][lane * kEach + e] = x[e];
    __syncthreads();
    if (threadIdx.x < D) {
      float y = 0.f, total = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) { y += sO[w][threadIdx.x]; total += sSum[w]; }
      y /= divisorOf(total, top, sees(row));
      if constexpr (std::is_same<T, __half>::value) place(row)[threadIdx.x] = __float2half_rn(y);
      else place(row)[threadIdx.x] = __float2bfloat16_rn(y);
    }
    __syncthreads();                               // before the next row's statistics
  }
}

// Whether the keys are cut into shares, the number of CTAs, the rows of a slot and the workspace's bytes.
struct Launch { bool split; unsigned ctas; int rows; long long bytes; };
template <int D, int MT> Launch launchOf(const PagedArgs& p) {
  const long long pairs = (long long)p.batch * p.kvHeads, slots = (long long)Config<D, MT>::kCtas * deviceSMs();
  long long longest = p.reach;                     // keys that a sequence can see
  if ((long long)p.window + p.sinks + MT * 16 < longest) longest = (long long)p.window + p.sinks + MT * 16;
  const long long rows = p.maxQ * p.group;
  // a CTA a pair: up to 512 keys each, and no more work than one such pair a CTA, in at most two rounds of CTAs.  Against shares and a second
  // launch, us, 8 key heads of 128: one sequence of 256 / 512 / 1024 keys 7.5 / 12.1 / 21.4 and 11.3 / 11.6 / 11.9; 16 sequences 8 / 12.7 / 22 and
  // 14.6 / 15.3 / 20; 64 sequences of 256 keys 16.1 and 18.8, of 512 29.7 and 32.6 (which the third condition leaves to the shares: a ragged
  // batch would load its CTAs unevenly)
  const bool whole = longest <= 512 && pairs <= 2 * slots && pairs * longest <= 512 * slots;
  Launch l{!whole, 0, (int)(rows < MT * 16 ? rows : MT * 16), 0};
  l.ctas = (unsigned)(l.split ? slots : pairs);
  if (l.split) l.bytes = ((pairs * 8 + 15) & ~15LL) + kCutsOfAShare * slots * kWarps * l.rows * (D + kTail) * 4;
  return l;
}

template <typename T, int D, int MT, bool SPLIT>
int launchMain(const CUtensorMap& mk, const CUtensorMap& mv, const DecodeArgs& a, unsigned ctas, cudaStream_t st) {
  using C = Config<D, MT>;
  static DeviceOnce configured;
  const int dev = currentDevice();
  if (!configured.test(dev)) {
    LLC_CUDA_CHECK(cudaFuncSetAttribute(paged_decode_kernel<T, D, MT, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    configured.set(dev);
  }
  paged_decode_kernel<T, D, MT, SPLIT><<<ctas, kThreads, C::kSmem, st>>>(mk, mv, a);
  LLC_LAUNCH_CHECK("paged_decode_kernel");
  return LLC_OK;
}

template <typename T, int D, int MT>
int launch(const PagedArgs& p, void* workspace, long long bytes, cudaStream_t st) {
  CUtensorMap mk, mv;
  DecodeArgs a{};
  a.p = p;
  while ((1LL << a.pageShift) < p.pageSize) ++a.pageShift;
  if (!makePageMap(&mk, p.k, p.dtype, p, p.kcSp, p.kcSn, p.kcSh, kKeys) || !makePageMap(&mv, p.v, p.dtype, p, p.vcSp, p.vcSn, p.vcSh, kKeys))
    return setError(LLC_ERR_CUDA, "llc cuda: cuTensorMapEncodeTiled rejected the cache");
  const Launch l = launchOf<D, MT>(p);
  const long long pairs = (long long)p.batch * p.kvHeads;
  if (!l.split || !workspace || bytes < l.bytes) return launchMain<T, D, MT, false>(mk, mv, a, (unsigned)pairs, st);
  a.minBlocks = 4;
  a.slotRows = l.rows;
  a.warps = (int)l.ctas * kWarps;
  a.records = static_cast<int2*>(workspace);
  a.slots = reinterpret_cast<float*>(static_cast<char*>(workspace) + ((pairs * 8 + 15) & ~15LL));
  if (int rc = launchMain<T, D, MT, true>(mk, mv, a, l.ctas, st)) return rc;
  cudaLaunchConfig_t cfg{};
  // a row a block while that leaves the SMs with few blocks each: then the parts are many and their sums long
  a.joinRows = pairs * l.rows <= 8LL * deviceSMs() ? 1 : kJoinWarps;
  cfg.gridDim = dim3((unsigned)pairs, (unsigned)((l.rows + a.joinRows - 1) / a.joinRows));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.dynamicSmemBytes = l.ctas * kWarps * sizeof(float);   // a pair has at most a part in every warp
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  LLC_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_decode_join_kernel<T, D, MT>, a));
  return LLC_OK;
}

template <typename F> auto choose(const PagedArgs& p, bool wide, F f) {
  if (p.dtype == LLC_BFLOAT16) {
    if (p.d == 64) return wide ? f.template run<__nv_bfloat16, 64, 2>() : f.template run<__nv_bfloat16, 64, 1>();
    return wide ? f.template run<__nv_bfloat16, 128, 2>() : f.template run<__nv_bfloat16, 128, 1>();
  }
  if (p.d == 64) return wide ? f.template run<__half, 64, 2>() : f.template run<__half, 64, 1>();
  return wide ? f.template run<__half, 128, 2>() : f.template run<__half, 128, 1>();
}
struct Runner {
  const PagedArgs& p; void* workspace; long long bytes; cudaStream_t st;
  template <typename T, int D, int MT> int run() { return launch<T, D, MT>(p, workspace, bytes, st); }
};
struct Sizer {
  const PagedArgs& p;
  template <typename T, int D, int MT> long long run() {
    return launchOf<D, MT>(p).bytes;
  }
};

}  // namespace

// The sequences of at most 16 rows (new tokens x query heads of a key head), or 32 where wide; the others are left alone.
long long pagedDecodeWorkspace(const PagedArgs& p, bool wide) { return choose(p, wide, Sizer{p}); }
int pagedDecode(const PagedArgs& p, bool wide, void* workspace, long long bytes, cudaStream_t st) { return choose(p, wide, Runner{p, workspace, bytes, st}); }

int pagedDecodeStatus() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_pagedDecodeStatus, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_pagedDecodeStatus, &zero, sizeof(int));
  return v;
}

}  // namespace llc
