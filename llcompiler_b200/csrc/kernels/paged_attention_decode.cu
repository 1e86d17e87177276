// Paged attention for sequences of few new tokens (decoding): rows = new tokens x query heads of one key head, at most 16 or
// 32 of them, so that the cache is read once for all of them.
// Mathematics: out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m), s_j = scale log2(e) q.k_j, m any number near the maximum of s; sums
// over parts of the keys with maxima m_i join as sum_i 2^(m_i - m) (...)_i.
// Bound: the cache's bytes.  A block of 64 keys and values of one head (32 KB at d = 128) has to leave memory every 1400 cycles
// on every SM; the warps' 32 small matrix products a block take a third of that, so plain mma.sync from swizzled shared memory
// serves (tcgen05 would compute 128 rows for the 4 to 16 that exist, with a longer chain from scores to values).
//   producer warp   one lane a page: TMA boxes of page rows x 64 elements into a ring of stages (K and V of 64 keys)
//   4 warps         16 keys of the stage each, with a running maximum and sum of their own: no exchange between warps
//                   until the end of the sequence, where they meet in shared memory
// Work: the blocks of 64 keys of all (sequence, key head) pairs form one line, cut into equal shares, one a CTA, so that
// ragged batches and single long sequences load every SM alike.  A pair that is cut leaves partial sums in the workspace,
// which a second kernel joins (launched early, it waits for this one on the device).
#include "paged_attention.cuh"
#include "tc_common.cuh"
#include "tensor_map.h"

namespace llc {
__device__ int g_pagedDecodeStatus = 0;   // non-zero after a bounded wait gave up: 8 producer, 9 consumer

namespace {
using namespace tc;

constexpr int kConsumers = 4;                      // warps
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr int kKeys = 64;                          // keys of a block (and of a stage)

template <int D, int MT> struct Config {
  static constexpr int kRows = 16 * MT;
  static constexpr int kCtas = MT == 1 ? 2 : 1;    // of an SM; 32 rows need the registers of both
  static constexpr int kHalf = kKeys * 128;        // bytes of 64 keys x 64 elements
  static constexpr int kTensor = kHalf * (D / 64); // K or V of a stage
  static constexpr int kStage = 2 * kTensor;
  static constexpr int kStages = (kCtas == 2 ? 96 : 160) * 1024 / kStage;
  static constexpr int kMerge = kConsumers * 8 * D * 4;   // 8 rows of every warp
  static constexpr int kMisc = 256 + 2 * kConsumers * kRows * 4;   // barriers and the share's start, then m and l of every warp's rows
  static constexpr int kSmem = kStages * kStage + kMerge + kMisc;
  static_assert(kStages <= 12 && kCtas * (kSmem + 1024) <= 228 * 1024, "the CTAs of an SM share 228 KB");
  static constexpr int kSlot = kRows * (D + 2);    // floats of a partial sum in the workspace: O, then m, then l
};

struct DecodeArgs {
  PagedArgs p;
  int pageShift, boxRows;      // page_size = 1 << pageShift; rows of a TMA box
  int split;                   // 0: one CTA a pair
  int minBlocks;               // least share of a CTA
  int4* records;               // [CTAs]: pair that starts in this CTA and goes on (or -1), number of CTAs it goes on in
  float* slots;                // [2 * CTAs][kSlot]
};

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
__device__ __forceinline__ void consumerBarrier() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); }

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kThreads, Config<D, MT>::kCtas)
paged_decode_kernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV, const __grid_constant__ DecodeArgs a) {
  using C = Config<D, MT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;
  float* sMerge = reinterpret_cast<float*>(smem + C::kStages * C::kStage);
  uint8_t* misc = smem + C::kStages * C::kStage + C::kMerge;
  uint64_t* full = reinterpret_cast<uint64_t*>(misc);
  uint64_t* empty = full + 12;
  volatile int* abortWord = reinterpret_cast<volatile int*>(misc + 192);
  long long* sScan = reinterpret_cast<long long*>(misc + 200);      // [4] sums of the warps' sequences
  long long* sStart = sScan + kConsumers;                           // first block of this CTA's share within its sequence
  int* sSeq = reinterpret_cast<int*>(sStart + 1);                   // that sequence
  float* sM = reinterpret_cast<float*>(misc + 256);                 // [4][kRows]
  float* sL = sM + kConsumers * C::kRows;
  const PagedArgs& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (smemAddr(smem) & 1023) {                     // the swizzled tiles need it; no static shared memory lies before them
    if (threadIdx.x == 0) { atomicExch(&g_pagedDecodeStatus, 8); if (a.split) a.records[blockIdx.x] = make_int4(-1, 0, 0, 0); }
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) { mbarInit(&full[i], 1); mbarInit(&empty[i], kConsumers); }
    *abortWord = 0;
    fenceBarrierInit();
  }
  asm volatile("griddepcontrol.launch_dependents;");
  // This CTA's share of the line of blocks.
  int b, h;                    // sequence and key head of the current pair
  long long unit, left;        // its first block here, blocks left in the share
  long long share = 0;
  if (!a.split) {
    __syncthreads();
    b = blockIdx.x / p.kvHeads;
    h = blockIdx.x - b * p.kvHeads;
    unit = 0;
    left = countOf(p, b, C::kRows);
  } else {
    const int per = (p.batch + kConsumers * 32 - 1) / (kConsumers * 32);
    const int first = threadIdx.x * per;
    long long mine = 0, before = 0;
    if (warp < kConsumers) {
      for (int i = first; i < first + per && i < p.batch; ++i) mine += countOf(p, i, C::kRows);
      long long run = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const long long x = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += x; }
      if (lane == 31) sScan[warp] = run;
      before = run - mine;
    }
    if (threadIdx.x == 0) *sSeq = -1;
    __syncthreads();
    long long all = 0;
#pragma unroll
    for (int w = 0; w < kConsumers; ++w) { if (w < warp) before += sScan[w]; all += sScan[w]; }
    all *= p.kvHeads;
    share = (all + gridDim.x - 1) / gridDim.x;
    if (share < a.minBlocks) share = a.minBlocks;
    const long long start = blockIdx.x * share;
    if (warp < kConsumers && start >= before * p.kvHeads && start < (before + mine) * p.kvHeads) {
      for (int i = first; i < first + per && i < p.batch; ++i) {
        const long long c = countOf(p, i, C::kRows);
        if (start < (before + c) * p.kvHeads) { *sSeq = i; sStart[0] = start - before * p.kvHeads; break; }
        before += c;
      }
    }
    __syncthreads();
    b = *sSeq;
    left = all - start < share ? all - start : share;
    if (b < 0 || left <= 0) {                      // more CTAs than shares
      if (threadIdx.x == 0) a.records[blockIdx.x] = make_int4(-1, 0, 0, 0);
      return;
    }
    const int c = countOf(p, b, C::kRows);
    h = (int)(sStart[0] / c);
    unit = sStart[0] - (long long)h * c;
  }
  uint32_t it = 0;                                 // stages so far: stage it % kStages, phase it / kStages
  bool ok = true;

  if (warp == kConsumers) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) { prefetchTensorMap(&mapK); prefetchTensorMap(&mapV); }
    const int boxes = kKeys / a.boxRows, loads = boxes * (D / 64) * 2;
    const int box = lane % boxes, half = lane / boxes % (D / 64), which = lane / (boxes * (D / 64));   // this lane's load of every stage
    while (left > 0 && ok) {
      const Sequence s = sequenceOf(p, b);
      const Seen seen = seenBy(p, clipPlace((long long)s.len - s.n), s.len - 1);
      const Blocks bl = blocksOf(p, s, seen, C::kRows);
      if (bl.count == 0) { ++b; h = 0; continue; }
      const long long end = unit + left < bl.count ? unit + left : bl.count;
      left -= end - unit;
      for (; unit < end && ok; ++unit, ++it) {
        const int st = it % C::kStages;
        const long long j = keyOf(bl, (int)unit, kKeys) + (long long)box * a.boxRows;
        // a box that no token sees any key of is not looked up: it reads as zeros, as does one with a bad page number
        const bool wanted = lane < loads && (j < seen.sinkEnd || (j < seen.hi && j + a.boxRows > seen.lo));
        long long page = -1;
        if (wanted) {
          page = pageOf(p, b, j >> a.pageShift);
          if (page < 0 && which == 0 && half == 0 && p.badPages) atomicAdd(p.badPages, 1);
        }
        if (it >= C::kStages) ok = __all_sync(0xffffffffu, mbarWait(&empty[st], (it / C::kStages - 1) & 1u, abortWord));
        if (!ok) break;
        if (lane == 0) mbarExpectTx(&full[st], C::kStage);
        __syncwarp();
        if (lane < loads) {
          uint8_t* dst = ring + st * C::kStage + which * C::kTensor + half * C::kHalf + box * a.boxRows * 128;
          tmaLoad4d(dst, which ? &mapV : &mapK, &full[st], half * 64, (int)(j & ((1 << a.pageShift) - 1)), h, page < 0 ? (int)p.numPages : (int)page);
        }
      }
      unit = 0;
      if (++h == p.kvHeads) { h = 0; ++b; }
    }
    if (!ok) {
      if (lane == 0) atomicExch(&g_pagedDecodeStatus, 8);
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);   // copies in flight land before the CTA gives its memory back
    }
    return;
  }
  // -------------------------------------------------------------------- consumers
  const uint32_t ringAddr = smemAddr(ring);
  const int g4 = lane >> 2, c4 = lane & 3;         // a thread's row (and row + 8) of a tile, its pair of columns
  // K: matrices (keys 0-7, d 0-7), (keys 0-7, d 8-15), (keys 8-15, d 0-7), (keys 8-15, d 8-15) of a 16 x 16 step
  const int kRow = warp * 16 + (lane & 7) + ((lane >> 4) << 3), kChunk = (lane >> 3) & 1;
  // V, transposed on the way: (keys 0-7, d 0-7), (keys 8-15, d 0-7), (keys 0-7, d 8-15), (keys 8-15, d 8-15)
  const int vRow = warp * 16 + (lane & 15), vChunk = lane >> 4;
  const uint32_t kBase = ringAddr + kRow * 128, vBase = ringAddr + C::kTensor + vRow * 128;
  constexpr float kShift = weightShift<T>();
  int4 record = make_int4(-1, 0, 0, 0);
  while (left > 0) {
    const Sequence s = sequenceOf(p, b);
    const Seen seen = seenBy(p, clipPlace((long long)s.len - s.n), s.len - 1);
    const Blocks bl = blocksOf(p, s, seen, C::kRows);
    if (bl.count == 0) { ++b; h = 0; continue; }
    const long long begin = unit, end = unit + left < bl.count ? unit + left : bl.count;
    left -= end - unit;
    const int rows = (int)s.n * p.group;
    const T* q = reinterpret_cast<const T*>(p.q);
    uint32_t qf[MT][D / 16][4];
    long long pos[MT][2];                          // places of this thread's rows
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = mt * 16 + r * 8 + g4;
        const int tok = row / p.group;
        pos[mt][r] = s.len - s.n + tok;
        const T* src = q + (s.begin + tok) * p.qSt + (h * p.group + row - tok * p.group) * p.qSh + c4 * 2;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          qf[mt][ks][r] = row < rows ? *reinterpret_cast<const uint32_t*>(src + ks * 16) : 0u;
          qf[mt][ks][2 + r] = row < rows ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8) : 0u;
        }
      }
    float o[MT][D / 8][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) { o[mt][i][0] = o[mt][i][1] = o[mt][i][2] = o[mt][i][3] = 0.f; }
      m[mt][0] = m[mt][1] = -INFINITY;
      l[mt][0] = l[mt][1] = 0.f;
    }
    for (; unit < end; ++unit, ++it) {
      const int st = it % C::kStages;
      const long long j0 = keyOf(bl, (int)unit, kKeys) + warp * 16;   // this warp's keys
      if (ok && !mbarWait(&full[st], (it / C::kStages) & 1u, abortWord)) { ok = false; atomicExch(&g_pagedDecodeStatus, 9); }
      __syncwarp();
      const uint32_t kAddr = kBase + st * C::kStage, vAddr = vBase + st * C::kStage;
      float sc[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[mt][0][i] = sc[mt][1][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t bf[4];
        ldmatrix4(kAddr + (ks / 4) * C::kHalf + ((((ks % 4) * 2 + kChunk) ^ (kRow & 7)) << 4), bf);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) { mma16816<T>(sc[mt][0], qf[mt][ks], bf[0], bf[1]); mma16816<T>(sc[mt][1], qf[mt][ks], bf[2], bf[3]); }
      }
      // every row sees all 16 keys: they lie before the first token, and inside the last one's window or among the sinks
      const bool whole = j0 + 15 <= s.len - s.n && (j0 > s.len - 1 - p.window || j0 + 16 <= p.sinks);
      uint32_t vMask[2] = {0xffffffffu, 0xffffffffu}, hidden = 0;   // bits of the scores that are not seen: mt, row, column
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {              // columns c4 * 2 + {0, 1} and 8 more
          const long long j = j0 + c4 * 2 + (i & 1) + (i >> 1) * 8;
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
        ldmatrix4t(vAddr + (c / 4) * C::kHalf + ((((c % 4) * 2 + vChunk) ^ (vRow & 7)) << 4), bf);
        bf[0] &= vMask[0]; bf[1] &= vMask[1]; bf[2] &= vMask[0]; bf[3] &= vMask[1];
        if (!whole && s.n > 1 && __any_sync(0xffffffffu, notFinite<T>(bf[0]) || notFinite<T>(bf[1]) || notFinite<T>(bf[2]) || notFinite<T>(bf[3]))) {
          // a value that some tokens see and others do not is NaN or infinite: token by token, its rows take the product
          // with the values that it sees
          for (int tok = 0; tok < s.n; ++tok) {
            const long long at = s.len - s.n + tok;
            uint32_t tm[2] = {0u, 0u};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const long long j = j0 + c4 * 2 + (i & 1) + (i >> 1) * 8;
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
      __syncwarp();
      if (lane == 0) mbarArrive(&empty[st]);
    }
    // The four warps meet: statistics first, then 8 rows at a time.
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[mt][r] += __shfl_xor_sync(0xffffffffu, l[mt][r], 1);
        l[mt][r] += __shfl_xor_sync(0xffffffffu, l[mt][r], 2);
        if (c4 == 0) { sM[warp * C::kRows + mt * 16 + r * 8 + g4] = m[mt][r]; sL[warp * C::kRows + mt * 16 + r * 8 + g4] = l[mt][r]; }
      }
    consumerBarrier();
    const bool wholePair = begin == 0 && end == bl.count;
    float* slot = a.slots + (2LL * blockIdx.x + (begin == 0)) * C::kSlot;
    if (!wholePair && begin == 0) record = make_int4(b, h, (int)((bl.count - end + share - 1) / share), 0);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row0 = mt * 16 + r * 8;
        if (row0 < rows) {
          {
            const int row = row0 + g4;
            float top = sM[row];
#pragma unroll
            for (int w = 1; w < kConsumers; ++w) top = fmaxf(top, sM[w * C::kRows + row]);
            const float f = m[mt][r] == -INFINITY ? 0.f : exp2Fast(m[mt][r] - top);
            float* dst = sMerge + (warp * 8 + g4) * D + c4 * 2;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(dst + ((i ^ g4) << 3)) = make_float2(o[mt][i][2 * r] * f, o[mt][i][2 * r + 1] * f);
          }
          consumerBarrier();
          constexpr int kEach = D / 16;            // elements of a thread: 16 threads a row
          const int row = row0 + (threadIdx.x >> 4), at = (threadIdx.x & 15) * kEach;
          if (row < rows) {
            float x[kEach], top = sM[row], sum = 0.f;
#pragma unroll
            for (int w = 1; w < kConsumers; ++w) top = fmaxf(top, sM[w * C::kRows + row]);
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) { const float mw = sM[w * C::kRows + row]; sum += mw == -INFINITY ? 0.f : sL[w * C::kRows + row] * exp2Fast(mw - top); }
#pragma unroll
            for (int e = 0; e < kEach; ++e) x[e] = 0.f;
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) {
              const float* src = sMerge + (w * 8 + (row & 7)) * D + (((at >> 3) ^ (row & 7)) << 3) + (at & 7);
#pragma unroll
              for (int e = 0; e < kEach; e += 4) {
                const float4 v = *reinterpret_cast<const float4*>(src + e);
                x[e] += v.x; x[e + 1] += v.y; x[e + 2] += v.z; x[e + 3] += v.w;
              }
            }
            if (wholePair) {
              const int tok = row / p.group;
              const float inv = sum == 0.f ? 0.f : 1.f / sum;
              T* dst = reinterpret_cast<T*>(p.out) + (s.begin + tok) * p.oSt + (h * p.group + row - tok * p.group) * p.oSh + at;
              uint32_t w[kEach / 2];
#pragma unroll
              for (int e = 0; e < kEach / 2; ++e) w[e] = pack2<T>(x[2 * e] * inv, x[2 * e + 1] * inv);
              if constexpr (kEach == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
              else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
            } else {
#pragma unroll
              for (int e = 0; e < kEach; e += 4) *reinterpret_cast<float4*>(slot + row * D + at + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
              if ((threadIdx.x & 15) == 0) { slot[C::kRows * D + row] = top; slot[C::kRows * (D + 1) + row] = sum; }
            }
          }
          consumerBarrier();
        }
      }
    unit = 0;
    if (++h == p.kvHeads) { h = 0; ++b; }
  }
  if (a.split && threadIdx.x == 0) a.records[blockIdx.x] = record;
}

// Joins the parts of a pair that was cut: block (i, r) row r of the pair that starts in CTA i of the first kernel.  Its parts are
// that CTA's second slot and the first slots of the CTAs it goes on in, taken in that order.
template <typename T, int D, int MT>
__global__ void __launch_bounds__(256) paged_decode_join_kernel(const DecodeArgs a) {
  using C = Config<D, MT>;
  __shared__ float sTop[8], sSum[8], sO[8][D];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 rec = a.records[blockIdx.x];
  if (rec.x < 0) return;
  const PagedArgs& p = a.p;
  const Sequence s = sequenceOf(p, rec.x);
  const int row = blockIdx.y, parts = rec.z + 1;
  if (row >= s.n * p.group) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto slotOf = [&](int i) { return a.slots + (2LL * (blockIdx.x + i) + (i == 0)) * C::kSlot; };
  float top = -INFINITY;
  for (int i = threadIdx.x; i < parts; i += 256) top = fmaxf(top, slotOf(i)[C::kRows * D + row]);
  top = warpMax(top);
  if (lane == 0) sTop[warp] = top;
  __syncthreads();
  top = sTop[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) top = fmaxf(top, sTop[w]);
  constexpr int kEach = D / 32;
  float x[kEach], sum = 0.f;
#pragma unroll
  for (int e = 0; e < kEach; ++e) x[e] = 0.f;
#pragma unroll 4
  for (int i = warp; i < parts; i += 8) {
    const float* slot = slotOf(i);
    const float m = slot[C::kRows * D + row], l = slot[C::kRows * (D + 1) + row];
    const float f = m == -INFINITY ? 0.f : exp2Fast(m - top);
    sum += l * f;
#pragma unroll
    for (int e = 0; e < kEach; ++e) x[e] = fmaf(slot[row * D + lane + 32 * e], f, x[e]);
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) sO[warp][lane + 32 * e] = x[e];
  if (lane == 0) sSum[warp] = sum;
  __syncthreads();
  if (threadIdx.x < D) {
    float v = 0.f, total = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) { v += sO[w][threadIdx.x]; total += sSum[w]; }
    const int tok = row / p.group;
    T* dst = reinterpret_cast<T*>(p.out) + (s.begin + tok) * p.oSt + (rec.y * p.group + row - tok * p.group) * p.oSh;
    const float y = total == 0.f ? 0.f : v / total;
    if constexpr (std::is_same<T, __half>::value) dst[threadIdx.x] = __float2half_rn(y);
    else dst[threadIdx.x] = __float2bfloat16_rn(y);
  }
}

// Whether a pair's keys are cut, and how many CTAs the first kernel has.
struct Launch { bool split; unsigned ctas; };
template <int D, int MT> Launch launchOf(const PagedArgs& p) {
  const long long pairs = (long long)p.batch * p.kvHeads;
  long long longest = p.reach;                     // keys that a sequence can see
  if ((long long)p.window + p.sinks + MT * 16 < longest) longest = (long long)p.window + p.sinks + MT * 16;
  const long long slots = (long long)Config<D, MT>::kCtas * deviceSMs();
  // up to 512 keys a pair the second launch costs more than a cut saves
  if (longest <= 512) return {false, (unsigned)pairs};
  return {true, (unsigned)slots};
}

template <typename T, int D, int MT>
int launch(const PagedArgs& p, void* workspace, long long bytes, cudaStream_t st) {
  using C = Config<D, MT>;
  CUtensorMap mk, mv;
  DecodeArgs a{};
  a.p = p;
  a.boxRows = p.pageSize < kKeys ? (int)p.pageSize : kKeys;
  while ((1LL << a.pageShift) < p.pageSize) ++a.pageShift;
  if (!makePageMap(&mk, p.k, p.dtype, p, p.kcSp, p.kcSn, p.kcSh, a.boxRows) || !makePageMap(&mv, p.v, p.dtype, p, p.vcSp, p.vcSn, p.vcSh, a.boxRows))
    return setError(LLC_ERR_CUDA, "llc cuda: cuTensorMapEncodeTiled rejected the cache");
  Launch l = launchOf<D, MT>(p);
  const long long need = l.ctas * 16LL + 2LL * l.ctas * C::kSlot * 4;
  if (l.split && (!workspace || bytes < need)) l = {false, (unsigned)(p.batch * p.kvHeads)};
  a.split = l.split;
  a.minBlocks = 2;
  a.records = static_cast<int4*>(workspace);
  a.slots = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.ctas * 16LL);
  static DeviceOnce configured;
  const int dev = currentDevice();
  if (!configured.test(dev)) {
    LLC_CUDA_CHECK(cudaFuncSetAttribute(paged_decode_kernel<T, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    configured.set(dev);
  }
  paged_decode_kernel<T, D, MT><<<l.ctas, kThreads, C::kSmem, st>>>(mk, mv, a);
  LLC_LAUNCH_CHECK("paged_decode_kernel");
  if (l.split) {
    const long long rows = p.maxQ * p.group < C::kRows ? p.maxQ * p.group : C::kRows;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(l.ctas, (unsigned)rows);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    LLC_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_decode_join_kernel<T, D, MT>, a));
  }
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
    const Launch l = launchOf<D, MT>(p);
    return l.split ? l.ctas * 16LL + 2LL * l.ctas * Config<D, MT>::kSlot * 4 : 0;
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
