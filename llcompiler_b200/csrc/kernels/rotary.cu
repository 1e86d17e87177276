// Rotary positions and the writing side of the paged key / value cache.
//   llc_cuda_rotary     out = x turned by its positions' angles
//   llc_cuda_kv_append  the new tokens' keys (turned) and values into their cache slots, the queries (turned) to a tensor
// Mathematics: pair i of a head is a point of the plane and turns by a = position * inv_freq[i].  Positions go far past
// 2^17, where a product in 32 bits is off by more than the angle's meaning, so turns = position * (inv_freq / 2 pi) is a
// 64-bit product, its whole part is dropped there, and only the fraction (at most half a turn) becomes a float.
// Bound: memory; every element is read once and written once.  The sine and cosine of a (token, pair) are computed once per
// block into shared memory and used by all heads of the token; the block's loads of x are under way meanwhile.  Measured, bf16: 20736 tokens
// of 32 heads of 128 54 us replayed (6.3 TB/s), 59 call after call or with L2 flushed; 15285 tokens of 32 + 2 x 8 heads into a cache 68 - 71 us (5.5 TB/s).
// (The 16-bit form with split pairs and without a cache holds 24 bytes of a thread in memory at its 64 registers.)
#include <cuda_fp16.h>

#include "common.cuh"

namespace llc {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;       // tokens of a block, at most; a power of two
// Rows of a thread whose loads are in flight together: 4 vectors of 16 bytes twice over are 32 registers; the writing of a cache holds more
// beside them.  With 3 and with 4, us: 15285 tokens of 32 + 2 x 8 heads of 128, bf16 67.8 and 70.9, 4096 of 64-wide heads 10.8 and 12.7, 2048 of 12 + 2 x 12
// heads of 64, f16 6.5 and 7.4, 64 tokens 4.05 and 4.4; 8192 of 16 + 2 x 4 in f32 37.6 and 35.7.  Rotary of 20736 x 32 x 128 66 and 55.
template <bool CACHE> constexpr int unrolled() { return CACHE ? 3 : 4; }

struct RotArgs {
  // rows of a token: nQ heads of q (turned), then nK of k (turned, into the cache), then nK of v (copied, into the cache)
  const void* q; void* qOut; const void* k; const void* v; void* kCache; void* vCache;
  const void* positions; const double* invFreq;
  const int* table; const int* qStart; const int* kvLen; int* badPages;
  long long qSt, qSh, qoSt, qoSh, kSt, kSh, vSt, vSh, kcSp, kcSn, kcSh, vcSp, vcSn, vcSh, posSa, tableS0, numPages, pageSize, reach;
  long long tokens;
  int batch, nQ, nK, d, pairs, axes, interleaved, pos64, tokensPerBlock, rows, perRow;
  int sectionEnd[LLC_ROTARY_MAX_AXES];
};

// The sequence that row t belongs to: the number of sequences that end at or before t (batch if t is behind the last one).
// Executed by a whole warp: each step reads 32 of the ends that are left.
__device__ __forceinline__ int findSequence(const int* qStart, int batch, long long t, int lane) {
  int lo = 0, n = batch;                               // the answer lies in [lo, lo + n]
  while (n > 0) {
    const int step = (n + 31) / 32;
    const int i = lo + (lane + 1) * step;              // ends of sequences lo + step - 1, lo + 2 step - 1, ...
    const bool before = i <= lo + n && (long long)qStart[i] <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, before));
    const int left = n - c * step;
    lo += c * step;
    n = left < step - 1 ? left : step - 1;
  }
  return lo;
}

// A vector of a row as it lies in memory: 16 bytes, or one element.  (An array of 16-bit elements would cost a register each.)
template <typename T, int VEC> struct PackOf { using type = uint4; };
template <typename T> struct PackOf<T, 1> { using type = T; };
template <typename T> __device__ __forceinline__ float asFloat(T v);
template <> __device__ __forceinline__ float asFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ float asFloat<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float asFloat<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T fromFloat(float v);
template <> __device__ __forceinline__ float fromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half fromFloat<__half>(float v) { return __float2half_rn(v); }

template <typename T> __device__ __forceinline__ float2 twoFloats(uint32_t x);
template <> __device__ __forceinline__ float2 twoFloats<__nv_bfloat16>(uint32_t x) { return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 twoFloats<__half>(uint32_t x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }
template <typename T> __device__ __forceinline__ uint32_t twoRounded(float x, float y);
template <> __device__ __forceinline__ uint32_t twoRounded<__nv_bfloat16>(float x, float y) { __nv_bfloat162 v = __floats2bfloat162_rn(x, y); return *reinterpret_cast<uint32_t*>(&v); }
template <> __device__ __forceinline__ uint32_t twoRounded<__half>(float x, float y) { __half2 v = __floats2half2_rn(x, y); return *reinterpret_cast<uint32_t*>(&v); }

// Turns the pairs of two vectors: their elements e are the pair w[e], or (INTER) neighbours are a pair, VEC / 2 of them in each.
template <typename T, int VEC, bool INTER, typename P> __device__ __forceinline__ void turn(P& a, P& b, const float2* w) {
  if constexpr (VEC == 1) {
    const float x = asFloat(a), y = asFloat(b);
    a = fromFloat<T>(x * w[0].x - y * w[0].y);
    b = fromFloat<T>(x * w[0].y + y * w[0].x);
  } else {
    uint32_t* u = reinterpret_cast<uint32_t*>(&a);
    uint32_t* v = reinterpret_cast<uint32_t*>(&b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) {
        const float2 x = twoFloats<T>(u[i]), y = twoFloats<T>(v[i]);
        if constexpr (INTER) {
          const float2 wa = w[i], wb = w[4 + i];
          u[i] = twoRounded<T>(x.x * wa.x - x.y * wa.y, x.x * wa.y + x.y * wa.x);
          v[i] = twoRounded<T>(y.x * wb.x - y.y * wb.y, y.x * wb.y + y.y * wb.x);
        } else {
          const float2 w0 = w[2 * i], w1 = w[2 * i + 1];
          u[i] = twoRounded<T>(x.x * w0.x - y.x * w0.y, x.y * w1.x - y.y * w1.y);
          v[i] = twoRounded<T>(x.x * w0.y + y.x * w0.x, x.y * w1.y + y.y * w1.x);
        }
      } else if constexpr (!INTER) {
        const float x = __uint_as_float(u[i]), y = __uint_as_float(v[i]);
        u[i] = __float_as_uint(x * w[i].x - y * w[i].y);
        v[i] = __float_as_uint(x * w[i].y + y * w[i].x);
      } else if (i % 2 == 0) {
        const float x0 = __uint_as_float(u[i]), y0 = __uint_as_float(u[i + 1]), x1 = __uint_as_float(v[i]), y1 = __uint_as_float(v[i + 1]);
        const float2 wa = w[i / 2], wb = w[2 + i / 2];
        u[i] = __float_as_uint(x0 * wa.x - y0 * wa.y); u[i + 1] = __float_as_uint(x0 * wa.y + y0 * wa.x);
        v[i] = __float_as_uint(x1 * wb.x - y1 * wb.y); v[i + 1] = __float_as_uint(x1 * wb.y + y1 * wb.x);
      }
    }
  }
}

// A thread's unit is two vectors of a row that belong together: the two halves of VEC pairs, or two neighbours that are copied.
template <typename T, int VEC, bool CACHE, bool INTER>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(const RotArgs p) {
  extern __shared__ float2 sTurn[];                    // [tokensPerBlock][pairs]: (cos, sin), a token's in the order of turnAt
  // Neighbouring threads read neighbouring vectors' pairs two at a time: two pairs of every vector side by side, then the next two.
  auto turnAt = [&](int pair) {
    if (VEC < 2) return pair;
    const int j = pair / VEC, e = pair % VEC;
    return ((e >> 1) * (p.pairs / VEC) + j) * 2 + (e & 1);
  };
  __shared__ long long sPlace[kMaxTokens];             // the token's place in its sequence
  __shared__ long long sK[kMaxTokens], sV[kMaxTokens]; // element offsets of its cache slot, -1: not stored
  __shared__ int sLive[kMaxTokens];                    // the token belongs to a sequence
  __shared__ int sSeq[kMaxTokens], sStart[kThreads + 1], sLen[kThreads];
  const long long t0 = (long long)blockIdx.x * p.tokensPerBlock;
  const int nTok = (int)(p.tokens - t0 < p.tokensPerBlock ? p.tokens - t0 : p.tokensPerBlock);
  const int nTurn = p.pairs / VEC;
  // A thread stays with one token and one pair of vectors j of its rows, so that its sines and cosines are read once: rows first,
  // first + step, ...  (a row longer than a token's threads: several j).
  const int per = kThreads / p.tokensPerBlock, tok = threadIdx.x / per, lane = threadIdx.x - tok * per;
  const int step = per >= p.perRow ? per / p.perRow : 1, first = per >= p.perRow ? lane / p.perRow : 0, j0 = lane - first * p.perRow;
  const bool busy = tok < nTok && first < step;
  const long long t = t0 + tok;
  using P = typename PackOf<T, VEC>::type;
  constexpr int kUnroll = unrolled<CACHE>();
  const int turnedRows = p.pairs == 0 ? 0 : CACHE ? p.nQ + p.nK : p.nQ;
  P a[kUnroll], b[kUnroll];
  // Element offsets in a row of the two vectors j; the second may be past the row's end.
  auto offA = [&](int r, int j) { return r < turnedRows && j < nTurn && !INTER ? j * VEC : 2 * j * VEC; };
  auto offB = [&](int r, int j) { return r < turnedRows && j < nTurn && !INTER ? p.pairs + j * VEC : (2 * j + 1) * VEC; };
  auto fetch = [&](int r0, int j) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = r0 + u * step;
      if (r >= p.rows) continue;
      const T* from;
      if (!CACHE || r < p.nQ) from = reinterpret_cast<const T*>(p.q) + t * p.qSt + r * p.qSh;
      else if (r < p.nQ + p.nK) from = reinterpret_cast<const T*>(p.k) + t * p.kSt + (r - p.nQ) * p.kSh;
      else from = reinterpret_cast<const T*>(p.v) + t * p.vSt + (r - p.nQ - p.nK) * p.vSh;
      a[u] = *reinterpret_cast<const P*>(from + offA(r, j));
      if (offB(r, j) < p.d) b[u] = *reinterpret_cast<const P*>(from + offB(r, j));
    }
  };
  if (busy) fetch(first, j0);

  if (CACHE) {
    // Which sequence: the number of sequences that end at or before the token.  Up to kThreads sequences the whole table of starts and
    // lengths comes in one read; larger batches are searched, a warp a token.
    if (p.batch <= kThreads) {
      const int i = threadIdx.x;
      int end = 0x7fffffff;
      if (i < p.batch) { end = p.qStart[i + 1]; sStart[i + 1] = end; sLen[i] = p.kvLen[i]; }
      if (i == 0) sStart[0] = p.qStart[0];
      for (int n = 0; n < nTok; ++n) {
        const int c = __syncthreads_count(i < p.batch && end <= t0 + n);
        if (i == 0) sSeq[n] = c;
      }
    } else {
      for (int n = threadIdx.x >> 5; n < nTok; n += kThreads / 32) {
        const int c = findSequence(p.qStart, p.batch, t0 + n, threadIdx.x & 31);
        if ((threadIdx.x & 31) == 0) sSeq[n] = c;
      }
    }
    __syncthreads();
    // the last warp looks up the slots, while the others begin with the angles
    if (threadIdx.x >= kThreads - 32 && threadIdx.x - (kThreads - 32) < nTok) {
      const int i = threadIdx.x - (kThreads - 32), q = sSeq[i];
      const long long row = t0 + i;
      const bool few = p.batch <= kThreads;
      long long place = 0, ko = -1, vo = -1;
      bool live = q < p.batch;
      if (live) {
        const int begin = few ? sStart[q] : p.qStart[q], end = few ? sStart[q + 1] : p.qStart[q + 1];
        live = row >= begin;
        if (live) {
          long long len = few ? sLen[q] : p.kvLen[q];
          len = len < 0 ? 0 : len > p.reach ? p.reach : len;
          place = len - ((long long)end - begin) + (row - begin);
          const long long page = place >= 0 && place < p.reach ? p.table[q * p.tableS0 + place / p.pageSize] : -1;
          if (page >= 0 && page < p.numPages) {
            ko = page * p.kcSp + (place % p.pageSize) * p.kcSn;
            vo = page * p.vcSp + (place % p.pageSize) * p.vcSn;
          } else if (p.badPages) {
            atomicAdd(p.badPages, 1);
          }
        }
      }
      sPlace[i] = place; sK[i] = ko; sV[i] = vo; sLive[i] = live;
    }
    if (!p.positions) __syncthreads();
  }
  for (int i = threadIdx.x; i < nTok * p.pairs; i += kThreads) {
    const int n = i / p.pairs, pair = i - n * p.pairs;
    int axis = 0;
    while (axis < p.axes - 1 && pair >= p.sectionEnd[axis]) ++axis;
    long long pos;
    if (CACHE && !p.positions) pos = sPlace[n];
    else {
      const long long at = axis * p.posSa + t0 + n;
      pos = p.pos64 ? reinterpret_cast<const long long*>(p.positions)[at] : reinterpret_cast<const int*>(p.positions)[at];
    }
    double turns = (double)pos * (p.invFreq[pair] * 0.15915494309189533577);   // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif(2.f * (float)turns, &s, &c);
    sTurn[n * p.pairs + turnAt(pair)] = make_float2(c, s);
  }
  __syncthreads();
  if (!busy) return;

  const bool live = !CACHE || sLive[tok];
  const long long kSlot = CACHE ? sK[tok] : -1, vSlot = CACHE ? sV[tok] : -1;
  for (int j = j0; j < p.perRow; j += per) {
    float2 w[VEC];
    if (j < nTurn) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = sTurn[tok * p.pairs + turnAt(j * VEC + e)];
    }
    for (int r0 = first; r0 < p.rows; r0 += kUnroll * step) {
      if (r0 != first || j != j0) fetch(r0, j);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int r = r0 + u * step;
        if (r >= p.rows) continue;
        T* to;
        if (!CACHE || r < p.nQ) {
          if (!live) continue;
          to = reinterpret_cast<T*>(p.qOut) + t * p.qoSt + r * p.qoSh;
        } else if (r < p.nQ + p.nK) {
          if (kSlot < 0) continue;
          to = reinterpret_cast<T*>(p.kCache) + kSlot + (r - p.nQ) * p.kcSh;
        } else {
          if (vSlot < 0) continue;
          to = reinterpret_cast<T*>(p.vCache) + vSlot + (r - p.nQ - p.nK) * p.vcSh;
        }
        if (r < turnedRows && j < nTurn) turn<T, VEC, INTER>(a[u], b[u], w);
        *reinterpret_cast<P*>(to + offA(r, j)) = a[u];
        if (offB(r, j) < p.d) *reinterpret_cast<P*>(to + offB(r, j)) = b[u];
      }
    }
  }
}

template <typename T, int VEC, bool CACHE>
int launch(RotArgs& a, cudaStream_t st) {
  constexpr int kUnroll = unrolled<CACHE>();
  // Tokens of a block: a power of two, as many as give every thread kUnroll rows (twice that when it writes a cache, whose lookups are
  // then shared by more rows: 15285 tokens of 32 + 2 x 8 heads of 128 67.8 us against 69.3, 8192 of 64 + 2 x 8 61.2 against 68.5, 4096 of 32 + 2 x 8 of 64
  // 10.8 against 11.3), fewer while the grid has less than two blocks an SM,
  // and no more than shared memory has room for (48 KB without an opt-in).
  a.rows = CACHE ? a.nQ + 2 * a.nK : a.nQ;
  a.perRow = (a.d + 2 * VEC - 1) / (2 * VEC);
  int tok = 1;
  while (2 * tok <= kMaxTokens && 2LL * tok * a.rows * a.perRow <= kThreads * kUnroll * (CACHE ? 2 : 1) && 2LL * tok * a.perRow <= kThreads && 2LL * tok * a.pairs * (long long)sizeof(float2) <= 40960 &&
         a.tokens >= 2LL * tok * 2 * deviceSMs())
    tok *= 2;
  a.tokensPerBlock = tok;
  const long long grid = (a.tokens + tok - 1) / tok;
  if (a.interleaved) rotary_kernel<T, VEC, CACHE, true><<<(unsigned)grid, kThreads, tok * a.pairs * sizeof(float2), st>>>(a);
  else rotary_kernel<T, VEC, CACHE, false><<<(unsigned)grid, kThreads, tok * a.pairs * sizeof(float2), st>>>(a);
  LLC_LAUNCH_CHECK("rotary_kernel");
  return LLC_OK;
}
// 16-byte vectors where every pointer, stride and boundary allows them, else single elements.
template <typename T, bool CACHE>
int chooseVector(RotArgs& a, bool aligned, cudaStream_t st) {
  return aligned ? launch<T, 16 / (int)sizeof(T), CACHE>(a, st) : launch<T, 1, CACHE>(a, st);
}
template <bool CACHE>
int chooseType(RotArgs& a, int dtype, bool aligned, cudaStream_t st) {
  if (dtype == LLC_FLOAT32) return chooseVector<float, CACHE>(a, aligned, st);
  if (dtype == LLC_BFLOAT16) return chooseVector<__nv_bfloat16, CACHE>(a, aligned, st);
  return chooseVector<__half, CACHE>(a, aligned, st);
}

bool floatType(int dt) { return dt == LLC_FLOAT32 || dt == LLC_BFLOAT16 || dt == LLC_FLOAT16; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The rotary part of a parameter block: pairs, axes and sections.
int checkTurn(const char* who, int64_t d, int64_t pairs, int32_t axes, const int32_t* sections, const void* positions, int32_t posDtype, RotArgs* a) {
  const std::string w = std::string("llc argument: ") + who + " ";
  if (pairs < 1 || 2 * pairs > d) return setError(LLC_ERR_ARGUMENT, w + "pairs must lie between 1 and d / 2");
  if (axes < 1 || axes > LLC_ROTARY_MAX_AXES) return setError(LLC_ERR_ARGUMENT, w + "1 to 4 axes");
  int64_t sum = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0) return setError(LLC_ERR_ARGUMENT, w + "negative section");
    sum += sections[i];
    a->sectionEnd[i] = (int)sum;
  }
  if (sum != pairs) return setError(LLC_ERR_ARGUMENT, w + "the sections must add up to pairs");
  if (positions && posDtype != LLC_INT32 && posDtype != LLC_INT64) return setError(LLC_ERR_UNSUPPORTED, w + "positions must be i32 or i64");
  a->pairs = (int)pairs; a->axes = axes; a->pos64 = posDtype == LLC_INT64;
  return LLC_OK;
}

}  // namespace
}  // namespace llc

using namespace llc;

extern "C" int llc_cuda_rotary(const LlcRotaryParams* p, void* stream) {
  if (!p) return setError(LLC_ERR_ARGUMENT, "llc argument: rotary null parameter block");
  if (p->tokens < 0 || p->heads < 0 || p->d < 1 || p->d > 16384) return setError(LLC_ERR_ARGUMENT, "llc argument: rotary extents");
  if (!floatType(p->dtype)) return setError(LLC_ERR_UNSUPPORTED, "llc argument: rotary tensors must be f32, bf16 or f16");
  RotArgs a{};
  if (int rc = checkTurn("rotary", p->d, p->pairs, p->axes, p->sections, p->positions, p->pos_dtype, &a)) return rc;
  if (p->tokens == 0 || p->heads == 0) return LLC_OK;
  if (!p->x || !p->out || !p->positions || !p->inv_freq) return setError(LLC_ERR_ARGUMENT, "llc argument: rotary null operand");
  if (p->tokens > 0x7FFFFFFFLL || p->heads > 16384 || p->heads * p->d > (1LL << 22) || p->pairs > 4096) return setError(LLC_ERR_UNSUPPORTED, "llc argument: rotary too large");
  a.q = p->x; a.qOut = p->out; a.positions = p->positions; a.invFreq = p->inv_freq;
  a.qSt = p->x_st; a.qSh = p->x_sh; a.qoSt = p->o_st; a.qoSh = p->o_sh; a.posSa = p->pos_sa;
  a.tokens = p->tokens; a.nQ = (int)p->heads; a.d = (int)p->d; a.interleaved = p->interleaved != 0;
  const int64_t vec = 16 / dtypeBytes(p->dtype);
  if (p->tokens == 1) a.qSt = a.qoSt = 0;              // the stride of a dim of one element says nothing
  if (p->heads == 1) a.qSh = a.qoSh = 0;
  const bool al = aligned16(p->x) && aligned16(p->out) && p->d % vec == 0 && p->pairs % vec == 0 && a.qSt % vec == 0 && a.qSh % vec == 0 &&
                  a.qoSt % vec == 0 && a.qoSh % vec == 0;
  return chooseType<false>(a, p->dtype, al, (cudaStream_t)stream);
}

extern "C" int llc_cuda_kv_append(const LlcKvAppendParams* p, void* stream) {
  if (!p) return setError(LLC_ERR_ARGUMENT, "llc argument: kv_append null parameter block");
  if (p->tokens < 0 || p->batch < 0 || p->heads < 0 || p->kv_heads < 1 || p->d < 1 || p->d > 16384 || p->num_pages < 0 || p->page_size < 1 || p->table_width < 0)
    return setError(LLC_ERR_ARGUMENT, "llc argument: kv_append extents");
  if (!floatType(p->dtype)) return setError(LLC_ERR_UNSUPPORTED, "llc argument: kv_append tensors must be f32, bf16 or f16");
  RotArgs a{};
  if (p->inv_freq) {
    if (int rc = checkTurn("kv_append", p->d, p->pairs, p->axes, p->sections, p->positions, p->pos_dtype, &a)) return rc;
  }
  if (p->q && !p->q_out) return setError(LLC_ERR_ARGUMENT, "llc argument: kv_append queries without a place to go");
  if (p->tokens == 0 || p->batch == 0) return LLC_OK;
  if (!p->k || !p->v || !p->q_start || !p->kv_len || (p->table_width > 0 && !p->page_table) || (p->num_pages > 0 && (!p->k_cache || !p->v_cache)))
    return setError(LLC_ERR_ARGUMENT, "llc argument: kv_append null operand");
  const int64_t nq = p->q ? p->heads : 0;
  if (p->tokens > 0x7FFFFFFFLL || p->batch > (1 << 20) || nq > 16384 || p->kv_heads > 8192 || (nq + 2 * p->kv_heads) * p->d > (1LL << 22) || p->pairs > 4096 ||
      p->num_pages > 0x7FFFFFFFLL || p->table_width > 0x7FFFFFFFLL || p->page_size > (1 << 20))
    return setError(LLC_ERR_UNSUPPORTED, "llc argument: kv_append too large");
  a.q = p->q; a.qOut = p->q_out; a.k = p->k; a.v = p->v; a.kCache = p->k_cache; a.vCache = p->v_cache;
  a.positions = p->positions; a.invFreq = p->inv_freq; a.table = p->page_table; a.qStart = p->q_start; a.kvLen = p->kv_len; a.badPages = p->bad_pages;
  a.qSt = p->q_st; a.qSh = p->q_sh; a.qoSt = p->qo_st; a.qoSh = p->qo_sh; a.kSt = p->k_st; a.kSh = p->k_sh; a.vSt = p->v_st; a.vSh = p->v_sh;
  a.kcSp = p->kc_sp; a.kcSn = p->kc_sn; a.kcSh = p->kc_sh; a.vcSp = p->vc_sp; a.vcSn = p->vc_sn; a.vcSh = p->vc_sh;
  a.posSa = p->pos_sa; a.tableS0 = p->table_s0; a.numPages = p->num_pages; a.pageSize = p->page_size;
  a.reach = p->table_width * p->page_size;
  a.tokens = p->tokens; a.batch = (int)p->batch; a.nQ = (int)nq; a.nK = (int)p->kv_heads; a.d = (int)p->d; a.interleaved = p->interleaved != 0;
  const int64_t vec = 16 / dtypeBytes(p->dtype);
  bool al = p->d % vec == 0 && a.pairs % vec == 0;
  for (const void* x : {p->k, p->v, (const void*)p->k_cache, (const void*)p->v_cache}) al = al && aligned16(x);
  if (p->tokens == 1) a.qSt = a.qoSt = a.kSt = a.vSt = 0;   // the stride of a dim of one element says nothing
  if (nq <= 1) a.qSh = a.qoSh = 0;
  if (p->kv_heads == 1) a.kSh = a.vSh = a.kcSh = a.vcSh = 0;
  if (nq) al = al && aligned16(p->q) && aligned16(p->q_out);
  for (long long s : {a.qSt, a.qSh, a.qoSt, a.qoSh, a.kSt, a.kSh, a.vSt, a.vSh, a.kcSp, a.kcSn, a.kcSh, a.vcSp, a.vcSn, a.vcSh}) al = al && s % vec == 0;
  return chooseType<true>(a, p->dtype, al, (cudaStream_t)stream);
}
