// Rotary positions and the writing side of the paged key / value cache.
//   llc_cuda_rotary     out = x turned by its positions' angles
//   llc_cuda_kv_append  the new tokens' keys (turned) and values into their cache slots, the queries (turned) to a tensor
// Mathematics: pair i of a head is a point of the plane and turns by a = position * inv_freq[i].  Positions go far past
// 2^17, where a product in 32 bits is off by more than the angle's meaning, so turns = position * (inv_freq / 2 pi) is a
// 64-bit product, its whole part is dropped there, and only the fraction (at most half a turn) becomes a float.
// Bound: memory; every element is read once and written once.  The sine and cosine of a (token, pair) are computed once per
// block into shared memory and used by all heads of the token.
#include <cuda_fp16.h>

#include "common.cuh"

namespace llc {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;       // tokens of a block
constexpr int kUnroll = 4;           // items of a thread whose loads are in flight together

struct RotArgs {
  // rows of a token: nQ heads of q (turned), then nK of k (turned, into the cache), then nK of v (copied, into the cache)
  const void* q; void* qOut; const void* k; const void* v; void* kCache; void* vCache;
  const void* positions; const double* invFreq;
  const int* table; const int* qStart; const int* kvLen; int* badPages;
  long long qSt, qSh, qoSt, qoSh, kSt, kSh, vSt, vSh, kcSp, kcSn, kcSh, vcSp, vcSn, vcSh, posSa, tableS0, numPages, pageSize, reach;
  long long tokens;
  int batch, nQ, nK, d, pairs, axes, interleaved, pos64, tokensPerBlock;
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

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };
template <typename T> __device__ __forceinline__ float asFloat(T v);
template <> __device__ __forceinline__ float asFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ float asFloat<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float asFloat<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T fromFloat(float v);
template <> __device__ __forceinline__ float fromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half fromFloat<__half>(float v) { return __float2half_rn(v); }

// An item is two vectors of a row that belong together: the two halves of VEC pairs, or two neighbours that are copied.
template <typename T, int VEC, bool CACHE>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotArgs p) {
  extern __shared__ float2 sTurn[];                    // [tokensPerBlock][pairs]: (cos, sin)
  __shared__ long long sPlace[kMaxTokens];             // the token's place in its sequence
  __shared__ long long sK[kMaxTokens], sV[kMaxTokens]; // element offsets of its cache slot, -1: not stored
  __shared__ int sLive[kMaxTokens];                    // the token belongs to a sequence
  const long long t0 = (long long)blockIdx.x * p.tokensPerBlock;
  const int nTok = (int)(p.tokens - t0 < p.tokensPerBlock ? p.tokens - t0 : p.tokensPerBlock);
  if (CACHE) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = warp; i < nTok; i += kThreads / 32) {
      const long long t = t0 + i;
      const int b = findSequence(p.qStart, p.batch, t, lane);
      if (lane == 0) {
        long long place = 0, ko = -1, vo = -1;
        const bool live = b < p.batch && t >= p.qStart[b];
        if (live) {
          const int begin = p.qStart[b], end = p.qStart[b + 1];
          long long len = p.kvLen[b];
          len = len < 0 ? 0 : len > p.reach ? p.reach : len;
          place = len - ((long long)end - begin) + (t - begin);
          const long long page = place >= 0 && place < p.reach ? p.table[b * p.tableS0 + place / p.pageSize] : -1;
          if (page >= 0 && page < p.numPages) {
            ko = page * p.kcSp + (place % p.pageSize) * p.kcSn;
            vo = page * p.vcSp + (place % p.pageSize) * p.vcSn;
          } else if (p.badPages) {
            atomicAdd(p.badPages, 1);
          }
        }
        sPlace[i] = place; sK[i] = ko; sV[i] = vo; sLive[i] = live;
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < nTok * p.pairs; i += kThreads) {
    const int tok = i / p.pairs, pair = i - tok * p.pairs;
    int axis = 0;
    while (axis < p.axes - 1 && pair >= p.sectionEnd[axis]) ++axis;
    long long pos;
    if (CACHE && !p.positions) pos = sPlace[tok];
    else {
      const long long at = axis * p.posSa + t0 + tok;
      pos = p.pos64 ? reinterpret_cast<const long long*>(p.positions)[at] : reinterpret_cast<const int*>(p.positions)[at];
    }
    double turns = (double)pos * (p.invFreq[pair] * 0.15915494309189533577);   // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif(2.f * (float)turns, &s, &c);
    sTurn[i] = make_float2(c, s);
  }
  __syncthreads();

  const int rows = CACHE ? p.nQ + 2 * p.nK : p.nQ;
  const int perRow = (p.d + 2 * VEC - 1) / (2 * VEC), nTurn = p.pairs / VEC;
  const int items = nTok * rows * perRow;
  using P = Pack<T, VEC>;
  for (int base = threadIdx.x; base < items; base += kThreads * kUnroll) {
    P a[kUnroll], b[kUnroll];
    T* to[kUnroll];
    int offA[kUnroll], offB[kUnroll], at[kUnroll];     // element offsets in the row (-1: none), index into sTurn (-1: a copy)
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int idx = base + u * kThreads;
      to[u] = nullptr;
      if (idx >= items) continue;
      const int row = idx / perRow, j = idx - row * perRow;
      const int tok = row / rows, r = row - tok * rows;
      const long long t = t0 + tok;
      const T* from;
      bool turned = p.pairs > 0;
      if (!CACHE || r < p.nQ) {
        if (CACHE && !sLive[tok]) continue;
        from = reinterpret_cast<const T*>(p.q) + t * p.qSt + r * p.qSh;
        to[u] = reinterpret_cast<T*>(p.qOut) + t * p.qoSt + r * p.qoSh;
      } else if (r < p.nQ + p.nK) {
        if (sK[tok] < 0) continue;
        from = reinterpret_cast<const T*>(p.k) + t * p.kSt + (r - p.nQ) * p.kSh;
        to[u] = reinterpret_cast<T*>(p.kCache) + sK[tok] + (r - p.nQ) * p.kcSh;
      } else {
        if (sV[tok] < 0) continue;
        from = reinterpret_cast<const T*>(p.v) + t * p.vSt + (r - p.nQ - p.nK) * p.vSh;
        to[u] = reinterpret_cast<T*>(p.vCache) + sV[tok] + (r - p.nQ - p.nK) * p.vcSh;
        turned = false;
      }
      if (turned && j < nTurn) {
        offA[u] = p.interleaved ? 2 * j * VEC : j * VEC;
        offB[u] = p.interleaved ? 2 * j * VEC + VEC : p.pairs + j * VEC;
        at[u] = tok * p.pairs + j * VEC;
      } else {
        offA[u] = 2 * j * VEC;
        offB[u] = offA[u] + VEC < p.d ? offA[u] + VEC : -1;
        at[u] = -1;
      }
      a[u] = *reinterpret_cast<const P*>(from + offA[u]);
      if (offB[u] >= 0) b[u] = *reinterpret_cast<const P*>(from + offB[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (!to[u]) continue;
      if (at[u] >= 0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          if (!p.interleaved || VEC == 1) {
            const float2 cs = sTurn[at[u] + e];
            const float x = asFloat(a[u].v[e]), y = asFloat(b[u].v[e]);
            a[u].v[e] = fromFloat<T>(x * cs.x - y * cs.y);
            b[u].v[e] = fromFloat<T>(x * cs.y + y * cs.x);
          } else if (e < VEC / 2) {                    // a vector of neighbours holds VEC / 2 whole pairs
            const float2 ca = sTurn[at[u] + e], cb = sTurn[at[u] + VEC / 2 + e];
            const float xa = asFloat(a[u].v[2 * e % VEC]), ya = asFloat(a[u].v[(2 * e + 1) % VEC]);
            const float xb = asFloat(b[u].v[2 * e % VEC]), yb = asFloat(b[u].v[(2 * e + 1) % VEC]);
            a[u].v[2 * e % VEC] = fromFloat<T>(xa * ca.x - ya * ca.y);
            a[u].v[(2 * e + 1) % VEC] = fromFloat<T>(xa * ca.y + ya * ca.x);
            b[u].v[2 * e % VEC] = fromFloat<T>(xb * cb.x - yb * cb.y);
            b[u].v[(2 * e + 1) % VEC] = fromFloat<T>(xb * cb.y + yb * cb.x);
          }
        }
      }
      *reinterpret_cast<P*>(to[u] + offA[u]) = a[u];
      if (offB[u] >= 0) *reinterpret_cast<P*>(to[u] + offB[u]) = b[u];
    }
  }
}

template <typename T, int VEC, bool CACHE>
int launch(RotArgs& a, cudaStream_t st) {
  // Tokens of a block: as many as give every thread kUnroll items, fewer while the grid has less than two blocks an SM,
  // and no more than shared memory has room for (48 KB without an opt-in).
  const long long rows = CACHE ? a.nQ + 2LL * a.nK : a.nQ, perToken = rows * ((a.d + 2 * VEC - 1) / (2 * VEC));
  long long tok = kThreads * kUnroll / perToken;
  const long long room = a.pairs > 0 ? 40960 / (a.pairs * (long long)sizeof(float2)) : kMaxTokens;
  const long long spread = a.tokens / (2LL * deviceSMs());
  if (tok > spread) tok = spread;
  if (tok > room) tok = room;
  if (tok > kMaxTokens) tok = kMaxTokens;
  if (tok < 1) tok = 1;
  a.tokensPerBlock = (int)tok;
  const long long grid = (a.tokens + tok - 1) / tok;
  rotary_kernel<T, VEC, CACHE><<<(unsigned)grid, kThreads, tok * a.pairs * sizeof(float2), st>>>(a);
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
  if (p->tokens < 0 || p->heads < 0 || p->d < 1 || p->d > 65536) return setError(LLC_ERR_ARGUMENT, "llc argument: rotary extents");
  if (!floatType(p->dtype)) return setError(LLC_ERR_UNSUPPORTED, "llc argument: rotary tensors must be f32, bf16 or f16");
  RotArgs a{};
  if (int rc = checkTurn("rotary", p->d, p->pairs, p->axes, p->sections, p->positions, p->pos_dtype, &a)) return rc;
  if (p->tokens == 0 || p->heads == 0) return LLC_OK;
  if (!p->x || !p->out || !p->positions || !p->inv_freq) return setError(LLC_ERR_ARGUMENT, "llc argument: rotary null operand");
  if (p->tokens > 0x7FFFFFFFLL || p->heads > 65536 || p->heads * p->d > (1LL << 26) || p->pairs > 4096) return setError(LLC_ERR_UNSUPPORTED, "llc argument: rotary too large");
  a.q = p->x; a.qOut = p->out; a.positions = p->positions; a.invFreq = p->inv_freq;
  a.qSt = p->x_st; a.qSh = p->x_sh; a.qoSt = p->o_st; a.qoSh = p->o_sh; a.posSa = p->pos_sa;
  a.tokens = p->tokens; a.nQ = (int)p->heads; a.d = (int)p->d; a.interleaved = p->interleaved != 0;
  const int64_t vec = 16 / dtypeBytes(p->dtype);
  const bool al = aligned16(p->x) && aligned16(p->out) && p->d % vec == 0 && p->pairs % vec == 0 && p->x_st % vec == 0 && p->x_sh % vec == 0 &&
                  p->o_st % vec == 0 && p->o_sh % vec == 0;
  return chooseType<false>(a, p->dtype, al, (cudaStream_t)stream);
}

extern "C" int llc_cuda_kv_append(const LlcKvAppendParams* p, void* stream) {
  if (!p) return setError(LLC_ERR_ARGUMENT, "llc argument: kv_append null parameter block");
  if (p->tokens < 0 || p->batch < 0 || p->heads < 0 || p->kv_heads < 1 || p->d < 1 || p->d > 65536 || p->num_pages < 0 || p->page_size < 1 || p->table_width < 0)
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
  if (p->tokens > 0x7FFFFFFFLL || p->batch > (1 << 20) || nq > 65536 || p->kv_heads > 65536 || (nq + 2 * p->kv_heads) * p->d > (1LL << 26) || p->pairs > 4096 ||
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
  if (nq) al = al && aligned16(p->q) && aligned16(p->q_out) && p->q_st % vec == 0 && p->q_sh % vec == 0 && p->qo_st % vec == 0 && p->qo_sh % vec == 0;
  for (int64_t s : {p->k_st, p->k_sh, p->v_st, p->v_sh, p->kc_sp, p->kc_sn, p->kc_sh, p->vc_sp, p->vc_sn, p->vc_sh}) al = al && s % vec == 0;
  return chooseType<true>(a, p->dtype, al, (cudaStream_t)stream);
}
