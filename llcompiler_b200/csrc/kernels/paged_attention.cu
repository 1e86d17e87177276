// Attention of new tokens over a paged key / value cache: argument checks, the choice of kernel, and the kernel of plain
// multiply-adds that takes every type, head size, page size and stride.
#include "paged_attention.cuh"

namespace llc {
long long pagedDecodeWorkspace(const PagedArgs& p, bool wide);
int pagedDecode(const PagedArgs& p, bool wide, void* workspace, long long bytes, cudaStream_t st);
long long pagedChunkWorkspace(const PagedArgs& p);
int pagedChunk(const PagedArgs& p, int doneRows, void* workspace, long long bytes, cudaStream_t st);

namespace {

constexpr int kWarps = 8;
constexpr int kMaxD = 256;

// One block per (token, head): the warps take the visible keys in turn, each with a running maximum and sum, lane l holding
// elements l, l + 32, ... of the row, and meet in shared memory at the end.  out = sum_w o_w 2^(m_w - m) / sum_w l_w 2^(m_w - m).
// Bound: the latency of a key at a time and the instructions of its dot product; every head of a group reads the keys anew.  16 sequences
// of up to 4096 keys, 32 heads of 128 in bf16: 572 us, where the tensor-core kernels take 38; it is for what those do not take.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) paged_rows_kernel(const PagedArgs p) {
  __shared__ float sM[kWarps], sL[kWarps], sO[kWarps][kMaxD];
  __shared__ int sSeq;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = blockIdx.x / p.heads;
  const int h = (int)(blockIdx.x - t * p.heads);
  if (warp == 0) {
    // sequences that end at or before row t, 32 ends at a time
    int c = 0;
    for (int i = lane; i < p.batch; i += 32) c += p.qStart[i + 1] <= t;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) sSeq = c;
  }
  __syncthreads();
  const int b = sSeq;
  if (b >= p.batch || t < p.qStart[b]) return;         // a row of nobody
  const Sequence s = sequenceOf(p, b);
  if (t - s.begin >= s.n) return;                      // none of its rows: starts that do not grow would name places past the table
  const long long pos = s.len - s.n + (t - s.begin);
  const long long lo = pos + 1 - p.window > 0 ? pos + 1 - p.window : 0, first = p.sinks < lo ? p.sinks : lo;
  const long long keys = pos < 0 ? 0 : first + (pos + 1 - lo);
  const int g = h / p.group;
  constexpr int kPer = kMaxD / 32;
  float q[kPer], o[kPer], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + 32 * i;
    q[i] = e < p.d ? loadAs(p.q, t * p.qSt + h * p.qSh + e, p.dtype) * p.scaleLog2 : 0.f;
    o[i] = 0.f;
  }
  for (long long idx = warp; idx < keys; idx += kWarps) {
    const long long j = idx < first ? idx : idx - first + lo;
    const long long page = pageOf(p, b, j / p.pageSize), slot = j % p.pageSize;
    if (page < 0 && lane == 0 && p.badPages) atomicAdd(p.badPages, 1);
    const T* k = reinterpret_cast<const T*>(p.k) + page * p.kcSp + slot * p.kcSn + g * p.kcSh;
    const T* v = reinterpret_cast<const T*>(p.v) + page * p.vcSp + slot * p.vcSn + g * p.vcSh;
    float dot = 0.f, vv[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      const bool in = page >= 0 && e < p.d;
      dot = fmaf(in ? (float)k[e] : 0.f, q[i], dot);
      vv[i] = in ? (float)v[e] : 0.f;
    }
    dot = warpSum(dot);
    const float mNew = fmaxf(m, dot);
    const float base = mNew == -INFINITY ? 0.f : mNew;
    const float keep = exp2f(m - base), w = exp2f(dot - base);
    m = mNew;
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = fmaf(w, vv[i], o[i] * keep);
  }
  if (lane == 0) { sM[warp] = m; sL[warp] = l; }
#pragma unroll
  for (int i = 0; i < kPer; ++i) sO[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float top = sM[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sM[w]);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f, f[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) { f[w] = exp2f(sM[w] - base); sum += sL[w] * f[w]; }
  const float divisor = divisorOf(sum, top, pos >= 0);
  for (int e = threadIdx.x; e < p.d; e += kWarps * 32) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) x += sO[w][e] * f[w];
    storeAs(p.out, t * p.oSt + h * p.oSh + e, p.dtype, x / divisor);
  }
}

int pagedRows(const PagedArgs& a, cudaStream_t st) {
  const long long grid = a.tokens * a.heads;
  if (grid > 0x7FFFFFFFLL) return setError(LLC_ERR_UNSUPPORTED, "llc argument: paged_attention too many rows");
  if (a.dtype == LLC_FLOAT32) paged_rows_kernel<float><<<(unsigned)grid, kWarps * 32, 0, st>>>(a);
  else if (a.dtype == LLC_BFLOAT16) paged_rows_kernel<__nv_bfloat16><<<(unsigned)grid, kWarps * 32, 0, st>>>(a);
  else paged_rows_kernel<__half><<<(unsigned)grid, kWarps * 32, 0, st>>>(a);
  LLC_LAUNCH_CHECK("paged_rows_kernel");
  return LLC_OK;
}

int checkAndFill(const LlcPagedAttentionParams* p, PagedArgs* a) {
  if (!p) return setError(LLC_ERR_ARGUMENT, "llc argument: paged_attention null parameter block");
  if (p->tokens < 0 || p->batch < 0 || p->heads < 1 || p->kv_heads < 1 || p->d < 1 || p->max_q < 0 || p->num_pages < 0 || p->page_size < 1 || p->table_width < 0)
    return setError(LLC_ERR_ARGUMENT, "llc argument: paged_attention extents");
  if (p->heads % p->kv_heads) return setError(LLC_ERR_ARGUMENT, "llc argument: paged_attention heads must be a multiple of kv_heads");
  if (p->window < 0 || p->sinks < 0) return setError(LLC_ERR_ARGUMENT, "llc argument: paged_attention negative window or sinks");
  if (p->dtype != LLC_FLOAT32 && p->dtype != LLC_BFLOAT16 && p->dtype != LLC_FLOAT16)
    return setError(LLC_ERR_UNSUPPORTED, "llc argument: paged_attention tensors must be f32, bf16 or f16");
  if (p->d > kMaxD) return setError(LLC_ERR_UNSUPPORTED, "llc argument: paged_attention head size above 256");
  if (p->tokens > 0x7FFFFFFFLL || p->batch > (1 << 20) || p->heads > 65536 || p->num_pages > 0x7FFFFFFFLL || p->page_size > (1 << 20) || p->table_width > 0x7FFFFFFFLL)
    return setError(LLC_ERR_UNSUPPORTED, "llc argument: paged_attention too large");
  if (p->table_width * p->page_size > 0x7FFFFF00LL) return setError(LLC_ERR_UNSUPPORTED, "llc argument: paged_attention table reaches past 2^31 slots");
  a->q = p->q; a->k = p->k_cache; a->v = p->v_cache; a->out = p->out;
  a->table = p->page_table; a->qStart = p->q_start; a->kvLen = p->kv_len; a->badPages = p->bad_pages;
  a->qSt = p->q_st; a->qSh = p->q_sh; a->oSt = p->o_st; a->oSh = p->o_sh;
  a->kcSp = p->kc_sp; a->kcSn = p->kc_sn; a->kcSh = p->kc_sh; a->vcSp = p->vc_sp; a->vcSn = p->vc_sn; a->vcSh = p->vc_sh;
  // the stride of a dim of one element says nothing: one that fits every kernel
  if (p->tokens == 1) a->qSt = a->oSt = 0;
  if (p->heads == 1) a->qSh = a->oSh = 0;
  if (p->kv_heads == 1) a->kcSh = a->vcSh = (p->d + 7) / 8 * 8;
  if (p->num_pages == 1) a->kcSp = a->vcSp = (p->d + 7) / 8 * 8;
  a->tableS0 = p->table_s0; a->tokens = p->tokens; a->numPages = p->num_pages; a->pageSize = p->page_size;
  a->reach = (int)(p->table_width * p->page_size);
  a->maxQ = p->max_q < p->tokens ? p->max_q : p->tokens;
  a->window = p->window > 0 && p->window < a->reach ? (int)p->window : a->reach + 1;
  a->sinks = p->sinks < a->reach ? (int)p->sinks : a->reach;
  a->batch = (int)p->batch; a->heads = (int)p->heads; a->kvHeads = (int)p->kv_heads; a->group = (int)(p->heads / p->kv_heads);
  a->d = (int)p->d; a->dtype = p->dtype;
  a->scaleLog2 = p->scale * 1.4426950408889634f;
  return LLC_OK;
}

// What the tensor-core kernels take: the types, head sizes and pages they have tiles for, and 16-byte steps everywhere.
bool tensorTypes(const PagedArgs& a) {
  bool ok = a.dtype != LLC_FLOAT32 && (a.d == 64 || a.d == 128) && a.pageSize >= 16 && (a.pageSize & (a.pageSize - 1)) == 0 && a.numPages > 0 && a.reach > 0 &&
            (long long)a.batch * a.kvHeads <= 0x7FFFFFFFLL && a.tokens * a.group < 0x7FFFFF00LL;
  for (long long s : {a.qSt, a.qSh, a.oSt, a.oSh}) ok = ok && s % 8 == 0;
  for (long long s : {a.kcSp, a.kcSn, a.kcSh, a.vcSp, a.vcSn, a.vcSh}) ok = ok && s % 8 == 0 && s > 0 && s < (1LL << 38);
  for (const void* x : {a.q, a.k, a.v, (const void*)a.out}) ok = ok && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  return ok;
}

// Rows of a sequence up to which the decode kernel takes it.  A call whose sequences all have at most 32 rows runs there alone; beside
// longer chunks of other sequences it takes the sequences of single tokens (16 rows, which leave two CTAs on an SM, or 32 for large groups).
int decodeRows(const PagedArgs& a) {
  const long long rows = a.maxQ * a.group;
  if (rows <= 32) return rows <= 16 ? 16 : 32;
  // few sequences of few keys fit beside the chunks' tiles, and launches less are worth more.  One kernel against both, us: nine sequences of up to
  // 2048 keys, one of them a single token 32 / 43; 16 single tokens and two chunks of 40 over 1000 keys 24 / 41; 60 single tokens and four chunks of
  // 100 over 1000 keys (2 key heads) 21 / 35; eight single tokens over 3500 keys and eight chunks of 64 over 1500 55 / 70.  At the border the
  // other way round: 12 single tokens and four chunks of 200 over 4000 keys 124 / 115; past it 24 single tokens and eight chunks of 128 over 2000
  // keys (256 pairs) 103 / 88, three single tokens and a chunk of 256 over 16000 keys 184 / 181.
  const long long seen = (long long)a.window + a.sinks < a.reach ? (long long)a.window + a.sinks : a.reach;   // keys that a token can see
  if (a.batch == 1 || (seen <= 4096 && a.batch * a.kvHeads <= deviceSMs())) return 0;
  return a.group <= 16 ? 16 : a.group <= 32 ? 32 : 0;
}

}  // namespace
}  // namespace llc

using namespace llc;

extern "C" int64_t llc_cuda_paged_attention_workspace(const LlcPagedAttentionParams* p) {
  PagedArgs a{};
  if (checkAndFill(p, &a) != LLC_OK || !tensorTypes(a) || a.tokens == 0 || a.batch == 0 || a.maxQ == 0) return 0;
  // the two kernels of a mixed batch run one after the other and share it
  const int few = decodeRows(a);
  const int64_t d = few ? pagedDecodeWorkspace(a, few == 32) : 0, c = a.maxQ * a.group > few ? pagedChunkWorkspace(a) : 0;
  return d > c ? d : c;
}

extern "C" int llc_cuda_paged_attention(const LlcPagedAttentionParams* p, void* stream) {
  PagedArgs a{};
  if (int rc = checkAndFill(p, &a)) return rc;
  if (a.tokens == 0 || a.batch == 0 || a.maxQ == 0) return LLC_OK;
  if (!p->q || !p->out || !p->q_start || !p->kv_len || (a.reach > 0 && !p->page_table) || (p->num_pages > 0 && (!p->k_cache || !p->v_cache)))
    return setError(LLC_ERR_ARGUMENT, "llc argument: paged_attention null operand");
  if (reinterpret_cast<uintptr_t>(p->workspace) & 15) return setError(LLC_ERR_ARGUMENT, "llc argument: paged_attention workspace must be 16-byte aligned");
  const cudaStream_t st = (cudaStream_t)stream;
  if (!tensorTypes(a)) return pagedRows(a, st);
  const int few = decodeRows(a);
  if (few) {
    if (int rc = pagedDecode(a, few == 32, p->workspace, p->workspace_bytes, st)) return rc;
  }
  return a.maxQ * a.group > few ? pagedChunk(a, few, p->workspace, p->workspace_bytes, st) : LLC_OK;
}
