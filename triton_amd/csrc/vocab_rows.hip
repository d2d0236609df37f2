// Operators over rows of logits of a whole vocabulary: log probabilities of given tokens with entropy and top alternatives, the
// distillation loss against a teacher's top logits, and the gradients of both.
#include "row_math.h"

namespace tk {
namespace {

constexpr float NEG_INF = -__builtin_inff();

__device__ __forceinline__ float block_max(float v, float* buf) {
  __syncthreads();
  buf[threadIdx.x] = v;
  __syncthreads();
  for (int d = 128; d; d >>= 1) {
    if ((int)threadIdx.x < d) buf[threadIdx.x] = fmaxf(buf[threadIdx.x], buf[threadIdx.x + d]);
    __syncthreads();
  }
  return buf[0];
}

// Order of a logit as an unsigned number; the two zeros are one value.
__device__ __forceinline__ uint32_t order_of(float f) {
  const uint32_t u = f32_bits(f + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int64_t index_at(const void* p, int is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

// m = the largest logit, ln s = ln sum exp((x - m) / t), and the entropy of a row.
struct RowSums {
  float m, log_s, entropy;
  bool bad, empty;
};
template <int DT>
__device__ RowSums row_sums(const void* row, int V, float inv_t, float* buf) {
  float m = NEG_INF;
  for (int v = threadIdx.x; v < V; v += 256) m = fmaxf(m, RowType<DT>::load(row, v));
  m = block_max(m, buf);
  const float ref = m == NEG_INF ? 0.f : m;
  float s = 0.f, e = 0.f;
  for (int v = threadIdx.x; v < V; v += 256) {
    const float d = (RowType<DT>::load(row, v) - ref) * inv_t, p = expf(d);
    s += p;
    e = fmaf(p, fmaxf(d, -200.f), e);
  }
  s = block_sum<256>(s, buf);
  e = block_sum<256>(e, buf);
  RowSums r;
  r.m = m;
  r.log_s = logf(s);
  r.bad = !(s >= 0.f) || m == __builtin_inff();
  r.empty = !r.bad && s == 0.f;
  r.entropy = r.bad ? __builtin_nanf("") : r.empty ? 0.f : r.log_s - e / s;
  return r;
}

template <int DT>
__global__ __launch_bounds__(256) void token_logprobs_kernel(tk_vocab_desc d, float inv_t) {
  __shared__ float buf[256];
  __shared__ unsigned long long best;
  for (int t = blockIdx.x; t < d.n_rows; t += gridDim.x) {
    const void* row = static_cast<const char*>(d.logits) + (int64_t)t * d.logits_stride_m * RowType<DT>::BYTES;
    const RowSums r = row_sums<DT>(row, d.vocab, inv_t, buf);
    if (threadIdx.x == 0) {
      const int64_t at = index_at(d.tokens, d.tokens_i64, t);
      float lp = 0.f;
      if (at >= 0 && at < d.vocab) lp = r.bad ? __builtin_nanf("") : r.empty ? NEG_INF : (RowType<DT>::load(row, at) - r.m) * inv_t - r.log_s;
      d.logprobs[t] = lp;
      d.entropy[t] = r.entropy;
      if (d.stats) {
        d.stats[t] = r.m;
        d.stats[d.n_rows + t] = r.bad ? __builtin_nanf("") : r.log_s;
      }
    }
    // the next one in the order (larger logit, then lower index), one after the other
    unsigned long long last = ~0ull;
    for (int j = 0; j < d.k; ++j) {
      __syncthreads();
      if (threadIdx.x == 0) best = 0;
      __syncthreads();
      unsigned long long mine = 0;
      for (int v = threadIdx.x; v < d.vocab; v += 256) {
        const unsigned long long key = (unsigned long long)order_of(RowType<DT>::load(row, v)) << 32 | (uint32_t)~v;
        if (key < last && key > mine) mine = key;
      }
      atomicMax(&best, mine);
      __syncthreads();
      last = best;
      const int at = (int)~(uint32_t)last;
      if (threadIdx.x == 0) {
        const int64_t o = (int64_t)t * d.k + j;
        d.top_indx[o] = r.bad ? -1 : at;
        d.top_logprobs[o] = r.bad ? __builtin_nanf("") : r.empty ? NEG_INF : (RowType<DT>::load(row, at) - r.m) * inv_t - r.log_s;
      }
    }
    __syncthreads();
  }
}

template <int DT>
__global__ __launch_bounds__(256) void token_logprobs_backward_kernel(tk_vocab_desc d, float inv_t) {
  for (int t = blockIdx.x; t < d.n_rows; t += gridDim.x) {
    const void* row = static_cast<const char*>(d.logits) + (int64_t)t * d.logits_stride_m * RowType<DT>::BYTES;
    void* out = static_cast<char*>(d.d_logits) + (int64_t)t * d.d_logits_stride_m * RowType<DT>::BYTES;
    const int64_t at = index_at(d.tokens, d.tokens_i64, t);
    const float g_lp = d.d_logprobs && at >= 0 && at < d.vocab ? d.d_logprobs[t * d.d_logprobs_stride] : 0.f;
    const float g_h = d.d_entropy ? d.d_entropy[t * d.d_entropy_stride] : 0.f;
    const float m = d.stats[t], log_s = d.stats[d.n_rows + t], h = d.entropy[t];
    const bool zero = (g_lp == 0.f && g_h == 0.f) || log_s == NEG_INF;  // (a sum of nothing)
    for (int v = threadIdx.x; v < d.vocab; v += 256) {
      const float lp = (RowType<DT>::load(row, v) - m) * inv_t - log_s, p = expf(lp);
      float g = -p * (g_lp + g_h * (fmaxf(lp, -200.f) + h));
      if (v == at) g += g_lp;
      if (lp != lp) g = lp;
      RowType<DT>::store(out, v, zero ? 0.f : g * inv_t);
    }
  }
}

// The teacher's entry j of row t: its index, or -1 where it carries no weight, and its logit.
template <int DT>
__device__ __forceinline__ int teacher_entry(const tk_vocab_desc& d, int t, int j, float* q) {
  *q = load_any(d.teacher_logits, d.teacher_dtype, (int64_t)t * d.teacher_stride_m + j);
  const int64_t i = index_at(d.teacher_indx, d.teacher_indx_i64, (int64_t)t * d.teacher_indx_stride_m + j);
  return i < 0 || i >= d.vocab || *q == NEG_INF ? -1 : (int)i;
}

template <int DT>
__global__ __launch_bounds__(256) void distill_kernel(tk_vocab_desc d, float inv_t) {
  __shared__ float buf[256];
  for (int t = blockIdx.x; t < d.n_rows; t += gridDim.x) {
    const void* row = static_cast<const char*>(d.logits) + (int64_t)t * d.logits_stride_m * RowType<DT>::BYTES;
    const RowSums r = row_sums<DT>(row, d.vocab, inv_t, buf);
    float qm = NEG_INF, q, qs = 0.f, loss = 0.f;
    int bad = 0;
    for (int j = threadIdx.x; j < d.n_teacher; j += 256)
      if (teacher_entry<DT>(d, t, j, &q) >= 0) {
        qm = fmaxf(qm, q);
        bad |= q != q;
      }
    qm = block_max(qm, buf);
    bad = __syncthreads_or(bad) || qm == __builtin_inff();
    for (int j = threadIdx.x; j < d.n_teacher; j += 256)
      if (teacher_entry<DT>(d, t, j, &q) >= 0) qs += expf((q - qm) * inv_t);
    qs = block_sum<256>(qs, buf);
    const float log_qs = bad ? __builtin_nanf("") : logf(qs);
    for (int j = threadIdx.x; j < d.n_teacher; j += 256) {
      const int at = teacher_entry<DT>(d, t, j, &q);
      if (at < 0) continue;
      const float la = (q - qm) * inv_t - log_qs, a = expf(la);
      const float lp = r.bad ? __builtin_nanf("") : r.empty ? NEG_INF : (RowType<DT>::load(row, at) - r.m) * inv_t - r.log_s;
      if (a != 0.f) loss = fmaf(a, la - lp, loss);
    }
    loss = block_sum<256>(loss, buf);
    if (threadIdx.x == 0) {
      d.loss[t] = loss;
      if (d.stats) {
        d.stats[t] = r.m;
        d.stats[d.n_rows + t] = r.bad ? __builtin_nanf("") : r.log_s;
      }
      if (d.teacher_stats) {
        d.teacher_stats[t] = bad ? __builtin_nanf("") : qm;
        d.teacher_stats[d.n_rows + t] = log_qs;
      }
    }
    __syncthreads();
  }
}

template <int DT>
__global__ __launch_bounds__(256) void distill_backward_kernel(tk_vocab_desc d, float inv_t) {
  __shared__ float a[TK_VOCAB_MAX_TEACHER];
  __shared__ int at[TK_VOCAB_MAX_TEACHER];
  for (int t = blockIdx.x; t < d.n_rows; t += gridDim.x) {
    const void* row = static_cast<const char*>(d.logits) + (int64_t)t * d.logits_stride_m * RowType<DT>::BYTES;
    void* out = static_cast<char*>(d.d_logits) + (int64_t)t * d.d_logits_stride_m * RowType<DT>::BYTES;
    const float m = d.stats[t], log_s = d.stats[d.n_rows + t], qm = d.teacher_stats[t], log_qs = d.teacher_stats[d.n_rows + t];
    const float g = d.d_loss ? d.d_loss[t * d.d_loss_stride] : 0.f;
    const bool zero = g == 0.f || log_s == NEG_INF || qm == NEG_INF;  // (sums of nothing)
    __syncthreads();
    for (int j = threadIdx.x; j < d.n_teacher; j += 256) {
      float q;
      at[j] = teacher_entry<DT>(d, t, j, &q);
      a[j] = expf((q - qm) * inv_t - log_qs);
    }
    __syncthreads();
    for (int v = threadIdx.x; v < d.vocab; v += 256) {
      float p = expf((RowType<DT>::load(row, v) - m) * inv_t - log_s);
      for (int j = 0; j < d.n_teacher; ++j)
        if (at[j] == v) p -= a[j];
      RowType<DT>::store(out, v, zero ? 0.f : qm != qm ? qm : p * g * inv_t);
    }
  }
}

int32_t check(const tk_vocab_desc* d, const char* who) {
  if (!d) return fail(TK_ERR_INVALID, "%s: null descriptor", who);
  if (d->n_rows < 0 || d->vocab <= 0) return fail(TK_ERR_INVALID, "%s: bad sizes %d x %d", who, d->n_rows, d->vocab);
  if (!(d->temperature > 0.f) || d->temperature == __builtin_inff()) return fail(TK_ERR_INVALID, "%s: the temperature must be positive and finite", who);
  if (!is_row_dtype(d->logits_dtype)) return fail(TK_ERR_UNSUPPORTED, "%s: logits are fp32, bf16 or fp16", who);
  if (d->n_rows && !d->logits) return fail(TK_ERR_INVALID, "%s: null logits", who);
  return TK_OK;
}

int32_t check_teacher(const tk_vocab_desc* d, const char* who) {
  if (d->n_teacher < 0) return fail(TK_ERR_INVALID, "%s: bad number of teacher entries %d", who, d->n_teacher);
  if (d->n_teacher > TK_VOCAB_MAX_TEACHER) return fail(TK_ERR_UNSUPPORTED, "%s: %d teacher entries a row, at most %d", who, d->n_teacher, TK_VOCAB_MAX_TEACHER);
  if (!is_row_dtype(d->teacher_dtype)) return fail(TK_ERR_UNSUPPORTED, "%s: teacher logits are fp32, bf16 or fp16", who);
  if (d->n_rows && d->n_teacher && (!d->teacher_logits || !d->teacher_indx)) return fail(TK_ERR_INVALID, "%s: null teacher", who);
  return TK_OK;
}

unsigned rows_grid(int n) { return n < 65536 ? n : 65536; }

}  // namespace
}  // namespace tk

using namespace tk;

#define TK_VOCAB_LAUNCH(kernel)                                                                                                              \
  do {                                                                                                                                       \
    auto f = d->logits_dtype == TK_F32 ? kernel<TK_F32> : d->logits_dtype == TK_BF16 ? kernel<TK_BF16> : kernel<TK_F16>;                        \
    hipLaunchKernelGGL(f, dim3(rows_grid(d->n_rows)), dim3(256), 0, static_cast<hipStream_t>(stream), *d, 1.0f / d->temperature);             \
  } while (0)

extern "C" int64_t tk_vocab_workspace_bytes(int32_t n_rows, int32_t vocab, int32_t k) { return 0; }

extern "C" int32_t tk_token_logprobs(const tk_vocab_desc* d, tk_stream_t stream) {
  if (int32_t e = check(d, "tk_token_logprobs")) return e;
  if (d->k < 0 || d->k > d->vocab) return fail(TK_ERR_INVALID, "tk_token_logprobs: %d alternatives of %d", d->k, d->vocab);
  if (d->k > TK_VOCAB_MAX_TOP || (d->k && d->vocab > TK_VOCAB_MAX_TOP_COLUMNS))
    return fail(TK_ERR_UNSUPPORTED, "tk_token_logprobs: at most %d alternatives, of at most %d columns", TK_VOCAB_MAX_TOP, TK_VOCAB_MAX_TOP_COLUMNS);
  if (d->n_rows == 0) return TK_OK;
  if (!d->tokens || !d->logprobs || !d->entropy || (d->k && (!d->top_logprobs || !d->top_indx))) return fail(TK_ERR_INVALID, "tk_token_logprobs: null pointer");
  TK_VOCAB_LAUNCH(token_logprobs_kernel);
  return check_launch("token_logprobs_kernel");
}

extern "C" int32_t tk_token_logprobs_backward(const tk_vocab_desc* d, tk_stream_t stream) {
  if (int32_t e = check(d, "tk_token_logprobs_backward")) return e;
  if (d->n_rows == 0) return TK_OK;
  if (!d->tokens || !d->entropy || !d->stats || !d->d_logits) return fail(TK_ERR_INVALID, "tk_token_logprobs_backward: null pointer");
  TK_VOCAB_LAUNCH(token_logprobs_backward_kernel);
  return check_launch("token_logprobs_backward_kernel");
}

extern "C" int32_t tk_distill_topk(const tk_vocab_desc* d, tk_stream_t stream) {
  if (int32_t e = check(d, "tk_distill_topk")) return e;
  if (int32_t e = check_teacher(d, "tk_distill_topk")) return e;
  if (d->n_rows == 0) return TK_OK;
  if (!d->loss) return fail(TK_ERR_INVALID, "tk_distill_topk: null pointer");
  TK_VOCAB_LAUNCH(distill_kernel);
  return check_launch("distill_kernel");
}

extern "C" int32_t tk_distill_topk_backward(const tk_vocab_desc* d, tk_stream_t stream) {
  if (int32_t e = check(d, "tk_distill_topk_backward")) return e;
  if (int32_t e = check_teacher(d, "tk_distill_topk_backward")) return e;
  if (d->n_rows == 0) return TK_OK;
  if (!d->stats || !d->teacher_stats || !d->d_logits) return fail(TK_ERR_INVALID, "tk_distill_topk_backward: null pointer");
  TK_VOCAB_LAUNCH(distill_backward_kernel);
  return check_launch("distill_backward_kernel");
}
