// fgt_loss.cu — cross-entropy over the vocabulary, and its gradient.
//
// With lse = log(sum_v exp(x_v)) of a row x of logits and its target t:
//   loss = lse - (1 - e) x_t - (e / V) sum_v x_v + z lse^2
//   dx_v = g (softmax_v (1 + 2 z lse) - (1 - e) [v = t] - e / V)
#include "fgt_vocab.cuh"

namespace fgt {
namespace {

constexpr int kThreads = 256;

struct Row {
  fgt_i64 rows, vocab, ignore;
  float smoothing, z, grad_scale;
  int reduction;
};

__device__ __forceinline__ float block_sum(float v, float* s) {
  for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(~0u, v, m);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s[threadIdx.x / 32] = v;
  __syncthreads();
  float t = 0.0f;
  for (int w = 0; w < kThreads / 32; ++w) t += s[w];
  return t;
}

__device__ __forceinline__ float block_max(float v, float* s) {
  for (int m = 16; m; m >>= 1) v = fgt_fmax(v, __shfl_xor_sync(~0u, v, m));
  __syncthreads();
  if (threadIdx.x % 32 == 0) s[threadIdx.x / 32] = v;
  __syncthreads();
  float t = s[0];
  for (int w = 1; w < kThreads / 32; ++w) t = fgt_fmax(t, s[w]);
  return t;
}

// MEAN: the number of counted rows, at least 1 (whole numbers below 2^24 are exact in f32; above, rounded once).
__global__ void __launch_bounds__(1024) loss_count(Index targets, Row r, float* counted) {
  __shared__ int s_n;
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  int n = 0;
  for (fgt_i64 i = threadIdx.x; i < r.rows; i += blockDim.x) {
    const fgt_i64 t = targets[i];
    n += t != r.ignore && t >= 0 && t < r.vocab;
  }
  n = __reduce_add_sync(~0u, n);
  if (threadIdx.x % 32 == 0) atomicAdd(&s_n, n);
  __syncthreads();
  if (threadIdx.x == 0) *counted = (float)(s_n > 0 ? s_n : 1);
}

template <class T>
__global__ void __launch_bounds__(kThreads)
    loss_rows(const typename T::S* __restrict__ logits, Index targets, Row r, const float* seed, const float* counted,
              float* losses, typename T::S* __restrict__ dlogits) {
  __shared__ float s[kThreads / 32];
  const fgt_i64 row = blockIdx.x;
  const typename T::S* x = logits + row * r.vocab;
  const fgt_i64 t = targets[row];
  if (t == r.ignore || t < 0 || t >= r.vocab) {
    if (losses && threadIdx.x == 0) losses[row] = 0.0f;
    if (dlogits)
      for (fgt_i64 c = threadIdx.x; c < r.vocab; c += kThreads) dlogits[row * r.vocab + c] = T::put(0.0f);
    return;
  }
  float m = __int_as_float(0xff800000), all = 0.0f, sum = 0.0f;
  for (fgt_i64 c = threadIdx.x; c < r.vocab; c += kThreads) m = fgt_fmax(m, T::get(x[c]));
  m = block_max(m, s);
  for (fgt_i64 c = threadIdx.x; c < r.vocab; c += kThreads) {
    const float v = T::get(x[c]);
    sum += expf(v - m);
    all += v;
  }
  sum = block_sum(sum, s);
  const float lse = m + logf(sum), share = r.smoothing / (float)r.vocab;
  if (losses) {
    all = block_sum(all, s);
    if (threadIdx.x == 0) {
      float l = lse - (1.0f - r.smoothing) * T::get(x[t]);
      if (r.smoothing != 0.0f) l -= share * all;
      if (r.z != 0.0f) l += r.z * lse * lse;
      losses[row] = l;
    }
  }
  if (!dlogits) return;
  float g = r.grad_scale;
  if (seed) g *= seed[r.reduction == FGT_LOSS_NONE ? row : 0];
  if (r.reduction == FGT_LOSS_MEAN) g /= *counted;
  const float k = r.z != 0.0f ? 1.0f + 2.0f * r.z * lse : 1.0f;
  for (fgt_i64 c = threadIdx.x; c < r.vocab; c += kThreads) {
    float d = expf(T::get(x[c]) - m) / sum * k - share;
    if (c == t) d -= 1.0f - r.smoothing;
    dlogits[row * r.vocab + c] = T::put(g * d);
  }
}

// SUM / MEAN: row losses added in f64, in a fixed order.
__global__ void __launch_bounds__(kThreads) loss_total(const float* losses, fgt_i64 rows, const float* counted, float* loss) {
  __shared__ double s[kThreads];
  double v = 0.0;
  for (fgt_i64 i = threadIdx.x; i < rows; i += kThreads) v += losses[i];
  s[threadIdx.x] = v;
  for (int h = kThreads / 2; h; h /= 2) {
    __syncthreads();
    if (threadIdx.x < h) s[threadIdx.x] += s[threadIdx.x + h];
  }
  if (threadIdx.x == 0) *loss = (float)(counted ? s[0] / *counted : s[0]);
}

void check(const fgt_cross_entropy_desc* d) {
  require(d != nullptr, "desc is NULL");
  check_index_dtype(d->target_dtype, "targets");
  require(is_float(d->dtype), "dtype must be f32, f16 or bf16");
  require(d->reduction >= FGT_LOSS_NONE && d->reduction <= FGT_LOSS_MEAN, "unknown reduction");
  require(d->label_smoothing >= 0.0f && d->label_smoothing <= 1.0f, "label_smoothing must be in [0, 1]");
  require(d->z_loss >= 0.0f && d->z_loss < 3.4e38f, "z_loss must be finite and not negative");
  require(d->vocab > 0, "vocab must be positive");
  size_product(d->rows, d->vocab, "rows x vocab");
  require(d->rows <= 0x7fffffff, "rows is too large for one launch");
}

// counted rows (one f32, padded), then the row losses that SUM / MEAN add up
size_t workspace_for(const fgt_cross_entropy_desc* d) {
  return d->reduction == FGT_LOSS_NONE ? 0 : 256 + (size_t)((d->rows * 4 + 255) / 256 * 256);
}

}  // namespace
}  // namespace fgt

using namespace fgt;

extern "C" fgt_status fgt_cross_entropy_workspace(const fgt_cross_entropy_desc* d, size_t* bytes) {
  return guarded_call("fgt_cross_entropy_workspace", [&] {
    require(bytes != nullptr, "bytes is NULL");
    check(d);
    *bytes = workspace_for(d);
  });
}

extern "C" fgt_status fgt_cross_entropy(const fgt_cross_entropy_desc* d, const void* logits, const void* targets,
                                        const float* seed, float* loss, void* dlogits, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  return guarded_call("fgt_cross_entropy", [&] {
    check(d);
    check_buffer(logits, d->rows * d->vocab, "logits");
    check_buffer(targets, d->rows, "targets");
    require(loss != nullptr || dlogits != nullptr, "neither loss nor dlogits is asked for");
    if (loss) check_buffer(loss, 1, "loss");
    if (dlogits) check_buffer(dlogits, d->rows * d->vocab, "dlogits");
    if (seed) check_buffer(seed, 1, "seed");
    const size_t need = workspace_for(d);
    require(workspace_bytes >= need, "workspace of " + std::to_string(workspace_bytes) + " bytes is smaller than the " +
                                         std::to_string(need) + " bytes needed", FGT_ERR_WORKSPACE);
    require(need == 0 || (workspace && (uintptr_t)workspace % 256 == 0),
            "workspace must be a 256-byte aligned device buffer", FGT_ERR_WORKSPACE);
    check_pending();
    const cudaStream_t st = (cudaStream_t)stream;
    const Row r{d->rows, d->vocab, d->ignore_index, d->label_smoothing, d->z_loss, d->grad_scale, d->reduction};
    const Index tg{targets, d->target_dtype == FGT_I64};
    float* counted = d->reduction == FGT_LOSS_MEAN ? (float*)workspace : nullptr;
    float* losses = !loss ? nullptr : d->reduction == FGT_LOSS_NONE ? loss : (float*)((char*)workspace + 256);
    if (counted) loss_count<<<1, 1024, 0, st>>>(tg, r, counted);
    if (d->rows > 0)
      for_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        using S = typename T::S;
        loss_rows<T><<<(unsigned)d->rows, kThreads, 0, st>>>((const S*)logits, tg, r, seed, counted, losses, (S*)dlogits);
      });
    if (loss && d->reduction != FGT_LOSS_NONE) loss_total<<<1, kThreads, 0, st>>>(losses, d->rows, counted, loss);
    cuda_check(cudaGetLastError(), "launch");
  });
}
