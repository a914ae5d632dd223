// fgt_embedding.cu — embedding lookup with scaling, and its gradient.
//
//   out[i, :]    = s * table[t_i, :]               (0 where t_i is outside [0, V))
//   dtable[v, :] = s * sum over {i : t_i = v} of dy[i, :], in the order of i
#include "fgt_vocab.cuh"

namespace fgt {
namespace {

constexpr int kThreads = 256;

template <class T>
__global__ void __launch_bounds__(kThreads)
    embedding_rows(const typename T::S* __restrict__ table, Index indices, fgt_i64 count, fgt_i64 vocab, fgt_i64 dim,
                   float scale, typename T::S* __restrict__ out) {
  const fgt_i64 row = blockIdx.x * (fgt_i64)(kThreads / 32) + threadIdx.x / 32;
  if (row >= count) return;
  const fgt_i64 t = indices[row];
  const bool in = t >= 0 && t < vocab;
  for (fgt_i64 c = threadIdx.x % 32; c < dim; c += 32)
    out[row * dim + c] = in ? T::put(__fmul_rn(T::get(table[t * dim + c]), scale)) : T::put(0.0f);
}

// One warp per table row and 32 columns: scans the indices in order.
template <class T>
__global__ void __launch_bounds__(kThreads)
    embedding_grad_scan(Index indices, fgt_i64 count, const typename T::S* __restrict__ dy, fgt_i64 vocab, fgt_i64 dim,
                        float scale, fgt_i64 padding, typename T::S* __restrict__ dtable) {
  const fgt_i64 row = blockIdx.x * (fgt_i64)(kThreads / 32) + threadIdx.x / 32;
  if (row >= vocab) return;
  const int lane = threadIdx.x % 32;
  for (fgt_i64 c0 = 0; c0 < dim; c0 += 256) {
    float acc[8] = {};
    for (fgt_i64 i0 = 0; i0 < count && row != padding; i0 += 32) {
      unsigned hits = __ballot_sync(~0u, i0 + lane < count && indices[i0 + lane] == row);
      for (; hits; hits &= hits - 1) {
        const fgt_i64 i = i0 + __ffs(hits) - 1;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const fgt_i64 c = c0 + k * 32 + lane;
          if (c < dim) acc[k] = __fadd_rn(acc[k], T::get(dy[i * dim + c]));
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const fgt_i64 c = c0 + k * 32 + lane;
      if (c < dim) dtable[row * dim + c] = T::put(__fmul_rn(acc[k], scale));
    }
  }
}

void check(const fgt_embedding_desc* d) {
  require(d != nullptr, "desc is NULL");
  check_index_dtype(d->index_dtype, "indices");
  require(is_float(d->dtype), "dtype must be f32, f16 or bf16");
  size_product(d->vocab, d->dim, "the table");
  size_product(d->count, d->dim, "indices x dim");
}

}  // namespace
}  // namespace fgt

using namespace fgt;

extern "C" fgt_status fgt_embedding(const fgt_embedding_desc* d, const void* table, const void* indices, void* out,
                                    void* stream) {
  return guarded_call("fgt_embedding", [&] {
    check(d);
    check_buffer(table, d->vocab * d->dim, "table");
    check_buffer(indices, d->count, "indices");
    check_buffer(out, d->count * d->dim, "out");
    if (d->count * d->dim == 0) return;
    check_pending();
    const unsigned grid = blocks_for(d->count, kThreads / 32, "indices");
    for_dtype(d->dtype, [&](auto t) {
      using T = decltype(t);
      using S = typename T::S;
      embedding_rows<T><<<grid, kThreads, 0, (cudaStream_t)stream>>>(
          (const S*)table, Index{indices, d->index_dtype == FGT_I64}, d->count, d->vocab, d->dim, d->scale, (S*)out);
    });
    cuda_check(cudaGetLastError(), "launch");
  });
}

extern "C" fgt_status fgt_embedding_grad_workspace(const fgt_embedding_desc* d, size_t* bytes) {
  return guarded_call("fgt_embedding_grad_workspace", [&] {
    require(bytes != nullptr, "bytes is NULL");
    check(d);
    *bytes = 0;
  });
}

extern "C" fgt_status fgt_embedding_grad(const fgt_embedding_desc* d, const void* indices, const void* dy, void* dtable,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  return guarded_call("fgt_embedding_grad", [&] {
    check(d);
    check_buffer(indices, d->count, "indices");
    check_buffer(dy, d->count * d->dim, "dy");
    check_buffer(dtable, d->vocab * d->dim, "dtable");
    if (d->vocab * d->dim == 0) return;
    check_pending();
    const unsigned grid = blocks_for(d->vocab, kThreads / 32, "vocab");
    for_dtype(d->dtype, [&](auto t) {
      using T = decltype(t);
      using S = typename T::S;
      embedding_grad_scan<T><<<grid, kThreads, 0, (cudaStream_t)stream>>>(
          Index{indices, d->index_dtype == FGT_I64}, d->count, (const S*)dy, d->vocab, d->dim, d->scale,
          d->padding_index, (S*)dtable);
    });
    cuda_check(cudaGetLastError(), "launch");
  });
}
