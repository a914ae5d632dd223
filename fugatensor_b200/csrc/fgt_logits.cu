// fgt_logits.cu — rules that edit logits before a token is chosen: penalties
// for tokens that occurred already, per-token biases, grammar masks.
#include "fgt_vocab.cuh"

namespace fgt {
namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 4096;             // tokens of a row that one CTA edits
constexpr unsigned kPrompt = 0x80000000u;  // a counter's top bit: the token is in the prompt

struct Rules {
  fgt_i64 rows, vocab, history, biases, words;
  Index tokens, lengths, prompt_lengths, bias_tokens;
  const float *repetition, *presence, *frequency, *bias;
  float repetition0, presence0, frequency0;
  const unsigned* allowed;
};

template <class T>
__global__ void __launch_bounds__(kThreads)
    adjust_slices(const typename T::S* __restrict__ logits, Rules r, fgt_i64 slices, typename T::S* __restrict__ out) {
  __shared__ unsigned count[kSlice];
  __shared__ float bias[kSlice];
  const fgt_i64 row = blockIdx.x / slices, v0 = blockIdx.x % slices * kSlice;
  for (int i = threadIdx.x; i < kSlice; i += kThreads) {
    count[i] = 0;
    bias[i] = 0.0f;
  }
  __syncthreads();
  if (r.tokens.p) {
    fgt_i64 n = r.lengths.p ? r.lengths[row] : r.history;
    n = n < 0 ? 0 : n > r.history ? r.history : n;
    const fgt_i64 np = r.prompt_lengths.p ? r.prompt_lengths[row] : 0;
    for (fgt_i64 i = threadIdx.x; i < n; i += kThreads) {
      const fgt_i64 t = r.tokens[row * r.history + i];
      if (t < v0 || t >= v0 + kSlice || t >= r.vocab) continue;
      if (i < np)
        atomicOr(&count[t - v0], kPrompt);
      else
        atomicAdd(&count[t - v0], 1u);
    }
  }
  if (threadIdx.x == 0 && r.bias)
    for (fgt_i64 k = 0; k < r.biases; ++k) {  // in the order of k
      const fgt_i64 t = r.bias_tokens[row * r.biases + k];
      if (t >= v0 && t < v0 + kSlice && t < r.vocab) bias[t - v0] = __fadd_rn(bias[t - v0], r.bias[row * r.biases + k]);
    }
  __syncthreads();
  const float rep = r.repetition ? r.repetition[row] : r.repetition0;
  const float pres = r.presence ? r.presence[row] : r.presence0;
  const float freq = r.frequency ? r.frequency[row] : r.frequency0;
  for (int i = threadIdx.x; i < kSlice; i += kThreads) {
    const fgt_i64 v = v0 + i;
    if (v >= r.vocab) return;
    float x = T::get(logits[row * r.vocab + v]);
    const unsigned c = count[i], made = c & ~kPrompt;
    if (c) x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    if (made) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)made)), pres);
    x = __fadd_rn(x, bias[i]);
    if (r.allowed && !(r.allowed[row * r.words + (v >> 5)] >> (v & 31) & 1)) x = __int_as_float(0xff800000);
    out[row * r.vocab + v] = T::put(x);
  }
}

}  // namespace
}  // namespace fgt

using namespace fgt;

extern "C" fgt_status fgt_adjust_logits(const fgt_adjust_logits_desc* d, const fgt_adjust_logits_buffers* b, void* stream) {
  return guarded_call("fgt_adjust_logits", [&] {
    require(d != nullptr && b != nullptr, "desc or buffers is NULL");
    require(is_float(d->dtype), "dtype must be f32, f16 or bf16");
    size_product(d->rows, d->vocab, "rows x vocab");
    const fgt_i64 words = (d->vocab + 31) / 32;
    check_buffer(b->logits, d->rows * d->vocab, "logits");
    check_buffer(b->out, d->rows * d->vocab, "out");
    if (b->tokens) {
      check_index_dtype(d->token_dtype, "tokens");
      check_buffer(b->tokens, size_product(d->rows, d->history, "tokens"), "tokens");
      require(d->history < kPrompt, "a history has at most 2^31 - 1 tokens");
      if (b->lengths || b->prompt_lengths) check_index_dtype(d->length_dtype, "lengths");
      if (b->lengths) check_buffer(b->lengths, d->rows, "lengths");
      if (b->prompt_lengths) check_buffer(b->prompt_lengths, d->rows, "prompt_lengths");
    } else {
      require(!b->lengths && !b->prompt_lengths, "lengths are given without tokens");
    }
    require((b->bias != nullptr) == (b->bias_tokens != nullptr), "bias and bias_tokens are given together");
    if (b->bias) {
      check_index_dtype(d->bias_dtype, "bias_tokens");
      check_buffer(b->bias_tokens, size_product(d->rows, d->biases, "bias_tokens"), "bias_tokens");
      check_buffer(b->bias, d->rows * d->biases, "bias");
    }
    if (b->repetition) check_buffer(b->repetition, d->rows, "repetition");
    if (b->presence) check_buffer(b->presence, d->rows, "presence");
    if (b->frequency) check_buffer(b->frequency, d->rows, "frequency");
    if (b->allowed) check_buffer(b->allowed, d->rows * words, "allowed");
    require(b->repetition || d->repetition > 0.0f, "repetition must be positive");
    if (d->rows * d->vocab == 0) return;
    check_pending();
    const Rules r{d->rows, d->vocab, d->history, d->biases, words,
                  Index{b->tokens, d->token_dtype == FGT_I64}, Index{b->lengths, d->length_dtype == FGT_I64},
                  Index{b->prompt_lengths, d->length_dtype == FGT_I64}, Index{b->bias_tokens, d->bias_dtype == FGT_I64},
                  b->repetition, b->presence, b->frequency, b->bias, d->repetition, d->presence, d->frequency,
                  b->allowed};
    const fgt_i64 slices = (d->vocab + kSlice - 1) / kSlice;
    const unsigned grid = blocks_for(size_product(d->rows, slices, "rows x vocab"), 1, "rows x vocab");
    for_dtype(d->dtype, [&](auto t) {
      using T = decltype(t);
      using S = typename T::S;
      adjust_slices<T><<<grid, kThreads, 0, (cudaStream_t)stream>>>((const S*)b->logits, r, slices, (S*)b->out);
    });
    cuda_check(cudaGetLastError(), "launch");
  });
}
