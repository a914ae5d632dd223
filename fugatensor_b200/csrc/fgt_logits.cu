// fgt_logits.cu — rules that edit logits before a token is chosen: penalties
// for tokens that occurred already, per-token biases, grammar masks.
//
// The work is a copy of the logits, bound by memory. What it needs beside them
// is how often each token of the vocabulary occurred in the row's history. A
// CTA edits a slice of a row: it counts its slice's tokens in shared memory
// (one 32-bit counter per token, cleared first), reading the row's whole
// history, and then streams its logits past the counters. A vector none of
// whose tokens occurred is copied as it is. The few tokens with a bias are done
// after the others, one thread each; longer lists of biases (kMany) are summed in
// shared memory, in their order.
// On B200 64 rows of 128000 bf16 with up to 4096 tokens, 32 biases and a mask
// take 18 us (a copy of them 9: the rest is a chain of loads and barriers), 384
// rows of 50021 f32 with up to 32768 tokens and 300 biases 55 us (a copy 24: the
// rest is instructions, half of them for the history, which every slice reads).
// Registers are what it is short of: three CTAs per SM leave 40 per thread, and
// four vectors of history in flight in place of two spill (73 us); two CTAs of
// larger slices read the history half as often but take 61 us.
#include <type_traits>

#include "fgt_vocab.cuh"

namespace fgt {
namespace {

constexpr int kThreads = 512;
constexpr int kBatch = 2;                  // vectors of logits per thread in flight, besides those at work
constexpr int kHistoryBatch = 2;           // vectors of tokens per thread in flight
constexpr int kLead = 8;                   // counters before a slice's first vector: a row's single values
constexpr int kListed = kThreads;          // biases per row that a slice's list has room for
constexpr unsigned kPrompt = 0x80000000u;  // a counter's top bits: the token is in the prompt,
constexpr unsigned kBiased = 0x40000000u;  // has a bias,
constexpr unsigned kTwice = 0x20000000u;   // has several

struct Rules {
  fgt_i64 rows, vocab, history, biases, words;
  Index tokens, lengths, prompt_lengths, bias_tokens;
  const float *repetition, *presence, *frequency, *bias;
  float repetition0, presence0, frequency0;
  const unsigned* allowed;
};

struct Listed {
  int token;
  float bias;
};

// For a token that occurred or has a bias. x / repetition is x times the rounded
// reciprocal (within 1.5 units of f32); the count's share, with the presence
// penalty, is one FMA, and a token that only has a bias is x * 1 - 0.
struct Penalty {
  float repetition, inverse, presence, frequency;
  __device__ __forceinline__ Penalty(float r, float p, float f)
      : repetition(r), inverse(1.0f / r), presence(p), frequency(f) {}
  __device__ __forceinline__ float operator()(float x, unsigned count) const {
    const unsigned made = count & ~(kPrompt | kBiased | kTwice);
    const bool occurred = count & ~(kBiased | kTwice);
    const float factor = x > 0.0f ? inverse : repetition, less = __fmaf_rn(frequency, (float)made, presence);
    return __fsub_rn(__fmul_rn(x, occurred ? factor : 1.0f), made ? less : 0.0f);
  }
};

// One instruction where a token is outside the slice: d is its distance from the slice's first.
FGT_DEV void count_token(unsigned counter, unsigned d, unsigned span) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.u32 p, %1, %2;\n\t@p red.shared.add.u32 [%0], 1;\n\t}" ::"r"(counter + d * 4), "r"(d), "r"(span) : "memory");
}
FGT_DEV void mark_token(unsigned counter, unsigned d, unsigned span) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.u32 p, %1, %2;\n\t@p red.shared.or.b32 [%0], %3;\n\t}" ::"r"(counter + d * 4), "r"(d), "r"(span), "r"(kPrompt) : "memory");
}

template <class T, bool kWide, bool kMany>  // kWide: the tokens are 64-bit; kMany: more than kListed biases per row
__global__ void __launch_bounds__(kThreads, kMany ? 1 : 3)
    adjust_slices(const typename T::S* __restrict__ logits, Rules r, int slices, int slice_vecs, typename T::S* __restrict__ out) {
  using E = typename T::S;
  constexpr int N = Vec<T>::kN;
  extern __shared__ __align__(16) unsigned count[];  // [kLead + slice_vecs * N + N], then the list or (kMany) as many sums
  grid_wait();
  grid_release();
  const fgt_i64 row = blockIdx.x / slices;
  const int slice = (int)(blockIdx.x % slices), vocab = (int)r.vocab;
  // the row: `lead` single values (the first slice's), aligned vectors, single values (the last slice's)
  const fgt_i64 e0 = row * r.vocab;
  const int lead = min((int)((N - e0 % N) % N), vocab), nvec = (vocab - lead) / N;
  const int first = min(slice * slice_vecs, nvec), end = slice + 1 == slices ? nvec : min(first + slice_vecs, nvec);
  const int base = lead + first * N;  // the token of the slice's first vector: its counter is kLead
  const int low = slice == 0 ? 0 : base, high = slice + 1 == slices ? vocab : lead + end * N;
  const E* const x = logits + e0;
  E* const y = out + e0;
  const uint4* const in = reinterpret_cast<const uint4*>(x + lead);

  const unsigned* const allowed = r.allowed ? r.allowed + row * r.words : nullptr;
  uint4 u[kBatch];
  unsigned bits[kBatch];  // of vector u: bit e set = its value e may be chosen
  const uint4* src = in + (first + threadIdx.x);  // this thread's next vectors, kThreads apart,
  int t0 = lead + (first + threadIdx.x) * N;      // and the first one's token
  int left = end - first - threadIdx.x;           // one more vector for every kThreads of them
  auto fetch = [&](int b, int ahead) {            // vector `ahead + b` from here into slot b, if there is one
    if (left <= (ahead + b) * kThreads) return;
    u[b] = __ldcs(src + (ahead + b) * kThreads);
    if (!allowed) return;
    const int t = t0 + (ahead + b) * (kThreads * N);
    bits[b] = __funnelshift_r(allowed[t >> 5], (t & 31) + N > 32 ? allowed[(t >> 5) + 1] : 0u, t & 31);
  };
#pragma unroll
  for (int b = 0; b < kBatch; ++b) fetch(b, 0);  // on their way while the history is counted

  // The row's history: `before` single tokens, then 16-byte vectors of `per` tokens, then single tokens.
  constexpr int per = kWide ? 2 : 4, size = 16 / per;
  const char* const history = static_cast<const char*>(r.tokens.p) + row * r.history * size;
  const int before = min((int)((16 - ((uintptr_t)history & 15)) & 15) / size, (int)r.history);
  uint4 h[kHistoryBatch];
  const uint4* past = reinterpret_cast<const uint4*>(history + before * size) + threadIdx.x;
  if (r.tokens.p) {  // before the lengths are known
    const int vectors = ((int)r.history - before) / per;
#pragma unroll
    for (int b = 0; b < kHistoryBatch; ++b)
      if ((int)threadIdx.x + b * kThreads < vectors) h[b] = __ldcs(past + b * kThreads);
  }

  // The slice's biases in their order: each warp appends its own after those of the warps before.
  const int counters = (kLead + slice_vecs * N + N + 3) / 4 * 4;
  Listed* const list = reinterpret_cast<Listed*>(count + counters);
  __shared__ int s_listed[kThreads / 32];
  const int biases = r.bias ? (int)r.biases : 0, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const bool listed = !kMany && biases > 0;
  int bias_token = -1;
  float bias_value = 0.0f;
  if (listed) {
    if ((int)threadIdx.x < biases) {
      const fgt_i64 v = r.bias_tokens[row * r.biases + threadIdx.x];
      bias_value = r.bias[row * r.biases + threadIdx.x];
      if (v >= low && v < high) bias_token = (int)v;
    }
    const int n = __popc(__ballot_sync(~0u, bias_token >= 0));
    if (lane == 0) s_listed[warp] = n;
  }

  Penalty penalty(1.0f, 0.0f, 0.0f);
  int n = 0, prompt = 0;
  if (r.tokens.p) {
    penalty = Penalty(r.repetition ? r.repetition[row] : r.repetition0, r.presence ? r.presence[row] : r.presence0,
                      r.frequency ? r.frequency[row] : r.frequency0);
    fgt_i64 len = r.lengths.p ? r.lengths[row] : r.history;
    n = (int)(len < 0 ? 0 : len > r.history ? r.history : len);
    len = r.prompt_lengths.p ? r.prompt_lengths[row] : 0;
    prompt = (int)(len < 0 ? 0 : len > n ? n : len);
  }
  float* const sums = reinterpret_cast<float*>(count + counters);
  const bool counting = r.tokens.p || biases > 0;
  if (counting) {
    uint4 *const clear = reinterpret_cast<uint4*>(count), *const clear_sums = reinterpret_cast<uint4*>(sums);
    for (int i = threadIdx.x; i < (kLead + (end - first) * N + N) / 4; i += kThreads) {
      clear[i] = make_uint4(0, 0, 0, 0);
      if (kMany) clear_sums[i] = make_uint4(0, 0, 0, 0);
    }
  }
  __syncthreads();
  int all_listed = 0;
  if (listed) {
    const unsigned in_slice = __ballot_sync(~0u, bias_token >= 0);
    int at = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      at += w < warp ? s_listed[w] : 0;
      all_listed += s_listed[w];
    }
    if (bias_token >= 0) {
      list[at + __popc(in_slice & ((1u << lane) - 1))] = Listed{bias_token, bias_value};
      unsigned* c = count + (bias_token - base + kLead);
      if (atomicOr(c, kBiased) & kBiased) atomicOr(c, kTwice);
    }
  }
  if constexpr (kMany) {
    // Every warp adds up the biases of its share of the slice's tokens and walks
    // the row's list for that, so a token's biases add in their order and the
    // work grows with the list's length: 64 rows of 128000 bf16 with 2500 biases
    // take 84 us, with 128000 4 ms; 2^20 for one row 5.3 ms, 90 ms where all are
    // one token's (85 ns from one to the next).
    constexpr int kAhead = 4, kWarps = kThreads / 32;  // loads in flight per lane
    const fgt_i64 from = row * r.biases;
    for (int k0 = lane; k0 - lane < biases; k0 += 32 * kAhead) {
      fgt_i64 v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) v[u] = k0 + 32 * u < biases ? r.bias_tokens[from + k0 + 32 * u] : -1;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const bool mine = v[u] >= low && v[u] < high && (int)v[u] % kWarps == warp;
        const float b = mine ? r.bias[from + k0 + 32 * u] : 0.0f;
        const int at = (int)v[u] - base + kLead;
        for (unsigned todo = __ballot_sync(~0u, mine); todo; todo &= todo - 1) {
          if (lane == __ffs(todo) - 1) {
            sums[at] = __fadd_rn(sums[at], b);
            atomicOr(count + at, kBiased);
          }
          __syncwarp();
        }
      }
    }
  }
  if (n > 0) {
    const unsigned span = (unsigned)(high - low);
    const unsigned counter = (unsigned)__cvta_generic_to_shared(count + (low - base + kLead));
    auto prompted = [&](int t) { mark_token(counter, (unsigned)(t - low), span); };
    auto generated = [&](int t) { count_token(counter, (unsigned)(t - low), span); };
    auto visit = [&](int t, int i) { i < prompt ? prompted(t) : generated(t); };
    auto narrow = [](fgt_i64 t) { return t >> 31 ? -1 : (int)t; };  // -1: none that a vocabulary has
    auto single = [&](int i) {
      visit(kWide ? narrow(reinterpret_cast<const fgt_i64*>(history)[i]) : reinterpret_cast<const int*>(history)[i], i);
    };
    const int vectors = n > before ? (n - before) / per : 0, after = before + vectors * per;
    if (threadIdx.x < min(before, n)) single(threadIdx.x);
    if (after + threadIdx.x < n) single(after + threadIdx.x);  // fewer than `per`
    int given = prompt - before - (int)threadIdx.x * per;  // tokens of the prompt from this thread's next vector on
    constexpr int step = kHistoryBatch * kThreads;
    for (int ahead = vectors - (int)threadIdx.x; ahead > 0; ahead -= step, given -= step * per, past += step) {
#pragma unroll
      for (int b = 0; b < kHistoryBatch; ++b) {
        if (ahead <= b * kThreads) break;
        const uint4 t = h[b];
        if (ahead > step + b * kThreads) h[b] = __ldcs(past + step + b * kThreads);
        const int g = given - b * (kThreads * per);
        if (kWide) {
          const int t0 = narrow((fgt_i64)t.x | (fgt_i64)(int)t.y << 32), t1 = narrow((fgt_i64)t.z | (fgt_i64)(int)t.w << 32);
          g > 0 ? prompted(t0) : generated(t0);
          g > 1 ? prompted(t1) : generated(t1);
        } else if (g <= 0) {
          generated((int)t.x);
          generated((int)t.y);
          generated((int)t.z);
          generated((int)t.w);
        } else if (g >= per) {
          prompted((int)t.x);
          prompted((int)t.y);
          prompted((int)t.z);
          prompted((int)t.w);
        } else {  // the prompt ends in this vector
          prompted((int)t.x);
          g > 1 ? prompted((int)t.y) : generated((int)t.y);
          g > 2 ? prompted((int)t.z) : generated((int)t.z);
          generated((int)t.w);
        }
      }
    }
  }
  __syncthreads();

  // one value by itself: the row's single values, and tokens with a bias
  auto edited = [&](int v, bool has_bias, float bias) {
    if (allowed && !(allowed[v >> 5] >> (v & 31) & 1)) return T::put(__int_as_float(0xff800000));
    const float f = penalty(T::get(x[v]), counting ? count[v - base + kLead] : 0);
    return T::put(has_bias ? __fadd_rn(f, bias) : f);
  };
  // A token with a bias is stored after the others, which do without biases.
  // Where a token has several entries, each of their threads adds all of them in
  // their order: they store the same value.
  E biased_value = 0;
  if (bias_token >= 0) {
    float sum = bias_value;
    if (count[bias_token - base + kLead] & kTwice) {
      sum = 0.0f;
      for (int j = 0; j < all_listed; ++j)
        if (list[j].token == bias_token) sum = __fadd_rn(sum, list[j].bias);
    }
    biased_value = edited(bias_token, true, sum);
  }

  constexpr unsigned kMinusInf = sizeof(E) == 4 ? 0xff800000u : std::is_same<T, F16>::value ? 0xfc00u : 0xff80u;
  constexpr int step = kBatch * kThreads;
  uint4* to = reinterpret_cast<uint4*>(y + lead) + (first + threadIdx.x);
  const uint4* counts = reinterpret_cast<const uint4*>(count + kLead) + threadIdx.x * (N / 4);
  for (; left > 0; left -= step, src += step, to += step, counts += step * (N / 4), t0 += step * N) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (left <= b * kThreads) break;
      uint4 now = u[b];
      const unsigned may = bits[b];
      fetch(b, kBatch);
      if (r.tokens.p) {
        const uint4* c = counts + b * (kThreads * (N / 4));
        uint4 n[N / 4];
        unsigned some = 0;
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
          n[k] = c[k];
          some |= n[k].x | n[k].y | n[k].z | n[k].w;
        }
        if (some) {
          float v[N];
          Vec<T>::unpack(now, v);
#pragma unroll
          for (int k = 0; k < N / 4; ++k) {
            // all of the vector's values: a vote on each, to skip those that occurred in no lane's, costs more than
            // it saves (384 x 50021, history 32768: 52.6 us against 53.7 f32, 45.8 against 48.3 bf16; with 300
            // tokens 28.7 and 19.5 both ways)
            v[4 * k] = penalty(v[4 * k], n[k].x);
            v[4 * k + 1] = penalty(v[4 * k + 1], n[k].y);
            v[4 * k + 2] = penalty(v[4 * k + 2], n[k].z);
            v[4 * k + 3] = penalty(v[4 * k + 3], n[k].w);
          }
          now = Vec<T>::pack(v);
        }
      }
      if (allowed) {
        unsigned w[4] = {now.x, now.y, now.z, now.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (sizeof(E) == 4) {
            w[k] = may >> k & 1 ? w[k] : kMinusInf;
          } else {
            const unsigned keep = (may >> (2 * k) & 1 ? 0xffffu : 0) | (may >> (2 * k + 1) & 1 ? 0xffff0000u : 0);
            w[k] = (w[k] & keep) | (kMinusInf * 0x10001u & ~keep);
          }
        }
        now = make_uint4(w[0], w[1], w[2], w[3]);
      }
      __stcs(to + b * kThreads, now);
    }
  }

  if (slice == 0 && threadIdx.x < lead) y[threadIdx.x] = edited(threadIdx.x, false, 0.0f);
  const int rest = lead + nvec * N + threadIdx.x;
  if (slice + 1 == slices && rest < vocab) y[rest] = edited(rest, false, 0.0f);
  if (!biases) return;
  __syncthreads();  // the values without their biases are written
  if constexpr (kMany) {
    for (int v = low + (int)threadIdx.x; v < high; v += kThreads)
      if (count[v - base + kLead] & kBiased) y[v] = edited(v, true, sums[v - base + kLead]);
  } else if (bias_token >= 0) {
    y[bias_token] = biased_value;
  }
}

// Slices of a row: at most kSliceTokens tokens (three CTAs of 512 threads fit an
// SM with their counters), and more of them where the rows are too few to give
// every SM three CTAs, down to one vector per thread. Every slice reads the
// row's whole history, so no more than that: 384 rows of 50021 f32 with 24576
// tokens of history each took 61 us with 4 slices, 87 with 8.
constexpr int64_t kSliceTokens = 16384;

int slices_for(int64_t rows, int64_t vocab, int64_t per_vec) {
  const int64_t most = std::max<int64_t>(1, vocab / (per_vec * kThreads)), least = (vocab + kSliceTokens - 1) / kSliceTokens;
  return (int)std::max(least, std::min(most, (3 * 148 + rows - 1) / rows));
}

}  // namespace
}  // namespace fgt

using namespace fgt;

extern "C" fgt_status fgt_adjust_logits(const fgt_adjust_logits_desc* d, const fgt_adjust_logits_buffers* b, void* stream) {
  return guarded_call("fgt_adjust_logits", [&] {
    require(d != nullptr && b != nullptr, "desc or buffers is NULL");
    require(is_float(d->dtype), "dtype must be f32, f16 or bf16");
    size_product(d->rows, d->vocab, "rows x vocab");
    require(d->vocab <= 1 << 30, "vocab must be at most 2^30");
    require(d->biases < (INT64_C(1) << 30), "a row has fewer than 2^30 biases");
    const fgt_i64 words = (d->vocab + 31) / 32;
    check_buffer(b->logits, d->rows * d->vocab, "logits");
    check_buffer(b->out, d->rows * d->vocab, "out");
    if (b->tokens) {
      check_index_dtype(d->token_dtype, "tokens");
      check_buffer(b->tokens, size_product(d->rows, d->history, "tokens"), "tokens");
      require(d->history < (int64_t)kTwice, "a history has fewer than 2^29 tokens");
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
    for_dtype(d->dtype, [&](auto t) {
      using T = decltype(t);
      using E = typename T::S;
      constexpr int N = Vec<T>::kN;
      const int slices = slices_for(d->rows, d->vocab, N);
      const int64_t nvec = d->vocab / N, slice_vecs = (nvec + slices - 1) / slices;
      const bool biased = b->bias && d->biases > 0, many = biased && d->biases > kListed;
      const size_t counters = b->tokens || biased ? (size_t)(kLead + slice_vecs * N + N + 3) / 4 * 16 : 0;
      const size_t smem = many ? 2 * counters : counters + (biased ? (size_t)d->biases * sizeof(Listed) : 0);
      const bool wide = b->tokens && d->token_dtype == FGT_I64;
      auto kernel = many ? (wide ? adjust_slices<T, true, true> : adjust_slices<T, false, true>)
                         : (wide ? adjust_slices<T, true, false> : adjust_slices<T, false, false>);
      active_clusters(kernel, kThreads, smem, 1);  // leave for the shared memory
      launch(Launch{(cudaStream_t)stream, programmatic((cudaStream_t)stream)}, kernel,
             blocks_for(size_product(d->rows, slices, "rows x vocab"), 1, "rows x vocab"), kThreads, smem, 1, (const E*)b->logits,
             r, slices, (int)slice_vecs, (E*)b->out);
    });
  });
}
