// fgt_loss.cu — cross-entropy over the vocabulary, and its gradient.
//
// With lse = log(sum_v exp(x_v)) of a row x of logits and its target t:
//   loss = lse - (1 - e) x_t - (e / V) sum_v x_v + z lse^2
//   dx_v = g (softmax_v (1 + 2 z lse) - (1 - e) [v = t] - e / V)
#include <cfloat>

#include "fgt_vocab.cuh"

namespace fgt {
namespace {

struct Row {
  fgt_i64 rows, vocab, ignore;
  float smoothing, z, grad_scale;
  int reduction;
  __device__ __forceinline__ bool counts(fgt_i64 t) const { return t != ignore && t >= 0 && t < vocab; }
};

// Exponentials are taken as 2^(x log2(e) - c) with c a whole number near the
// largest x log2(e): the product and the difference are one FMA, and partial
// sums with different c are brought together by exact powers of two. A factor
// below 2^-126 is flushed to 0, so a sum that has grown large gives its exponent
// to c first (settle): what is lost is below 2^-80 of the row's sum. The row's
// sum of exponentials is 2^c s, so lse = (c + log2(s)) ln 2. Rows that leave
// f32's range that way (overflow where the first values do not show the
// largest, values near the type's lowest, NaN), and rows so far from zero that
// not every whole number is an f32 value, are computed as 2^((x - m) log2(e))
// with m the maximum.
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
constexpr float kNegInf = -__builtin_huge_valf();

FGT_DEV float reference(float m) { return rintf(__fmul_rn(fmaxf(m, -1e30f), kLog2e)); }

// 2^((x + a) log2(e) + b) of two values, two f32 lanes per instruction
// (ex2.approx: 2 units of f32; results below the normals flush to 0).
FGT_DEV float2 both(float v) { return make_float2(v, v); }
template <bool kWhole> struct Exponent {
  float2 minus_c;
  __device__ __forceinline__ explicit Exponent(float c) : minus_c(both(-c)) {}
  __device__ __forceinline__ float2 operator()(float2 x) const {
    const float2 y = kWhole ? __ffma2_rn(x, both(kLog2e), minus_c) : __fmul2_rn(__fadd2_rn(x, minus_c), both(kLog2e));
    return make_float2(fgt_ex2_approx(y.x), fgt_ex2_approx(y.y));
  }
};

// ------------------------------------------------------- counted rows -----
// MEAN divides by the number of counted rows. Blocks of kCountRows rows are
// counted apart, and whoever needs the number adds the blocks up.
constexpr int kCountThreads = 1024, kCountRows = 8 * kCountThreads;

__global__ void __launch_bounds__(kCountThreads) loss_count(Index targets, Row r, int* counted, unsigned* ticket) {
  __shared__ int s_n;
  grid_wait();
  grid_release();
  if (threadIdx.x == 0) {
    s_n = 0;
    if (blockIdx.x == 0) *ticket = 0;
  }
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int u = 0; u < kCountRows / kCountThreads; ++u) {
    const fgt_i64 i = blockIdx.x * (fgt_i64)kCountRows + u * kCountThreads + threadIdx.x;
    n += i < r.rows && r.counts(targets[i]);
  }
  n = __reduce_add_sync(~0u, n);
  if (threadIdx.x % 32 == 0 && n) atomicAdd(&s_n, n);
  __syncthreads();
  if (threadIdx.x == 0) counted[blockIdx.x] = s_n;
}

// The number of counted rows (at least 1) for every lane of a full warp; whole
// numbers below 2^24 are exact in f32, larger ones rounded once. Without
// `counted` (few rows) the warp counts by itself.
constexpr fgt_i64 kFewRows = 1024;
__device__ __forceinline__ float counted_rows(const int* counted, const Index& targets, const Row& r) {
  fgt_i64 n = 0;
  if (counted) {
    const fgt_i64 blocks = (r.rows + kCountRows - 1) / kCountRows;
    for (fgt_i64 i = threadIdx.x % 32; i < blocks; i += 32) n += counted[i];
  } else {
#pragma unroll 8
    for (int i = threadIdx.x % 32; i < (int)r.rows; i += 32) n += r.counts(targets[i]);
  }
#pragma unroll
  for (int m = 16; m; m >>= 1) n += __shfl_xor_sync(~0u, n, m);
  return (float)(n > 0 ? n : 1);
}

// SUM / MEAN: row losses added in f64 in a fixed order, blocks of kCountRows
// by one CTA each and the blocks' sums by the CTA that finishes last.
__global__ void __launch_bounds__(kCountThreads)
    loss_total(const float* losses, Index targets, Row r, const int* counted, double* sums, unsigned* ticket, float* loss) {
  __shared__ double s[kCountThreads / 32];
  __shared__ bool s_last;
  grid_wait();
  grid_release();
  auto block_sum = [&](double v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(~0u, v, m);
    __syncthreads();
    if (threadIdx.x % 32 == 0) s[threadIdx.x / 32] = v;
    __syncthreads();
    v = s[threadIdx.x % 32];
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(~0u, v, m);
    return v;
  };
  double v = 0.0;
#pragma unroll
  for (int u = 0; u < kCountRows / kCountThreads; ++u) {
    const fgt_i64 i = blockIdx.x * (fgt_i64)kCountRows + u * kCountThreads + threadIdx.x;
    if (i < r.rows) v += losses[i];
  }
  v = block_sum(v);
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) {
      sums[blockIdx.x] = v;
      __threadfence();
      s_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
      __threadfence();
    }
    __syncthreads();
    if (!s_last) return;
    v = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += kCountThreads) v += __ldcg(sums + i);
    v = block_sum(v);
  }
  if (threadIdx.x < 32) {
    const float n = r.reduction == FGT_LOSS_MEAN ? counted_rows(counted, targets, r) : 1.0f;
    if (threadIdx.x == 0) *loss = (float)(v / n);
  }
}

// -------------------------------------------------------------- the rows ---
// Persistent groups of threads (a warp, a CTA, or a cluster of CTAs, by the
// row's length) walk the rows. A row is read twice, for the sum and for the
// gradient: the second reading comes from L2, since the rows at work hold about
// 40 MB in all (shape_for). Every thread copies its own vectors into a small
// ring in shared memory (cp.async), kStages - 1 batches ahead of its work, and
// that stream runs on from the first pass into the second and into the next
// row: neither the exchange of sums nor the writes stop the reads. A thread
// reads only what it copied itself, so the ring needs no barrier; one barrier
// per row makes the warps' sums known to the group.
// Rows of an odd vocabulary start anywhere: a row is its aligned vectors and up
// to 2 (N - 1) single values, one for each of the group's first threads.
// Bound by memory for f32 and long rows, by instructions (two exponentials a
// value, and about 300 instructions per warp and row) for 16-bit and short
// ones. Calls in a row on B200: 4096 x 32000 f32, loss alone, 87 us (0.92 of a
// copy's rate); 2048 x 128000 f32 with the gradient 387 us (0.83); 8192 x 128000
// bf16 777 us (0.82) under the power cap's clock, 683 before it sets in; 8192 x
// 32000 bf16 196 to 204 us (0.8); 2048 x 50021 f16 100 us (0.63). Rows held in
// registers, shared by a cluster, took 1250 us for the bf16 case (each phase
// waits for the one before); a ring of whole row slices per cluster 1350 to 3400.
// The second attempt reads a row twice more, one vector per thread at a time and
// outside the ring. Where it meets every row (normal logits with a deviation of
// 30, or a sixteenth of the columns at -1e4) these take 177, 560, 1085, 300 and
// 150 us; a few columns at -1e4 at the end of an odd vocabulary, the single
// values, 145 us in place of 113 for 2048 x 50021 f16.
enum Group { kWarp, kCta, kCluster };
constexpr int kBatch = 4, kStages = 3;  // 192 bytes per thread: 1024 threads keep 128 KB in flight per SM
constexpr int kWarpGroups = 4;          // warps of a CTA that has a row per warp

// The sum of exponentials is 2^c s with a whole c, else e^c s (c = -inf where s =
// 0); the sum of (e / V) x, each by itself: that of x overflows where a few columns
// are masked with the type's lowest value.
struct Stat {
  float c, s, all;
};

// A large s gives its exponent to c. At a join the factor of a smaller c is 0
// from 2^-127 on, and s must not be what would have made up for it: below 2^30,
// and with 8192 threads at most to a row, all that is lost is 2^-83, while the
// largest c's own s is 2^-0.5 or more. Settled once more, the row's s leaves g / s
// a normal number. Where c + e is no f32 value s becomes infinite, which calls for
// the second attempt; infinities and NaN stay.
constexpr float kSettled = 1073741824.0f;  // 2^30
constexpr float kWholes = 16777216.0f;     // 2^24: below, every whole number is an f32 value
FGT_DEV void settle(Stat& a) {
  if (!(a.s >= kSettled)) return;
  const unsigned bits = __float_as_uint(a.s);
  const float e = (float)((int)(bits >> 23) - 127), c = __fadd_rn(a.c, e);
  const bool exact = __fsub_rn(c, a.c) == e && bits < 0x7f800000u;
  a.s = __uint_as_float(exact ? (bits & 0x7fffffu) | 0x3f800000u : 0x7f800000u);
  a.c = exact ? c : a.c;
}

// The statistics of a warp's lanes joined; every lane gets the result.
template <bool kAll> __device__ __forceinline__ Stat warp_join(Stat a, bool whole) {
  const float c = fgt_redux_max(a.c), d = __fsub_rn(a.c, c == kNegInf ? 0.0f : c);
  float s = __fmul_rn(a.s, fgt_ex2_approx(whole ? d : __fmul_rn(d, kLog2e)));
#pragma unroll
  for (int k = 16; k; k >>= 1) {
    s += __shfl_xor_sync(~0u, s, k);
    if (kAll) a.all += __shfl_xor_sync(~0u, a.all, k);
  }
  return Stat{c, s, a.all};
}

template <class T, Group G, int kThreads, bool kAll>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
    loss_rows(const typename T::S* __restrict__ logits, Index targets, Row r, int per_cta, const float* __restrict__ seed,
              const int* __restrict__ counted, float* losses, typename T::S* __restrict__ dlogits) {
  using E = typename T::S;
  constexpr int N = Vec<T>::kN;
  constexpr int warps = kThreads / 32, threads = G == kWarp ? 32 : kThreads;  // of the CTA; of a row in it
  constexpr int kStep = kBatch * threads;
  extern __shared__ uint4 ring[];  // [kStages][kBatch][kThreads]
  __shared__ Stat s_stat[2][G == kCluster ? 8 * warps : warps];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int cta = G == kCluster ? (int)fgt_cluster_rank() : 0, ctas = G == kCluster ? (int)cluster_size() : 1;
  const int me = G == kWarp ? lane : threadIdx.x;  // this thread's place in its group's part of a row
  const fgt_i64 step = G == kWarp ? (fgt_i64)gridDim.x * warps : gridDim.x / ctas;
  const int vocab = (int)r.vocab;
  grid_wait();
  grid_release();
  if (G == kCluster) fgt_cluster_sync();  // every CTA has started before another writes to it

  const float g_all = r.grad_scale * (seed && r.reduction != FGT_LOSS_NONE ? seed[0] : 1.0f) /
                      (r.reduction == FGT_LOSS_MEAN ? counted_rows(counted, targets, r) : 1.0f);
  // a row: `lead` single values, aligned vectors, then single values again
  auto lead_of = [&](fgt_i64 q) { return min((int)((N - (q * r.vocab) % N) % N), vocab); };
  auto end_of = [&](int lead) { return min((cta + 1) * per_cta, (vocab - lead) / N); };
  auto target = [&](fgt_i64 q) { return q < r.rows ? targets[q] : r.ignore; };
  const int first = cta * per_cta;  // vectors [first, end) of a row are this CTA's

  // The stream: the vectors of every counted row, twice where a gradient is
  // wanted, kBatch per thread at a time and kStages - 1 batches ahead.
  const int passes = dlogits ? 2 : 1;
  fgt_i64 ahead = (G == kWarp ? blockIdx.x * (fgt_i64)warps + warp : blockIdx.x / ctas) - step, t_ahead = target(ahead + step);
  const uint4 *from = nullptr, *src = nullptr;  // this thread's first vector of the row, its next one
  int part = 0, left = 0, pass = passes - 1;    // the group's vectors of the row; those still to be copied
  constexpr unsigned kStage = kBatch * kThreads * 16;
  const unsigned mine = (unsigned)__cvta_generic_to_shared(ring + threadIdx.x);
  unsigned slot = mine;
  auto advance = [&]() {
    if (left <= 0) {
      if (++pass < passes) {
        src = from;
        left = part;
      } else {
        pass = 0;
        bool live;
        do {
          ahead += step;
          if (ahead >= r.rows) break;
          live = r.counts(t_ahead);
          t_ahead = target(ahead + step);
          const int lead = lead_of(ahead);
          part = end_of(lead) - first;
          src = from = reinterpret_cast<const uint4*>(logits + ahead * r.vocab + lead) + (first + me);
        } while (!live || part <= 0);
        left = ahead < r.rows ? part : 0;
        if (!left) pass = passes - 1;  // the rows are through
      }
    }
    if (left >= kStep) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) fgt_cp_async<16>(slot + b * kThreads * 16, src + b * threads);
    } else {
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (me + b * threads < left) fgt_cp_async<16>(slot + b * kThreads * 16, src + b * threads);
    }
    fgt_cp_commit();
    src += kStep;
    left -= kStep;
    slot = slot == mine + (kStages - 1) * kStage ? mine : slot + kStage;
  };
  for (int k = 0; k < kStages - 1; ++k) advance();
  int st = 0;
  // f(slot, vector) for this thread's vectors of a pass, kBatch per turn; turn() after each
  auto each = [&](int vectors, auto f, auto turn) {
    for (int n = vectors; n > 0; n -= kStep) {
      advance();
      fgt_cp_wait<kStages - 1>();
      const uint4* x = ring + st * (kBatch * kThreads) + threadIdx.x;
      if (n >= kStep) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) f(b, x[b * kThreads]);
      } else {
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
          if (me + b * threads < n) f(b, x[b * kThreads]);
      }
      turn();
      st = st + 1 == kStages ? 0 : st + 1;
    }
  };
  const float smoothed = r.smoothing / (float)r.vocab;

  fgt_i64 row = G == kWarp ? blockIdx.x * (fgt_i64)warps + warp : blockIdx.x / ctas;
  int parity = 0;
  // what a row needs besides its vectors is read a row ahead: nothing waits for it
  const bool seeds = r.reduction == FGT_LOSS_NONE && seed;
  struct Extra {
    fgt_i64 t;
    int lead, single;  // the group's first threads have one of the single values each
    float x_single, x_t, g;
  };
  auto extra = [&](fgt_i64 q, fgt_i64 t) {
    Extra x{t, 0, -1, kNegInf, 0.0f, g_all};
    if (q >= r.rows) return x;
    x.lead = lead_of(q);
    const int nvec = (vocab - x.lead) / N, singles = vocab - nvec * N;
    if (cta == 0 && me < singles) x.single = me < x.lead ? me : me + nvec * N;
    if (x.single >= 0) x.x_single = T::get(logits[q * r.vocab + x.single]);
    if (r.counts(t)) x.x_t = T::get(logits[q * r.vocab + t]);
    if (seeds) x.g = r.grad_scale * seed[q];
    return x;
  };
  Extra next = extra(row, target(row));
  fgt_i64 t_next = target(row + step);
  for (; row < r.rows; row += step) {
    const Extra now = next;
    next = extra(row + step, t_next);
    t_next = target(row + 2 * step);
    E* const dx = dlogits + row * r.vocab;
    uint4* const out = reinterpret_cast<uint4*>(dx + now.lead);
    const int end = end_of(now.lead);
    if (!r.counts(now.t)) {  // the same for the whole group
      if (losses && cta == 0 && me == 0) losses[row] = 0.0f;
      if (dlogits) {
        for (int i = first + me; i < end; i += threads) __stcs(out + i, make_uint4(0, 0, 0, 0));
        if (now.single >= 0) dx[now.single] = T::put(0.0f);
      }
      continue;
    }

    // With a whole c, a thread's comes from its first value or vector that is
    // not all -inf; the second attempt takes the maximum of all its values.
    Stat stat{kNegInf, 0.0f, 0.0f};
    bool whole = true;
    float2 sum[2] = {}, all = both(0.0f);
    if (now.x_single != kNegInf) {
      stat.c = reference(now.x_single);
      sum[0] = Exponent<true>(stat.c)(make_float2(now.x_single, kNegInf));
    }
    if (kAll && now.single >= 0) all.x = __fmul_rn(smoothed, now.x_single);
    Exponent<true> exp2(stat.c);
    each(end - first, [&](int b, const uint4& u) {
      float v[N];
      Vec<T>::unpack(u, v);
      if (kAll)
#pragma unroll
        for (int e = 0; e < N; e += 2) all = __ffma2_rn(both(smoothed), make_float2(v[e], v[e + 1]), all);
      if (stat.c == kNegInf) {
        float m = v[0];
#pragma unroll
        for (int e = 1; e < N; ++e) m = fgt_fmax(m, v[e]);
        if (m == kNegInf) return;
        stat.c = reference(m);
        exp2 = Exponent<true>(stat.c);
      }
#pragma unroll
      for (int e = 0; e < N; e += 2) sum[b % 2] = __fadd2_rn(sum[b % 2], exp2(make_float2(v[e], v[e + 1])));
    }, [] {});
    for (;; whole = false) {
      const float2 both_sums = __fadd2_rn(sum[0], sum[1]);
      stat.s = both_sums.x + both_sums.y;
      stat.all = all.x + all.y;
      if (whole) settle(stat);
      stat = warp_join<kAll>(stat, whole);
      if (G != kWarp) {
        Stat* slot = &s_stat[parity][cta * warps + warp];
        if (G == kCluster) {
          if (lane < ctas) {
            unsigned to;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"((unsigned)__cvta_generic_to_shared(slot)), "r"(lane));
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(stat.c) : "memory");
            asm volatile("st.shared::cluster.f32 [%0+4], %1;" ::"r"(to), "f"(stat.s) : "memory");
            asm volatile("st.shared::cluster.f32 [%0+8], %1;" ::"r"(to), "f"(stat.all) : "memory");
          }
          fgt_cluster_sync();
        } else {
          if (lane == 0) *slot = stat;
          __syncthreads();
        }
        Stat total{kNegInf, 0.0f, 0.0f};  // up to four warps' on each lane
        for (int i = lane; i < ctas * warps; i += 32) total.c = fgt_fmax(total.c, s_stat[parity][i].c);
        for (int i = lane; i < ctas * warps; i += 32) {
          const Stat o = s_stat[parity][i];
          const float d = o.c - (total.c == kNegInf ? 0.0f : total.c);
          total.s += o.s * fgt_ex2_approx(whole ? d : d * kLog2e);
          total.all += o.all;
        }
        stat = warp_join<kAll>(total, whole);
        parity ^= 1;  // the next exchange's writers do not meet this one's readers
      }
      if (whole) settle(stat);  // the row's, for the gradient's factor
      if (!whole || (stat.s > 0.0f && stat.s < __int_as_float(0x7f800000) && fabsf(stat.c) < kWholes)) break;  // the same decision for the whole group
      const uint4* in = reinterpret_cast<const uint4*>(logits + row * r.vocab + now.lead);
      float m = now.x_single;
      for (int i = first + me; i < end; i += threads) {
        float v[N];
        Vec<T>::unpack(__ldg(in + i), v);
#pragma unroll
        for (int e = 0; e < N; ++e) m = fgt_fmax(m, v[e]);
      }
      stat.c = m;
      const Exponent<false> exp2(m == kNegInf ? 0.0f : m);
      sum[0] = exp2(make_float2(now.x_single, kNegInf));
      sum[1] = both(0.0f);
      for (int i = first + me; i < end; i += threads) {
        float v[N];
        Vec<T>::unpack(__ldg(in + i), v);
#pragma unroll
        for (int e = 0; e < N; e += 2) sum[1] = __fadd2_rn(sum[1], exp2(make_float2(v[e], v[e + 1])));
      }
    }

    const bool tells = losses && cta == 0 && me == 0;
    float lse = 0.0f;  // for the thread that stores the loss, and for all where it is part of the gradient
    if (tells || r.z != 0.0f) lse = whole ? (stat.c + log2f(stat.s)) * kLn2 : stat.c + logf(stat.s);
    if (tells) {
      float l = lse - (1.0f - r.smoothing) * now.x_t;
      if (kAll) l -= stat.all;
      if (r.z != 0.0f) l += r.z * lse * lse;
      losses[row] = l;
    }
    if (!dlogits) continue;
    const float g = now.g;
    const float peak = g * (r.z != 0.0f ? 1.0f + 2.0f * r.z * lse : 1.0f) / stat.s, share = g * smoothed;
    const int in_vecs = (int)now.t - now.lead, hit = in_vecs >= 0 ? in_vecs / N : -1;  // the vector that holds the target
    auto gradient = [&](auto exp2) {
      auto of = [&](float2 x) { return __ffma2_rn(exp2(x), both(peak), both(-share)); };
      uint4* o = out + (first + me);
      each(end - first, [&](int b, const uint4& u) {
        float v[N];
        Vec<T>::unpack(u, v);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float2 d = of(make_float2(v[e], v[e + 1]));
          v[e] = d.x;
          v[e + 1] = d.y;
        }
        __stcs(o + b * threads, Vec<T>::pack(v));
      }, [&] { o += kStep; });
      // single values, and the target's place once more by the thread that wrote it
      const float hit_share = g * (1.0f - r.smoothing);
      if (now.single >= 0) dx[now.single] = T::put(of(both(now.x_single)).x - (now.single == now.t ? hit_share : 0.0f));
      if (hit >= first && hit < end && (hit - first) % threads == me) dx[now.t] = T::put(of(both(now.x_t)).x - hit_share);
    };
    if (whole)
      gradient(Exponent<true>(stat.c));
    else
      gradient(Exponent<false>(stat.c));
  }
  fgt_cp_wait<0>();
}

void check(const fgt_cross_entropy_desc* d) {
  require(d != nullptr, "desc is NULL");
  check_index_dtype(d->target_dtype, "targets");
  require(is_float(d->dtype), "dtype must be f32, f16 or bf16");
  require(d->reduction >= FGT_LOSS_NONE && d->reduction <= FGT_LOSS_MEAN, "unknown reduction");
  require(d->label_smoothing >= 0.0f && d->label_smoothing <= 1.0f, "label_smoothing must be in [0, 1]");
  require(d->z_loss >= 0.0f && d->z_loss <= FLT_MAX, "z_loss must be finite and not negative");
  require(d->vocab > 0, "vocab must be positive");
  require(d->vocab <= 1 << 30, "vocab must be at most 2^30");
  size_product(d->rows, d->vocab, "rows x vocab");
  require(d->rows <= 0x7fffffff, "rows is too large for one launch");
}

// Workspace of SUM and MEAN: a ticket, the blocks' counts and sums, the row losses.
struct LossPlan {
  int64_t blocks;
  size_t counted, sums, losses, bytes;
};

LossPlan plan_loss(const fgt_cross_entropy_desc* d) {
  check(d);
  LossPlan p{};
  if (d->reduction == FGT_LOSS_NONE) return p;
  p.blocks = (d->rows + kCountRows - 1) / kCountRows;
  auto pad = [](int64_t n) { return (size_t)((n + 255) / 256 * 256); };
  p.counted = 256;
  p.sums = p.counted + pad(p.blocks * 4);
  p.losses = p.sums + pad(p.blocks * 8);
  p.bytes = p.losses + pad(d->rows * 4);
  return p;
}

// How rows are shared: a group's CTAs per row, threads per CTA.
struct RowShape {
  Group group;
  int ctas, threads;
};

// Sixteen vectors per thread and row: fewer leave the work per row to its fixed
// part (its barrier, its targets), more keep more rows at work than L2 holds
// between their two readings. Where the rows do not fill the GPU that way
// (148 SMs x 1024 threads), four vectors per thread finish a row sooner.
RowShape shape_for(int64_t rows, int64_t nvec) {
  const int64_t per_thread = rows * nvec >= 16 * 148 * 1024 ? 16 : 4, threads = (nvec + per_thread - 1) / per_thread;
  if (threads <= 32) return RowShape{kWarp, 1, 32 * kWarpGroups};
  if (threads <= 1024) {
    int t = 64;
    while (t < threads) t *= 2;
    return RowShape{kCta, 1, t};
  }
  RowShape s{kCluster, 2, per_thread == 16 ? 1024 : 512};
  while (s.ctas < 8 && (int64_t)s.ctas * s.threads < threads) s.ctas *= 2;
  return s;
}

}  // namespace
}  // namespace fgt

using namespace fgt;

extern "C" fgt_status fgt_cross_entropy_workspace(const fgt_cross_entropy_desc* d, size_t* bytes) {
  return guarded_call("fgt_cross_entropy_workspace", [&] {
    require(bytes != nullptr, "bytes is NULL");
    check(d);
    *bytes = plan_loss(d).bytes;
  });
}

extern "C" fgt_status fgt_cross_entropy(const fgt_cross_entropy_desc* d, const void* logits, const void* targets,
                                        const float* seed, float* loss, void* dlogits, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  return guarded_call("fgt_cross_entropy", [&] {
    const LossPlan p = plan_loss(d);
    check_buffer(logits, d->rows * d->vocab, "logits");
    check_buffer(targets, d->rows, "targets");
    // outputs without elements have no address: with no rows, all but a reduced loss
    require(loss != nullptr || dlogits != nullptr || d->rows == 0, "neither loss nor dlogits is asked for");
    if (loss) check_buffer(loss, 1, "loss");
    if (dlogits) check_buffer(dlogits, d->rows * d->vocab, "dlogits");
    if (seed) check_buffer(seed, 1, "seed");
    require(workspace_bytes >= p.bytes, "workspace of " + std::to_string(workspace_bytes) + " bytes is smaller than the " +
                                         std::to_string(p.bytes) + " bytes needed", FGT_ERR_WORKSPACE);
    require(p.bytes == 0 || (workspace && (uintptr_t)workspace % 256 == 0),
            "workspace must be a 256-byte aligned device buffer", FGT_ERR_WORKSPACE);
    if (d->rows == 0 && (!loss || d->reduction == FGT_LOSS_NONE)) return;  // nothing to write
    check_pending();
    char* ws = (char*)workspace;
    const Launch l{(cudaStream_t)stream, programmatic((cudaStream_t)stream)};
    const Row r{d->rows, d->vocab, d->ignore_index, d->label_smoothing, d->z_loss, d->grad_scale, d->reduction};
    const Index tg{targets, d->target_dtype == FGT_I64};
    const bool reduced = d->reduction != FGT_LOSS_NONE;
    int* counted = d->reduction == FGT_LOSS_MEAN && d->rows > kFewRows ? (int*)(ws + p.counted) : nullptr;
    float* losses = loss && reduced ? (float*)(ws + p.losses) : loss;
    const unsigned blocks = (unsigned)std::max<int64_t>(1, p.blocks);
    // the count, or for SUM over several blocks only the ticket
    const bool prepare = reduced && (counted || (loss && blocks > 1));
    if (prepare) launch(l, loss_count, blocks, kCountThreads, 0, 1, tg, r, (int*)(ws + p.counted), (unsigned*)ws);
    if (d->rows > 0)
      for_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        using E = typename T::S;
        const int64_t nvec = d->vocab / Vec<T>::kN;  // of a row that starts aligned
        const RowShape sh = shape_for(d->rows, nvec);
        const int per_cta = (int)((nvec + sh.ctas - 1) / sh.ctas);
        auto go = [&](auto kernel) {
          const size_t smem = (size_t)kStages * kBatch * sh.threads * 16;
          const int64_t groups = (int64_t)active_clusters(kernel, sh.threads, smem, sh.ctas) * (sh.group == kWarp ? kWarpGroups : 1);
          const int64_t used = std::min<int64_t>(groups, d->rows);
          const unsigned grid = (unsigned)(sh.group == kWarp ? (used + kWarpGroups - 1) / kWarpGroups : used * sh.ctas);
          launch(l, kernel, grid, (unsigned)sh.threads, smem, (unsigned)sh.ctas, (const E*)logits, tg, r, per_cta, seed,
                 counted, losses, (E*)dlogits);
        };
        auto by_group = [&](auto all) {
          constexpr bool kAll = decltype(all)::value;
          if (sh.group == kWarp) return go(loss_rows<T, kWarp, 32 * kWarpGroups, kAll>);
          if (sh.group == kCluster) return sh.threads == 512 ? go(loss_rows<T, kCluster, 512, kAll>) : go(loss_rows<T, kCluster, 1024, kAll>);
          switch (sh.threads) {
            case 64: return go(loss_rows<T, kCta, 64, kAll>);
            case 128: return go(loss_rows<T, kCta, 128, kAll>);
            case 256: return go(loss_rows<T, kCta, 256, kAll>);
            case 512: return go(loss_rows<T, kCta, 512, kAll>);
            default: return go(loss_rows<T, kCta, 1024, kAll>);
          }
        };
        if (losses && d->label_smoothing != 0.0f)
          by_group(std::true_type{});
        else
          by_group(std::false_type{});
      });
    if (loss && reduced)
      launch(l, loss_total, blocks, kCountThreads, 0, 1, losses, tg, r, counted, (double*)(ws + p.sums), (unsigned*)ws, loss);
  });
}
