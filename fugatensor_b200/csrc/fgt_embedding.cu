// fgt_embedding.cu — embedding lookup with scaling, and its gradient.
//
//   out[i, :]    = s * table[t_i, :]               (0 where t_i is outside [0, V))
//   dtable[v, :] = s * sum over {i : t_i = v} of dy[i, :]
//
// Both are bound by memory: the lookup reads its rows and writes them, the
// gradient reads dy once and writes the whole table once. What is hard in the
// gradient is the skew of text: a few tokens make up a large share of a batch
// while most rows of the table get none, and adding rows with atomics would
// make the result depend on their order. So the (token, position) pairs are
// sorted (stable) and a token's rows are added in the order of i; runs of more
// than 64 are cut into pieces that different warps add in f32, and the last warp
// to finish adds the pieces' sums in their order, whichever warp that is. Rows
// without a token are zeroed while the sort runs.
#include <type_traits>

#include "fgt_vocab.cuh"

namespace fgt {
namespace {

// ---------------------------------------------------------------- lookup ---
constexpr int kLookupThreads = 256, kLookupVecs = 4;

// out as 16-byte vectors: kVec when rows are whole vectors (dim * size a
// multiple of 16), else each vector's elements are gathered one by one, with
// the last partial vector stored by element. Bound by memory: repeated rows
// come from L2, so it reads the distinct rows and writes them all. 32768 tokens
// x 4096 bf16 out of 128000 rows take 60 us on B200 (6.0 TB/s, 0.93 of a
// copy's rate), 63 us with a division per vector instead of one per thread.
template <class T, bool kVec>
__global__ void __launch_bounds__(kLookupThreads)
    embedding_rows(const typename T::S* __restrict__ table, Index indices, fgt_i64 count, fgt_i64 vocab, fgt_i64 dim,
                   float scale, unsigned step_rows, unsigned step_vecs, typename T::S* __restrict__ out) {
  constexpr int N = Vec<T>::kN;
  grid_wait();
  grid_release();
  const fgt_i64 total = count * dim;
  const fgt_i64 first = blockIdx.x * (fgt_i64)(kLookupThreads * kLookupVecs) + threadIdx.x;
  uint4 v[kLookupVecs];
  if constexpr (kVec) {
    // the first vector's row and place by a division, the others' by adding what kLookupThreads vectors are
    const unsigned per_row = (unsigned)(dim / N);
    fgt_i64 row = total >> 32 ? first / per_row : (fgt_i64)((unsigned)first / per_row);
    unsigned col = (unsigned)(first - row * per_row);
    const uint4* const rows = reinterpret_cast<const uint4*>(table);
#pragma unroll
    for (int k = 0; k < kLookupVecs; ++k) {
      v[k] = make_uint4(0, 0, 0, 0);
      if (row < count) {
        const fgt_i64 t = indices[row];
        if (t >= 0 && t < vocab) v[k] = rows[t * per_row + col];
      }
      row += step_rows;
      col += step_vecs;
      if (col >= per_row) {
        col -= per_row;
        ++row;
      }
    }
#pragma unroll
    for (int k = 0; k < kLookupVecs; ++k) {
      const fgt_i64 at = first + k * kLookupThreads;
      if (at * N >= total) continue;
      float f[N];
      Vec<T>::unpack(v[k], f);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = __fmul_rn(f[e], scale);
      __stcs(reinterpret_cast<uint4*>(out + at * N), Vec<T>::pack(f));
    }
  } else {
#pragma unroll
    for (int k = 0; k < kLookupVecs; ++k) {
      const fgt_i64 at = (first + k * kLookupThreads) * N;
      if (at >= total) continue;
      fgt_i64 row = at / dim, col = at - row * dim;
      float f[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        f[e] = 0.0f;
        if (at + e < total) {
          const fgt_i64 t = indices[row];
          if (t >= 0 && t < vocab) f[e] = __fmul_rn(T::get(table[t * dim + col]), scale);
        }
        if (++col == dim) {
          col = 0;
          ++row;
        }
      }
      if (at + N <= total) {
        __stcs(reinterpret_cast<uint4*>(out + at), Vec<T>::pack(f));
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (at + e < total) out[at + e] = T::put(f[e]);
      }
    }
  }
}

// -------------------------------------------------------- sorting tokens ---
// A least-significant-digit radix sort of (token, position), stable. A key is
// the token, or V for tokens that have no gradient (outside the table, the
// padding row): those end up last. Digits have at most 9 bits, so a vocabulary
// below 2^18 takes two passes. A CTA holds kSortThreads * E pairs in shared
// memory; each warp ranks its pairs 32 at a time, and the warps' counts are
// summed per digit. The lanes with the same digit find each other in a table
// of lane masks per warp and digit (a round of 32 warps took 2 us with
// match.any, which walks the distinct values, 0.5 us with a ballot per bit). A
// pass puts the CTA's pairs in order before it sends them on, so that what goes
// to another CTA goes in runs (sent singly, a pass over 8 pairs per thread
// spent 10,000 cycles on it).
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kSortCtas = 8, kMostSortCtas = 16;  // the largest portable cluster, the largest

struct Tokens {
  Index ids;
  unsigned count;
  fgt_i64 vocab, padding;
  __device__ __forceinline__ unsigned key(unsigned i) const {
    const unsigned none = (unsigned)vocab, skip = (unsigned)padding;
    if (ids.wide) {
      const fgt_i64 t = static_cast<const fgt_i64*>(ids.p)[i];
      return t >= 0 && t < vocab && t != padding ? (unsigned)t : none;
    }
    const int t = static_cast<const int*>(ids.p)[i];
    return t >= 0 && (unsigned)t < none && (unsigned)t != skip ? (unsigned)t : none;
  }
};

struct SortShared {
  unsigned short hist[kSortWarps][kDigits];  // per warp: a digit's count, then its start within the CTA's
  unsigned total[kDigits];                   // per digit: the CTA's count
  unsigned start[kDigits];                   // per digit: its first place in the CTA
  unsigned delta[kDigits];                   // per digit: from a place in the CTA to one among all pairs
  unsigned totals[kMostSortCtas][kDigits];   // every CTA's total
  unsigned warp_sum[2][kDigits / 32];
};

// Stable rank of each of a warp's E x 32 digits within the warp; hist[warp]
// ends as the warp's counts. `masks` is scratch: kSortWarps x kDigits words.
constexpr size_t kMaskBytes = (size_t)kSortWarps * kDigits * 4;
template <int E>
__device__ __forceinline__ void rank_digits(SortShared& s, const unsigned (&digit)[E], unsigned (&rank)[E], unsigned* masks) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  unsigned* const mask = masks + warp * kDigits;
  for (int d = lane; d < kDigits / 4; d += 32) reinterpret_cast<uint4*>(mask)[d] = make_uint4(0, 0, 0, 0);
  for (int d = lane; d < kDigits / 8; d += 32) reinterpret_cast<uint4*>(s.hist[warp])[d] = make_uint4(0, 0, 0, 0);
  __syncwarp();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    atomicOr(&mask[digit[e]], 1u << lane);
    __syncwarp();
    const unsigned same = mask[digit[e]], before = s.hist[warp][digit[e]];
    rank[e] = before + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (same >> lane == 1u) {  // the last of them
      s.hist[warp][digit[e]] = (unsigned short)(before + __popc(same));
      mask[digit[e]] = 0;
    }
    __syncwarp();
  }
}

// hist[warp][d] becomes the count of d in the warps before; total[d] the CTA's.
__device__ __forceinline__ void scan_warps(SortShared& s) {
  __syncthreads();
  if (threadIdx.x < kDigits) {
    unsigned run = 0;
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) {
      const unsigned n = s.hist[w][threadIdx.x];
      s.hist[w][threadIdx.x] = (unsigned short)run;
      run += n;
    }
    s.total[threadIdx.x] = run;
  }
}

// start[d] = the CTA's pairs with a smaller digit; delta[d] = (pairs with a
// smaller digit anywhere) + (pairs with digit d in the CTAs before) - start[d].
// Thread d < kDigits brings its digit's counts: the CTA's, all, the CTAs' before.
__device__ __forceinline__ void scan_digits(SortShared& s, unsigned own, unsigned all, unsigned before) {
  unsigned run_own = own, run_all = all;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const unsigned o = __shfl_up_sync(~0u, run_own, m), a = __shfl_up_sync(~0u, run_all, m);
    if (lane >= m) {
      run_own += o;
      run_all += a;
    }
  }
  if (threadIdx.x < kDigits && lane == 31) {
    s.warp_sum[0][warp] = run_own;
    s.warp_sum[1][warp] = run_all;
  }
  __syncthreads();
  if (threadIdx.x < kDigits) {
    unsigned place = run_own - own, to = run_all - all + before;
    for (int w = 0; w < warp; ++w) {
      place += s.warp_sum[0][w];
      to += s.warp_sum[1][w];
    }
    s.start[threadIdx.x] = place;
    s.delta[threadIdx.x] = to - place;
  }
  __syncthreads();
}

// The CTA's pairs in the order of their digits, into `staged`.
template <int E>
__device__ __forceinline__ void stage_pairs(SortShared& s, const uint2 (&pair)[E], int shift, unsigned mask, const unsigned (&rank)[E], uint2* staged) {
  const int warp = threadIdx.x / 32;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const unsigned d = pair[e].x >> shift & mask;
    staged[s.start[d] + s.hist[warp][d] + rank[e]] = pair[e];
  }
  __syncthreads();
}

// ------------------------------------------------- sums over sorted tokens ---
constexpr int kTile = 32;    // sorted pairs whose runs one warp starts
constexpr int kPiece = 64;   // a longer run is cut into pieces of this length
constexpr int kWindow = 128; // pairs that a warp may look at: kTile + kPiece + 1 at most
constexpr int kSumThreads = 128;

// A run that starts in tile t belongs to t's warps whole when it has at most
// kPiece pairs. A longer one is cut at s, s + kPiece, ...: each piece belongs
// to the tile that it starts in, which is at most one piece of a run from an
// earlier tile (slot 2t) and the first piece of at most one run (slot 2t + 1).
struct Sums {
  const unsigned *keys, *pos;  // sorted
  const unsigned* first;       // per tile: where the run of its first pair starts
  unsigned long long* done;    // per tile that a long run starts in, and chunk: pieces finished (low half), pieces in all (high half, once known)
  float* partial;              // [2 * tiles, dim]
  fgt_u16* present;            // per block of kBlock rows: bit k set = its row k has a token
  unsigned count, tiles, vocab;
};

constexpr int kBlock = 16;           // rows of the table that are zeroed together
constexpr int kFillBits = 1 << 18;   // rows that one CTA marks at a time

// Rows without a token are zero: `rows` of a block, by the warps of a CTA.
__device__ __forceinline__ void zero_row(char* p, fgt_i64 row_bytes) {
  const int lane = threadIdx.x % 32;
  const int head = (int)((16 - ((uintptr_t)p & 15)) & 15);  // rows start on element boundaries: 2 bytes at least
  const fgt_i64 lead = head < row_bytes ? head : row_bytes, body = (row_bytes - lead) / 16;
  if (lane < lead / 2) reinterpret_cast<fgt_u16*>(p)[lane] = 0;
  uint4* q = reinterpret_cast<uint4*>(p + lead);
  for (fgt_i64 i = lane; i < body; i += 32) __stcs(q + i, make_uint4(0, 0, 0, 0));
  const fgt_i64 tail = lead + body * 16;
  if (lane < (row_bytes - tail) / 2) reinterpret_cast<fgt_u16*>(p + tail)[lane] = 0;
}

// Blocks of rows are dealt out to the filling CTAs in turn, since the frequent
// tokens of a vocabulary lie together. The CTAs of a cluster mark the rows of
// their blocks that occur: they share out the tokens, and each marks what it
// finds in the owner's shared memory, so they wait for nothing but each other
// (every CTA reading all 65536 tokens by itself took 17 us, all that time on L2).
// Where the tokens are sorted already they are searched instead. Blocks below
// `now` are zeroed here, the marks of the others are left for the CTAs that zero
// them beside the sums.
__device__ void fill_rows(const Tokens& tk, const unsigned* sorted, unsigned me, unsigned ctas, char* table,
                          fgt_i64 row_bytes, unsigned now, fgt_u16* present, unsigned* bits) {
  const unsigned rows = (unsigned)tk.vocab;
  const unsigned mates = cluster_size(), rank = fgt_cluster_rank(), leader = me - rank;  // this cluster: CTAs [leader, leader + mates)
  const fgt_i64 step = (fgt_i64)ctas * kFillBits;  // rows that one round covers over all CTAs
  // block / ctas as a product: exact for block * ctas < 2^32 (blocks of a round: ctas * 2^14, ctas <= 512)
  const unsigned inverse = (unsigned)(0x100000000ull / ctas) + 1;
  for (fgt_i64 low = 0; low < rows; low += step) {  // low is a multiple of kBlock
    for (int i = threadIdx.x; i < kFillBits / 32; i += blockDim.x) bits[i] = 0;
    fgt_cluster_sync();
    if (sorted) {
      for (unsigned bit = threadIdx.x; bit < kFillBits; bit += blockDim.x) {
        const fgt_i64 row = low + ((fgt_i64)(bit / kBlock) * ctas + me) * kBlock + bit % kBlock;
        if (row >= rows) break;
        unsigned lo = 0, hi = tk.count;
        while (lo < hi) {
          const unsigned mid = lo + (hi - lo) / 2;
          if (sorted[mid] < row)
            lo = mid + 1;
          else
            hi = mid;
        }
        if (lo < tk.count && sorted[lo] == row) atomicOr(&bits[bit / 32], 1u << (bit % 32));
      }
    } else {
      constexpr int kBatch = 8;  // loads in flight per thread
      const unsigned span = (unsigned)min(step, rows - low), from = (unsigned)low, stride = mates * blockDim.x;
      const unsigned here = (unsigned)__cvta_generic_to_shared(bits);
      for (unsigned i = rank * blockDim.x + threadIdx.x; i < tk.count; i += kBatch * stride) {
        unsigned key[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) key[u] = i + u * stride < tk.count ? tk.key(i + u * stride) : rows;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const unsigned at = key[u] - from, block = at / kBlock, turn = __umulhi(block, inverse);
          const unsigned mate = block - turn * ctas - leader;  // of this cluster, if it is below mates
          if (at >= span || mate >= mates) continue;           // (a key below `from` wraps past span)
          const unsigned bit = turn * kBlock + at % kBlock;
          unsigned to;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(here + bit / 32 * 4), "r"(mate));
          asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(to), "r"(1u << (bit % 32)) : "memory");
        }
      }
    }
    fgt_cluster_sync();
    for (unsigned turn = threadIdx.x; turn < kFillBits / kBlock; turn += blockDim.x) {
      const fgt_i64 block = low / kBlock + (fgt_i64)turn * ctas + me;
      if (block * kBlock >= rows) break;
      if (block >= now) present[block] = reinterpret_cast<fgt_u16*>(bits)[turn];
    }
    for (unsigned bit = threadIdx.x / 32; bit < kFillBits; bit += blockDim.x / 32) {
      const fgt_i64 row = low + ((fgt_i64)(bit / kBlock) * ctas + me) * kBlock + bit % kBlock;
      if (row >= rows || row >= (fgt_i64)now * kBlock) break;  // rows grow with bit
      if (!(bits[bit / 32] >> (bit % 32) & 1)) zero_row(table + row * row_bytes, row_bytes);
    }
    __syncthreads();
  }
}

// On B200 a launch takes 8 us for 1000 tokens, 13 for 8192, 18 for 32768, 23
// for 65536 and 37 for 131072 (two passes), most of it in waiting: for the
// loads, the cluster's barriers and its slowest CTA.
//
// One launch does three things at once: the first cluster sorts up to
// kSortThreads * E pairs per CTA in its distributed shared memory, the other
// CTAs mark the table's rows that a token names and zero part of the rest, and
// all of them clear the counters that the sums use. (With sorting = 0 the
// tokens are sorted already.)
template <int E>
__global__ void __launch_bounds__(kSortThreads, 1)
    embedding_grad_sort(Tokens tk, const unsigned* sorted, int sorting, int digit_bits, int passes, Sums out,
                        unsigned* keys, unsigned* pos, unsigned* first, fgt_i64 counters, char* table,
                        fgt_i64 row_bytes, unsigned now) {
  extern __shared__ uint4 shared[];
  constexpr unsigned kPairs = kSortThreads * E;
  grid_wait();
  grid_release();
  for (fgt_i64 i = blockIdx.x * (fgt_i64)kSortThreads + threadIdx.x; i < counters; i += (fgt_i64)gridDim.x * kSortThreads)
    out.done[i] = 0;
  if (blockIdx.x >= sorting) {
    fill_rows(tk, sorted, blockIdx.x - sorting, gridDim.x - sorting, table, row_bytes, now, out.present,
              reinterpret_cast<unsigned*>(shared));
    return;
  }
  SortShared& s = *reinterpret_cast<SortShared*>(shared);
  uint2 *pairs = reinterpret_cast<uint2*>(&s + 1), *staged = pairs + kPairs;  // staged: the masks' scratch too
  if (cluster_size() > 1) fgt_cluster_sync();  // every CTA has started before another writes to it
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const unsigned cta = fgt_cluster_rank(), ctas = cluster_size();
  const unsigned own = warp * (32 * E) + lane;  // pairs own + 32 e: a warp's are consecutive
  const unsigned mask = (1u << digit_bits) - 1;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    uint2 pair[E];
    unsigned digit[E], rank[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (pass == 0) {
        const unsigned i = cta * kPairs + own + 32 * e;
        pair[e] = make_uint2(i < tk.count ? tk.key(i) : ~0u, i);  // slots past the end sort behind everything
      } else {
        pair[e] = pairs[own + 32 * e];
      }
      digit[e] = pair[e].x >> shift & mask;
    }
    rank_digits<E>(s, digit, rank, reinterpret_cast<unsigned*>(staged));
    scan_warps(s);
    const unsigned total = threadIdx.x < kDigits ? s.total[threadIdx.x] : 0;
    if (threadIdx.x < kDigits) {
      const unsigned at = (unsigned)__cvta_generic_to_shared(&s.totals[cta][threadIdx.x]);
      for (unsigned c = 0; c < ctas; ++c) {
        unsigned to;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(at), "r"(c));
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(total) : "memory");
      }
    }
    fgt_cluster_sync();  // every CTA's totals are there, and every pair is in registers
    unsigned all = 0, before = 0;
    if (threadIdx.x < kDigits)
      for (unsigned c = 0; c < ctas; ++c) {
        const unsigned n = s.totals[c][threadIdx.x];
        all += n;
        before += c < cta ? n : 0;
      }
    scan_digits(s, total, all, before);
    stage_pairs<E>(s, pair, shift, mask, rank, staged);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const unsigned i = threadIdx.x + e * kSortThreads;
      const uint2 p = staged[i];
      const unsigned to = i + s.delta[p.x >> shift & mask];
      unsigned at = (unsigned)__cvta_generic_to_shared(pairs + to % kPairs);
      asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(to / kPairs));
      asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(p.x), "r"(p.y) : "memory");
    }
    fgt_cluster_sync();
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const unsigned i = threadIdx.x + e * kSortThreads, to = cta * kPairs + i;
    if (to >= tk.count) continue;
    keys[to] = pairs[i].x;
    pos[to] = pairs[i].y;
  }
  // where the run of each tile's first pair starts: a binary search
  for (unsigned i = threadIdx.x * kTile; i < kPairs; i += kSortThreads * kTile) {
    const unsigned at = cta * kPairs + i;
    if (at >= tk.count) break;
    const unsigned key = pairs[i].x;
    unsigned lo = 0, hi = at;
    while (lo < hi) {
      const unsigned mid = (lo + hi) / 2;
      if (fgt_dsmem_ld(&pairs[mid % kPairs].x, mid / kPairs) < key)
        lo = mid + 1;
      else
        hi = mid;
    }
    first[at / kTile] = lo;
  }
  fgt_cluster_sync();  // no CTA leaves while its pairs are read
}

// Batches that exceed a cluster's shared memory: each pass is two launches, a
// CTA's digit counts and then its scatter through global memory. A scattering
// CTA adds up the counts of all CTAs by itself, so there are few of them where
// the pairs are many: 2 pairs per thread up to 2^18 pairs, 8 beyond.
__device__ __forceinline__ uint2 wide_pair(const Tokens& tk, const unsigned* keys, const unsigned* pos, unsigned i) {
  if (i >= tk.count) return make_uint2(~0u, i);
  return keys ? make_uint2(keys[i], pos[i]) : make_uint2(tk.key(i), i);
}

template <int E>
__global__ void __launch_bounds__(kSortThreads)
    embedding_grad_count(Tokens tk, const unsigned* keys, const unsigned* pos, int shift, unsigned mask, unsigned* totals) {
  __shared__ unsigned n[kDigits];
  grid_wait();
  grid_release();
  if (threadIdx.x < kDigits) n[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e)
    atomicAdd(&n[wide_pair(tk, keys, pos, (blockIdx.x * E + e) * kSortThreads + threadIdx.x).x >> shift & mask], 1u);
  __syncthreads();
  if (threadIdx.x < kDigits) totals[(fgt_i64)blockIdx.x * kDigits + threadIdx.x] = n[threadIdx.x];
}

template <int E>
__global__ void __launch_bounds__(kSortThreads, 1)
    embedding_grad_scatter(Tokens tk, const unsigned* keys, const unsigned* pos, int shift, unsigned mask,
                           const unsigned* totals, unsigned* keys_out, unsigned* pos_out) {
  extern __shared__ uint4 shared[];
  SortShared& s = *reinterpret_cast<SortShared*>(shared);
  uint2* staged = reinterpret_cast<uint2*>(&s + 1);
  grid_wait();
  grid_release();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint2 pair[E];
  unsigned digit[E], rank[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    pair[e] = wide_pair(tk, keys, pos, blockIdx.x * (kSortThreads * E) + warp * (32 * E) + 32 * e + lane);
    digit[e] = pair[e].x >> shift & mask;
  }
  rank_digits<E>(s, digit, rank, reinterpret_cast<unsigned*>(staged));
  scan_warps(s);
  unsigned all = 0, before = 0;
  if (threadIdx.x < kDigits) {
#pragma unroll 16
    for (unsigned c = 0; c < gridDim.x; ++c) {
      const unsigned n = totals[(fgt_i64)c * kDigits + threadIdx.x];
      all += n;
      before += c < blockIdx.x ? n : 0;
    }
  }
  scan_digits(s, threadIdx.x < kDigits ? s.total[threadIdx.x] : 0, all, before);
  stage_pairs<E>(s, pair, shift, mask, rank, staged);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const unsigned i = threadIdx.x + e * kSortThreads;
    const uint2 p = staged[i];
    const unsigned to = i + s.delta[p.x >> shift & mask];
    if (to >= tk.count) continue;  // slots past the end
    keys_out[to] = p.x;
    pos_out[to] = p.y;
  }
}

__global__ void __launch_bounds__(256) embedding_grad_first(const unsigned* keys, unsigned count, unsigned* first) {
  grid_wait();
  grid_release();
  const unsigned at = (blockIdx.x * 256 + threadIdx.x) * kTile;
  if (at >= count) return;
  unsigned lo = 0, hi = at;
  const unsigned key = keys[at];
  while (lo < hi) {
    const unsigned mid = (lo + hi) / 2;
    if (keys[mid] < key)
      lo = mid + 1;
    else
      hi = mid;
  }
  first[at / kTile] = lo;
}

// Bound by memory: dy is read once, a warp keeps 8 rows of 512 bytes in flight
// (fewer leave it waiting), and the rows of the table that the sort's launch
// did not zero are zeroed beside it. 65536 x 1024 f32 into 32000 rows take 62 us
// on B200 (5.5 TB/s), 16384 x 2048 bf16 into 128000 rows 80 us (6.1 TB/s).
//
// One warp: a tile's runs, over the 32 * N columns of one chunk (N = values in
// 16 bytes). kVec: rows are whole 16-byte vectors and a lane holds one vector;
// else a lane holds N single columns, 32 apart.
template <class T, bool kVec> struct Walk {
  static constexpr int N = Vec<T>::kN;
  static constexpr int kBatch = 8;  // rows in flight per warp
  const typename T::S* dy;
  typename T::S* table;
  const unsigned *pos, *key;  // the window, in shared memory
  unsigned ends[kWindow / 32];  // bit i: pair i is the last of its run
  fgt_i64 dim, col;
  float scale;

  __device__ __forceinline__ bool has(int k) const { return kVec ? col < dim : col + 32 * k < dim; }
  __device__ __forceinline__ fgt_i64 column(int k) const { return kVec ? col + k : col + 32 * k; }

  // The last pair of the run of pair i < 32 (kWindow - 1 if it goes on past the window).
  __device__ __forceinline__ int run_end(int i) const {
    const unsigned m = ends[0] & ~0u << i;
    if (m) return __ffs(m) - 1;
#pragma unroll
    for (int j = 1; j < kWindow / 32; ++j)
      if (ends[j]) return 32 * j + __ffs(ends[j]) - 1;
    return kWindow - 1;
  }
  __device__ __forceinline__ bool ends_at(int i) const {
    const unsigned m = i < 64 ? (i < 32 ? ends[0] : ends[1]) : (i < 96 ? ends[2] : ends[3]);
    return m >> (i % 32) & 1;
  }

  __device__ __forceinline__ void put_row(unsigned row, const float (&acc)[N]) const {
    typename T::S* p = table + (fgt_i64)row * dim;
    float v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = __fmul_rn(acc[k], scale);
    if constexpr (kVec) {
      if (has(0)) __stcs(reinterpret_cast<uint4*>(p + col), Vec<T>::pack(v));
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (has(k)) p[column(k)] = T::put(v[k]);
    }
  }

  // Adds pairs [lo, hi) of the window run by run. A finished run goes to its
  // row; with `partial`, the sum of [lo, hi) (one run's) goes there instead.
  __device__ __forceinline__ void run(int lo, int hi, float* partial) const {
    float acc[N] = {};
    for (int i = lo; i < hi; i += kBatch) {
      typename T::S raw[kBatch][kVec ? 1 : N];
      uint4 vec[kVec ? kBatch : 1];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (i + u >= hi) break;
        const typename T::S* p = dy + (fgt_i64)pos[i + u] * dim;
        if constexpr (kVec) {
          vec[u] = has(0) ? __ldcs(reinterpret_cast<const uint4*>(p + col)) : make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
          for (int k = 0; k < N; ++k) raw[u][k] = has(k) ? p[column(k)] : T::put(0.0f);
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (i + u >= hi) break;
        float v[N];
        if constexpr (kVec) {
          Vec<T>::unpack(vec[u], v);
        } else {
#pragma unroll
          for (int k = 0; k < N; ++k) v[k] = T::get(raw[u][k]);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = __fadd_rn(acc[k], v[k]);
        if (!partial && ends_at(i + u)) {
          put_row(key[i + u], acc);
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] = 0.0f;
        }
      }
    }
    if (partial)
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (has(k)) __stcg(partial + column(k), acc[k]);
  }

  // The finished pieces of the run of `row` that starts at pair s, in order.
  __device__ __forceinline__ void join(const float* partial, unsigned s, unsigned pieces, unsigned row) const {
    float acc[N] = {};
    constexpr int kAhead = 64 / N;  // pieces in flight
    for (unsigned j = 0; j < pieces; j += kAhead) {
      float v[kAhead][N];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const fgt_i64 tile = (s + (j + u) * kPiece) / kTile;
        const float* p = partial + (2 * tile + (j + u == 0)) * dim;
#pragma unroll
        for (int k = 0; k < N; ++k) v[u][k] = j + u < pieces && has(k) ? __ldcg(p + column(k)) : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (j + u < pieces) acc[k] = __fadd_rn(acc[k], v[u][k]);
    }
    put_row(row, acc);
  }
};

template <class T, bool kVec>
__global__ void __launch_bounds__(kSumThreads)
    embedding_grad_sums(Sums s, const typename T::S* __restrict__ dy, typename T::S* __restrict__ table, fgt_i64 dim,
                        fgt_i64 chunks, float scale, unsigned summing, unsigned filled) {
  __shared__ unsigned s_pos[kSumThreads / 32][kWindow], s_key[kSumThreads / 32][kWindow];
  constexpr int N = Vec<T>::kN;
  grid_wait();
  grid_release();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (blockIdx.x >= summing) {  // the rows that the sort's launch left: a block of rows per CTA
    const unsigned block = filled + (blockIdx.x - summing), marks = s.present[block];
    const fgt_i64 row_bytes = dim * (fgt_i64)sizeof(typename T::S);
    for (int k = warp; k < kBlock; k += kSumThreads / 32) {
      const fgt_i64 row = (fgt_i64)block * kBlock + k;
      if (row < s.vocab && !(marks >> k & 1)) zero_row(reinterpret_cast<char*>(table) + row * row_bytes, row_bytes);
    }
    return;
  }
  const fgt_i64 work = blockIdx.x * (fgt_i64)(kSumThreads / 32) + warp;
  const fgt_i64 tile = work / chunks, chunk = work % chunks;
  if (tile >= s.tiles) return;
  const unsigned i0 = (unsigned)tile * kTile;
  unsigned key[kWindow / 32];
#pragma unroll
  for (int j = 0; j < kWindow / 32; ++j) {
    const unsigned i = i0 + 32 * j + lane;
    key[j] = i < s.count ? s.keys[i] : s.vocab;
    s_key[warp][32 * j + lane] = key[j];
    s_pos[warp][32 * j + lane] = i < s.count ? s.pos[i] : 0;
  }
  const bool fresh = i0 == 0 || s.keys[i0 - 1] != s.keys[i0];  // the first pair starts a run
  __syncwarp();
  Walk<T, kVec> w;
  w.dy = dy;
  w.table = table;
  w.pos = s_pos[warp];
  w.key = s_key[warp];
  w.dim = dim;
  w.col = chunk * (32 * N) + (kVec ? lane * N : lane);
  w.scale = scale;
#pragma unroll
  for (int j = 0; j < kWindow / 32; ++j) {
    unsigned next = __shfl_down_sync(~0u, key[j], 1);
    const unsigned other = __shfl_sync(~0u, key[j + 1 < kWindow / 32 ? j + 1 : j], 0);
    if (lane == 31) next = j + 1 < kWindow / 32 ? other : key[j];
    w.ends[j] = __ballot_sync(~0u, key[j] != next);
  }
  const unsigned real = __ballot_sync(~0u, key[0] != s.vocab);
  const unsigned starts = (w.ends[0] << 1 | (fresh ? 1u : 0u)) & real;
  if (!real) return;  // tokens without a gradient sort last

  // A piece is stored, and its warp adds all of the run's pieces if it is the last to get here.
  auto piece = [&](unsigned start, unsigned j, int lo, int hi, bool last, int slot) {
    w.run(lo, hi, s.partial + (2 * tile + slot) * dim);
    __threadfence();
    __syncwarp();
    unsigned long long* done = s.done + (fgt_i64)(start / kTile) * chunks + chunk;
    unsigned long long now = 0;
    if (lane == 0) {
      const unsigned long long add = 1ull + (last ? (unsigned long long)(j + 1) << 32 : 0ull);
      now = atomicAdd(done, add) + add;
    }
    now = __shfl_sync(~0u, now, 0);
    if ((unsigned)now != (unsigned)(now >> 32)) return;
    __threadfence();
    w.join(s.partial, start, (unsigned)now, w.key[lo]);
  };

  if (!fresh) {  // a run from an earlier tile: its piece that starts here, if it is a long one
    const unsigned start = s.first[tile], off = i0 - start;
    const int end = w.run_end(0);
    const bool is_long = off + (unsigned)end >= kPiece;
    const int lo = (int)((off + kPiece - 1) / kPiece * kPiece - off);
    if (is_long && lo < kTile && lo <= end) {
      const bool last = end < lo + kPiece;
      piece(start, (off + lo) / kPiece, lo, last ? end + 1 : lo + kPiece, last, 0);
    }
  }
  if (!starts) return;
  const int lo = __ffs(starts) - 1, tail = 31 - __clz(starts), end = w.run_end(tail);
  const bool is_long = end - tail >= kPiece;
  w.run(lo, is_long ? tail : end + 1, nullptr);
  if (is_long) piece(i0 + tail, 0, tail, tail + kPiece, false, 1);
}

// ------------------------------------------------------------------ host ---
void check(const fgt_embedding_desc* d) {
  require(d != nullptr, "desc is NULL");
  check_index_dtype(d->index_dtype, "indices");
  require(is_float(d->dtype), "dtype must be f32, f16 or bf16");
  size_product(size_product(d->vocab, d->dim, "the table"), 4, "the table");
  size_product(size_product(d->count, d->dim, "indices x dim"), 4, "indices x dim");
  require(d->dim < (INT64_C(1) << 31), "dim must be below 2^31");
}

// How the workspace of the gradient is laid out (bytes from its start).
struct GradPlan {
  int wide_pairs;        // per thread of the sort through global memory (0: a cluster holds all pairs)
  int64_t tiles, chunks, blocks, sort_ctas;
  size_t keys, pos, first, done, present, partial, totals, keys2, pos2, bytes;
};

constexpr int64_t kClusterPairs = 8 * kSortThreads * kMostSortCtas;

GradPlan plan_grad(const fgt_embedding_desc* d) {
  check(d);
  require(d->vocab < 0xfffffffell, "the gradient takes a vocabulary below 2^32 - 2");
  require(d->count < 0x7fffffffll - 8 * kSortThreads, "the gradient takes fewer than 2^31 - 2^13 indices");
  GradPlan p{};
  const int64_t per_chunk = 32 * (16 / dtype_size(d->dtype));
  p.wide_pairs = d->count <= kClusterPairs ? 0 : d->count <= 1 << 18 ? 2 : 8;
  p.tiles = (d->count + kTile - 1) / kTile;
  p.chunks = (d->dim + per_chunk - 1) / per_chunk;
  p.blocks = (d->vocab + kBlock - 1) / kBlock;
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += (size_t)((bytes + 255) / 256 * 256);
    return here;
  };
  p.keys = take(d->count * 4);
  p.pos = take(d->count * 4);
  p.first = take(p.tiles * 4);
  p.done = take(p.tiles * p.chunks * 8);
  p.present = take(p.blocks * 2);
  p.partial = take(d->count > kPiece ? 2 * p.tiles * d->dim * 4 : 0);  // a run has a second piece at most
  if (p.wide_pairs) {
    p.sort_ctas = (d->count + kSortThreads * p.wide_pairs - 1) / (kSortThreads * p.wide_pairs);
    p.totals = take(p.sort_ctas * kDigits * 4);
    p.keys2 = take(d->count * 4);
    p.pos2 = take(d->count * 4);
  }
  p.bytes = at;
  return p;
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
    const Launch l{(cudaStream_t)stream, programmatic((cudaStream_t)stream)};
    const Index ids{indices, d->index_dtype == FGT_I64};
    const int64_t n = 16 / dtype_size(d->dtype);
    const unsigned grid = blocks_for((d->count * d->dim + n - 1) / n, kLookupThreads * kLookupVecs, "indices x dim");
    for_dtype(d->dtype, [&](auto t) {
      using T = decltype(t);
      using S = typename T::S;
      auto kernel = d->dim % n == 0 ? embedding_rows<T, true> : embedding_rows<T, false>;
      const unsigned per_row = (unsigned)std::max<int64_t>(1, d->dim / n);
      launch(l, kernel, grid, kLookupThreads, 0, 1, (const S*)table, ids, d->count, d->vocab, d->dim, d->scale,
             kLookupThreads / per_row, kLookupThreads % per_row, (S*)out);
    });
  });
}

extern "C" fgt_status fgt_embedding_grad_workspace(const fgt_embedding_desc* d, size_t* bytes) {
  return guarded_call("fgt_embedding_grad_workspace", [&] {
    require(bytes != nullptr, "bytes is NULL");
    *bytes = plan_grad(d).bytes;
  });
}

extern "C" fgt_status fgt_embedding_grad(const fgt_embedding_desc* d, const void* indices, const void* dy, void* dtable,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  return guarded_call("fgt_embedding_grad", [&] {
    const GradPlan p = plan_grad(d);
    check_buffer(indices, d->count, "indices");
    check_buffer(dy, d->count * d->dim, "dy");
    check_buffer(dtable, d->vocab * d->dim, "dtable");
    require(workspace_bytes >= p.bytes, "workspace of " + std::to_string(workspace_bytes) + " bytes is smaller than the " +
                                            std::to_string(p.bytes) + " bytes needed", FGT_ERR_WORKSPACE);
    require(p.bytes == 0 || (workspace && (uintptr_t)workspace % 256 == 0),
            "workspace must be a 256-byte aligned device buffer", FGT_ERR_WORKSPACE);
    if (d->vocab * d->dim == 0) return;
    check_pending();
    char* ws = (char*)workspace;
    const Launch l{(cudaStream_t)stream, programmatic((cudaStream_t)stream)};
    // a padding row outside the table is none: narrowed to 32 bits it could be another one
    const int64_t padding = d->padding_index >= 0 && d->padding_index < d->vocab ? d->padding_index : -1;
    const Tokens tk{Index{indices, d->index_dtype == FGT_I64}, (unsigned)d->count, d->vocab, padding};
    unsigned *keys = (unsigned*)(ws + p.keys), *pos = (unsigned*)(ws + p.pos), *first = (unsigned*)(ws + p.first);
    const Sums s{keys, pos, first, (unsigned long long*)(ws + p.done), (float*)(ws + p.partial), (fgt_u16*)(ws + p.present),
                 (unsigned)d->count, (unsigned)p.tiles, (unsigned)d->vocab};
    int bits = 1;
    while (d->vocab >> bits) ++bits;  // of the largest key, which is vocab itself
    const int passes = (bits + kDigitBits - 1) / kDigitBits, digit_bits = (bits + passes - 1) / passes;
    const int64_t row_bytes = d->dim * dtype_size(d->dtype);

    // The sort, beside CTAs that zero as many rows as take about its time
    // (4 MB/us: what is left of the GPU writes 5 to 6); the rest is zeroed
    // beside the sums. With sorting = 0 all of it is.
    unsigned now = 0;
    auto sort = [&](auto kernel, int pairs, unsigned cluster, int sorting) {
      const size_t held = (size_t)kSortThreads * pairs * sizeof(uint2);
      size_t smem = sorting ? sizeof(SortShared) + held + std::max(held, kMaskBytes) : 0;
      smem = std::max(smem, (size_t)kFillBits / 8);
      // as many clusters as run at once: a GPC's SMs do not all fit clusters of 8 or 16
      const unsigned grid = std::max(2u, active_clusters(kernel, kSortThreads, smem, cluster)) * cluster;
      if (sorting) now = (unsigned)std::min<int64_t>(p.blocks, (int64_t)(passes * (5 + 1.2 * pairs) + 3) * 4000000 / (row_bytes * kBlock));
      if (d->count == 0) now = (unsigned)p.blocks;
      launch(l, kernel, grid, kSortThreads, smem, cluster, tk, p.wide_pairs ? keys : nullptr, sorting, digit_bits, passes, s,
             keys, pos, first, p.tiles * p.chunks, (char*)dtable, row_bytes, now);
    };
    auto wide = [&](auto pairs) {
      constexpr int E = decltype(pairs)::value;
      const size_t smem = sizeof(SortShared) + std::max(kSortThreads * E * sizeof(uint2), kMaskBytes);
      active_clusters(embedding_grad_scatter<E>, kSortThreads, smem, 1);  // leave for the shared memory
      unsigned *from_k = nullptr, *from_p = nullptr;
      for (int pass = 0; pass < passes; ++pass) {
        const bool back = (passes - 1 - pass) % 2 == 1;  // the last pass writes keys and pos
        unsigned *to_k = back ? (unsigned*)(ws + p.keys2) : keys, *to_p = back ? (unsigned*)(ws + p.pos2) : pos;
        unsigned* totals = (unsigned*)(ws + p.totals);
        const int shift = pass * digit_bits;
        const unsigned mask = (1u << digit_bits) - 1;
        launch(l, embedding_grad_count<E>, (unsigned)p.sort_ctas, kSortThreads, 0, 1, tk, from_k, from_p, shift, mask, totals);
        launch(l, embedding_grad_scatter<E>, (unsigned)p.sort_ctas, kSortThreads, smem, 1, tk, from_k, from_p, shift, mask,
               totals, to_k, to_p);
        from_k = to_k;
        from_p = to_p;
      }
      launch(l, embedding_grad_first, blocks_for(p.tiles, 256, "indices"), 256, 0, 1, keys, (unsigned)d->count, first);
      sort(embedding_grad_sort<1>, 1, 1, 0);
    };
    if (p.wide_pairs == 2) {
      wide(std::integral_constant<int, 2>{});
    } else if (p.wide_pairs == 8) {
      wide(std::integral_constant<int, 8>{});
    } else if (d->count <= kSortThreads) {
      sort(embedding_grad_sort<1>, 1, 1, d->count > 0);
    } else if (d->count <= kSortCtas * kSortThreads) {
      sort(embedding_grad_sort<1>, 1, kSortCtas, kSortCtas);
    } else if (d->count <= kMostSortCtas * kSortThreads) {
      sort(embedding_grad_sort<1>, 1, kMostSortCtas, kMostSortCtas);
    } else if (d->count <= kMostSortCtas * kSortThreads * 2) {
      sort(embedding_grad_sort<2>, 2, kMostSortCtas, kMostSortCtas);
    } else if (d->count <= kMostSortCtas * kSortThreads * 4) {
      sort(embedding_grad_sort<4>, 4, kMostSortCtas, kMostSortCtas);
    } else {
      sort(embedding_grad_sort<8>, 8, kMostSortCtas, kMostSortCtas);
    }
    if (d->count == 0) return;
    const unsigned summing = blocks_for(p.tiles * p.chunks, kSumThreads / 32, "indices x dim");
    const unsigned filling = (unsigned)(p.blocks - now);
    require((int64_t)summing + filling <= 0x7fffffff, "indices x dim and vocab are too large for one launch");
    for_dtype(d->dtype, [&](auto t) {
      using T = decltype(t);
      using S = typename T::S;
      auto kernel = d->dim % Vec<T>::kN == 0 ? embedding_grad_sums<T, true> : embedding_grad_sums<T, false>;
      launch(l, kernel, summing + filling, kSumThreads, 0, 1, s, (const S*)dy, (S*)dtable, d->dim, p.chunks, d->scale, summing, now);
    });
  });
}
