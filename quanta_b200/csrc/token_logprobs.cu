// Rows of logits x[0..V): for a given token t its log probability, the entropy of the row, and the k most probable tokens.
//
//   m = max x, s = sum e^(x - m):   log p(t) = x[t] - m - log s,   entropy = log s - (sum e^(x - m) (x - m)) / s
//
// One pass over the row: every thread carries its own running maximum m with s and u = sum e^(x - m) (x - m), both rescaled where m grows; the
// parts are joined in a fixed order.  A token of probability zero (x = -inf) adds nothing.  A row with a NaN or +inf, or with nothing but -inf,
// has no distribution: its numbers are NaN, as log_softmax has it, and its k tokens are those of the order below.
//
// The k largest without sorting: the threads' maxima, taken together by fours, are 128 numbers; the k-th largest of them has at least k
// elements of the row at or above it, seldom many more.  The threads whose maximum reaches it read their elements once more (from L2)
// and lay those down that do; the candidates rank themselves by counting.  Where there are too many (rows of equal numbers, as masked ones
// are, or one thread's elements holding most of the largest) the largest are taken one by one instead.  Order: by value, -0 equal to 0 and
// NaN as -inf, equal ones by their place, the first first.
//
// A row is cut over the blocks of a cluster where rows are few; the first block joins what the others leave in shared memory.
// Bound by the row's bytes; for a few rows by the chain of a read, the joins and the second read.
#include "common.cuh"

namespace {

constexpr int TL_THREADS = 512, TL_WARPS = TL_THREADS / 32, TL_GROUPS = 128, TL_CAND = 1024, TL_MAX_TOP = 64, TL_MAX_CUT = 8;
constexpr float TL_LOG2E = 1.4426950408889634f;

struct TokenLogprobs {
  const void* logits;
  const int* tokens;
  float *logprob, *entropy;
  int* ids;
  float* best;
  int* status;
  int V, top, cut;
  long long stride;
};

__device__ __forceinline__ float tl_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float tl_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// larger numbers have larger keys; NaN as -inf, -0 as 0
__device__ __forceinline__ uint32_t tl_key(float x) {
  uint32_t b = __float_as_uint(x);
  if (x == 0.f) b = 0u;
  if (x != x) b = 0xff800000u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float tl_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// value and place in one number: equal values by their place, the first first
__device__ __forceinline__ unsigned long long tl_entry(float x, int i) { return (unsigned long long)tl_key(x) << 32 | (uint32_t)~i; }

struct TlSum {
  float m, s, u;
};
__device__ __forceinline__ TlSum tl_join(const TlSum& a, const TlSum& b) {
  const float m = tl_max_nan(a.m, b.m);
  if (m == -INFINITY) return TlSum{m, a.s + b.s, 0.f};      // zeros, or a NaN that has to be seen
  const float da = a.m - m, db = b.m - m;      // -inf: nothing yet
  const float fa = da == -INFINITY ? 0.f : expf(da), fb = db == -INFINITY ? 0.f : expf(db);
  return TlSum{m, a.s * fa + b.s * fb, (fa > 0.f ? (a.u + a.s * da) * fa : 0.f) + (fb > 0.f ? (b.u + b.s * db) * fb : 0.f)};
}

// A block's elements of a row as 16-byte pieces; the first and the last of a row may hang over its ends and are read one by one.
template <typename T> struct TlRow {
  static constexpr int PER = 16 / (int)sizeof(T);
  const T* row;
  int V, skip;            // elements of the first piece that lie before the row
  int pieces;
  __device__ TlRow(const void* logits, long long stride, int r, int V_) : row((const T*)logits + (size_t)r * stride), V(V_) {
    skip = (int)(((uintptr_t)row & 15) / sizeof(T));
    pieces = (skip + V + PER - 1) / PER;
  }
  __device__ int first(int piece) const { return piece * PER - skip; }
  __device__ bool whole(int piece) const { return first(piece) >= 0 && first(piece) + PER <= V; }
  __device__ uint4 load_whole(int piece) const { return *reinterpret_cast<const uint4*>(row + first(piece)); }
  __device__ static void numbers(const uint4& q, float (&v)[PER]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (PER == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  __device__ void load(int piece, float (&v)[PER]) const {
    if (whole(piece)) {
      numbers(load_whole(piece), v);
      return;
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int i = first(piece) + e;
      v[e] = i >= 0 && i < V ? qb_to_float<T>(row[i]) : -INFINITY;
    }
  }
};

struct TlShared {
  TlSum sums[TL_WARPS];
  float groups[TL_GROUPS];
  float threshold;
  int n_cand;
  unsigned long long cand[TL_CAND], sorted[TL_MAX_TOP], warp_best[TL_WARPS];
  TlSum total;
};

__device__ __forceinline__ unsigned long long tl_block_max(unsigned long long e, unsigned long long* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, e, o);
    e = other > e ? other : e;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = e;
  __syncthreads();
  e = scratch[0];
#pragma unroll
  for (int w = 1; w < TL_WARPS; ++w) e = scratch[w] > e ? scratch[w] : e;
  return e;
}

// the `top` largest of n entries (all different), largest first; 0 where there are fewer
__device__ __forceinline__ void tl_rank(const unsigned long long* e, int n, int top, unsigned long long* sorted) {
  for (int i = threadIdx.x; i < top; i += TL_THREADS) sorted[i] = 0ull;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += TL_THREADS) {
    const unsigned long long mine = e[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += e[j] > mine;
    if (above < top) sorted[above] = mine;
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(TL_THREADS) token_logprobs_kernel(TokenLogprobs a) {
  qb_follow();
  __shared__ TlShared sh;
  constexpr int PER = TlRow<T>::PER, AHEAD = 4;
  const int rank = a.cut > 1 ? (int)(blockIdx.x % a.cut) : 0, r = blockIdx.x / a.cut;
  const TlRow<T> row(a.logits, a.stride, r, a.V);
  const int share = (row.pieces + a.cut - 1) / a.cut, p_lo = rank * share, p_hi = min(row.pieces, p_lo + share);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) sh.n_cand = 0;

  // ---- the one pass ----
  TlSum mine{-INFINITY, 0.f, 0.f};
  for (int p0 = p_lo + (int)threadIdx.x; p0 < p_hi; p0 += AHEAD * TL_THREADS) {
    float v[AHEAD][PER];
    uint4 q[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int p = p0 + j * TL_THREADS;
      if (p < p_hi && row.whole(p)) q[j] = row.load_whole(p);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int p = p0 + j * TL_THREADS;
      if (p < p_hi && row.whole(p)) TlRow<T>::numbers(q[j], v[j]);
      else if (p < p_hi) row.load(p, v[j]);
      else {
#pragma unroll
        for (int e = 0; e < PER; ++e) v[j][e] = -INFINITY;
      }
    }
    float top = v[0][0];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
#pragma unroll
      for (int e = 0; e < PER; ++e) top = fmaxf(top, v[j][e]);
    if (top > mine.m) {
      const float d = mine.m - top;
      const float f = d == -INFINITY ? 0.f : tl_exp2(d * TL_LOG2E);
      mine.u = f > 0.f ? (mine.u + mine.s * d) * f : 0.f * mine.u;
      mine.s *= f;
      mine.m = top;
    }
    const float base = mine.m == -INFINITY ? 0.f : mine.m;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const float d = tl_max_nan(v[j][e] - base, -1e4f);      // e^d is zero there, and stays a number times d
        const float w = tl_exp2(d * TL_LOG2E);
        mine.s += w;
        mine.u = fmaf(w, d, mine.u);
      }
  }
  const float my_top = mine.m;      // NaN aside
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const TlSum other{__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o), __shfl_xor_sync(0xffffffffu, mine.u, o)};
    // the lower lane's part first, so that all lanes have the same sum
    mine = (lane & o) ? tl_join(other, mine) : tl_join(mine, other);
  }
  if (lane == 0) sh.sums[warp] = mine;

  // ---- the largest ----
  if (a.top > 0) {
    float g = my_top;
    g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 1));
    g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
    if ((threadIdx.x & 3) == 0) sh.groups[threadIdx.x >> 2] = g;
    __syncthreads();
    if (threadIdx.x < TL_GROUPS) {
      const float me = sh.groups[threadIdx.x];
      int above = 0;
#pragma unroll 8
      for (int j = 0; j < TL_GROUPS; ++j) above += sh.groups[j] > me || (sh.groups[j] == me && j < (int)threadIdx.x);
      if (above == a.top - 1) sh.threshold = me;
    }
    __syncthreads();
    const float threshold = sh.threshold;
    if (my_top >= threshold) {
      for (int p = p_lo + (int)threadIdx.x; p < p_hi; p += TL_THREADS) {
        float v[PER];
        row.load(p, v);
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const int i = row.first(p) + e;
          if ((v[e] >= threshold || v[e] != v[e]) && i >= 0 && i < a.V) {
            const int at = atomicAdd(&sh.n_cand, 1);
            if (at < TL_CAND) sh.cand[at] = tl_entry(v[e], i);
          }
        }
      }
    }
    __syncthreads();
    const int n = sh.n_cand;
    if (n <= TL_CAND) {
      tl_rank(sh.cand, n, a.top, sh.sorted);
    } else {
      // one by one: every thread holds the largest of its elements that is still to come
      unsigned long long last = ~0ull, best = 0ull;
      bool look = true;
      for (int k = 0; k < a.top; ++k) {
        if (look) {
          best = 0ull;
          for (int p = p_lo + (int)threadIdx.x; p < p_hi; p += TL_THREADS) {
            float v[PER];
            row.load(p, v);
#pragma unroll
            for (int e = 0; e < PER; ++e) {
              const int i = row.first(p) + e;
              const unsigned long long x = i >= 0 && i < a.V ? tl_entry(v[e], i) : 0ull;
              if (x < last && x > best) best = x;
            }
          }
        }
        const unsigned long long top = tl_block_max(best, sh.warp_best);
        if (threadIdx.x == 0) sh.sorted[k] = top;
        look = best == top;      // entries are all different: one thread's
        last = top;
      }
      __syncthreads();
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    TlSum total = sh.sums[0];
    for (int w = 1; w < TL_WARPS; ++w) total = tl_join(total, sh.sums[w]);
    sh.total = total;
  }
  __syncthreads();

  // ---- the blocks of a cluster joined ----
  if (a.cut > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0) {
      for (int i = threadIdx.x; i < a.cut * a.top; i += TL_THREADS) {
        uint32_t at = (uint32_t)__cvta_generic_to_shared(&sh.sorted[i % a.top]);
        asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(i / a.top));
        unsigned long long e;
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(e) : "r"(at) : "memory");
        sh.cand[i] = e != 0ull ? e : (unsigned long long)(uint32_t)i;      // none: below all others, and different
      }
      if (threadIdx.x == 0) {
        TlSum total = sh.total;
        for (int c = 1; c < a.cut; ++c) {
          float v[3];
          for (int i = 0; i < 3; ++i) {
            uint32_t at = (uint32_t)__cvta_generic_to_shared(&sh.total) + 4u * i;
            asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(c));
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[i]) : "r"(at) : "memory");
          }
          total = tl_join(total, TlSum{v[0], v[1], v[2]});
        }
        sh.total = total;
      }
      __syncthreads();
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0) return;
    if (a.top > 0) tl_rank(sh.cand, a.cut * a.top, a.top, sh.sorted);
  }

  const TlSum total = sh.total;
  const float none = __int_as_float(0x7fffffff);
  const bool is_one = total.m > -INFINITY && total.m < INFINITY;      // and s is NaN where an element is
  const float log_s = is_one ? logf(total.s) : none;
  if (threadIdx.x == 0) {
    if (a.logprob != nullptr) {
      const int t = a.tokens[r];
      if (t < 0 || t >= a.V) {
        qb_set_status(a.status, QB_STATUS_BAD_TOKEN, t, 12);
        a.logprob[r] = none;
      } else {
        a.logprob[r] = qb_to_float<T>(row.row[t]) - total.m - log_s;
      }
    }
    if (a.entropy != nullptr) a.entropy[r] = log_s - total.u / total.s;
  }
  for (int k = threadIdx.x; k < a.top; k += TL_THREADS) {
    const unsigned long long e = sh.sorted[k];
    a.ids[(size_t)r * a.top + k] = (int)~(uint32_t)e;
    a.best[(size_t)r * a.top + k] = tl_value((uint32_t)(e >> 32)) - total.m - log_s;
  }
}

}  // namespace

extern "C" int qb_token_logprobs(const void* logits, int dtype, long long stride, const int* tokens, float* logprob, float* entropy, int* ids,
                                 float* best, int n, int V, int top, int* status, cudaStream_t stream) {
  if (n <= 0) return 0;
  if (V <= 0 || top < 0 || (logprob != nullptr && tokens == nullptr)) return QB_ERR_BAD_ARG;
  if (top > TL_MAX_TOP || top > V) return QB_ERR_UNSUPPORTED;
  int dev = 0, sms = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (err != cudaSuccess) return (int)err;
  TokenLogprobs a{logits, tokens, logprob, entropy, ids, best, status, V, top, 1, stride};
  while (a.cut < TL_MAX_CUT && (long long)n * a.cut < sms && V / a.cut >= 4096) a.cut *= 2;
  if ((long long)n * a.cut > 0x7fffffffll) return QB_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = (unsigned)(n * a.cut);
  cfg.blockDim = TL_THREADS;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.cut;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  QB_DISPATCH_DTYPE(dtype, T, { err = cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a); });
  if (err != cudaSuccess) return (int)err;
  QB_LAUNCH_CHECK();
  return 0;
}
