// Rows of logits x[0..V): for a given token t its log probability, the entropy of the row, and the k most probable tokens.
//
//   m = max x, s = sum e^(x - m):   log p(t) = x[t] - m - log s,   entropy = log s - (sum e^(x - m) (x - m)) / s
//
// One pass over the row: every thread carries its own running maximum m with s and u = sum e^(x - m) (x - m), both rescaled where m grows; the
// parts are joined in a fixed order.  A token of probability zero (x = -inf) adds nothing.  A row with a NaN or +inf, or with nothing but -inf,
// has no distribution: its numbers are NaN, as log_softmax has it, and its k tokens are those of the order below.
//
// The k largest without sorting: the threads' maxima, taken together, are 128 numbers; the k-th largest of them has at least k elements of the row
// at or above it, seldom many more.  Every warp leaves the maximum of each 512 bytes that it reads; those that reach that number are read
// once more, and what reaches it there is a candidate; the candidates rank themselves by counting.  Where there are too many
// (rows of equal numbers, or with fewer possible tokens than are asked for) the largest are taken one by one instead, each after a thread has read its
// share once more, which takes many times as long (20 of a row of 200,064 with three possible tokens 53 us, of 2,048 such rows 4.2 ms).  Order: by value, -0 equal to 0 and NaN as -inf,
// equal ones by their place, the first first.  (Reading all elements of the threads that hold the 20 largest again, a third of a row's memory
// sectors, took 367 us at 2,048 rows of 200,064, where the pass alone takes 250.)
//
// A row is cut over the blocks of a cluster where rows are few; the first block joins what the others leave in shared memory.
// Bound by the row's bytes; in bfloat16 by the issue of instructions (two additions, a product, two exponentials and a multiply-add for two numbers);
// for a few rows by the chain of a read, the joins and the second read.  Measured on a B200, with 20 tokens a row: 2,048 rows of 200,064 float32 257 us (6.4
// TB/s), bfloat16 162 us (5.1 TB/s); 64 bfloat16 rows of 32,000 (5 tokens) 10 us, one row of 200,064 9.5 us.
#include "common.cuh"

namespace {

constexpr int TL_MAX_WARPS = 16, TL_GROUPS = 128, TL_CAND = 1024, TL_MAX_TOP = 64, TL_MAX_CUT = 16, TL_SLOTS = 2048;
constexpr float TL_LOG2E = 1.4426950408889634f;
constexpr float TL_LOW = -3.2964854295465914e+38f;      // near the lowest numbers, and a bfloat16

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
// two numbers at a time
__device__ __forceinline__ float2 tl_add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 tl_mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 tl_fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
// over the warp, NaN aside
__device__ __forceinline__ float tl_warp_max(float x) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
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
  float m, s, u;      // u: of what is below the maximum, sum e^(x - m) (x - m)
};
// Over the first `LANES` lanes (a power of two): the largest maximum, every part rescaled to it once, then plain sums in a tree, the same for all
// lanes.  A part without a number (m = -inf) has s = u = 0, or NaN, which stays.
template <int LANES>
__device__ __forceinline__ TlSum tl_join(TlSum v) {
  float m = v.m;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float d = v.m - m;
  if (v.m <= TL_LOW) v.u = 0.f * v.s;
  if (d >= -200.f) {      // (NaN where both are infinite)
    const float f = tl_exp2(d * TL_LOG2E);
    v.u = (v.u + v.s * d) * f;
    v.s *= f;
  } else if (m > -INFINITY) {
    v.s = v.u = 0.f * v.s;
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    v.s += __shfl_xor_sync(0xffffffffu, v.s, o);
    v.u += __shfl_xor_sync(0xffffffffu, v.u, o);
  }
  v.m = m;
  return v;
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
  // -inf where a piece hangs over
  __device__ uint4 load_edge(int piece) const {
    T v[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int i = first(piece) + e;
      v[e] = i >= 0 && i < V ? row[i] : qb_from_float<T>(-INFINITY);
    }
    return *reinterpret_cast<const uint4*>(v);
  }
  __device__ static uint4 nothing() {
    const uint32_t w = PER == 4 ? 0xff800000u : 0xff80ff80u;
    return make_uint4(w, w, w, w);
  }
  // What lies so far below the maximum m that its weight is zero anyway is raised to where it still is: differences stay numbers.  Below TL_LOW
  // there is no room for that; a -inf there leaves u without a number, which is zero then, all weights but those of m being zero (`tl_join`).
  __device__ static float floor_of(float m) { return m <= TL_LOW ? -INFINITY : fmaxf(m - fmaxf(200.f, fabsf(m) * 0.015625f), TL_LOW); }
  __device__ static void numbers_above(const uint4& q, float least, float (&v)[PER]) {
    if constexpr (PER == 4) {
      numbers(q, v);
#pragma unroll
      for (int e = 0; e < PER; ++e) v[e] = tl_max_nan(v[e], least);
    } else {
      uint4 c = q;
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&c);
      const __nv_bfloat162 l = __float2bfloat162_rn(least);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], l);
      numbers(c, v);
    }
  }
  // the largest number of a piece, NaN aside
  __device__ static float largest(const uint4& q) {
    if constexpr (PER == 4) {
      return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
    } else {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
      const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(__low2float(m), __high2float(m));
    }
  }
};

struct TlShared {
  TlSum sums[TL_MAX_WARPS], total, totals[TL_MAX_CUT];
  __align__(16) float groups[TL_GROUPS];
  float threshold;
  int n_cand, n_hits;
  float slots[TL_SLOTS + 4 * TL_MAX_WARPS];      // the largest of 32 pieces (of some such, in a very long row)
  unsigned short hits[TL_SLOTS];
  // the first block's `joined` receives the sorted entries of all blocks
  unsigned long long cand[TL_CAND], joined[TL_MAX_CUT * TL_MAX_TOP], sorted[TL_MAX_TOP], warp_best[TL_MAX_WARPS];
};

template <int THREADS>
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
  for (int w = 1; w < THREADS / 32; ++w) e = scratch[w] > e ? scratch[w] : e;
  return e;
}

// the `top` largest of n entries (all different), largest first; 0 where there are fewer
template <int THREADS>
__device__ __forceinline__ void tl_rank(const unsigned long long* e, int n, int top, unsigned long long* sorted) {
  for (int i = threadIdx.x; i < top; i += THREADS) sorted[i] = 0ull;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const unsigned long long mine = e[i];
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) above += e[j] > mine;
    if (above < top) sorted[above] = mine;
  }
  __syncthreads();
}

// N of a thread's pieces, `step` apart, all asked for before the first is looked at; -inf behind the end
template <typename T, int N>
__device__ __forceinline__ void tl_load(const TlRow<T>& row, int p0, int step, int p_hi, uint4 (&q)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int p = p0 + j * step;
    q[j] = TlRow<T>::nothing();
    if (p < p_hi) q[j] = row.whole(p) ? row.load_whole(p) : row.load_edge(p);
  }
}
// the same for a warp's pieces, whose first lane has p0 - lane; turns that lie inside the row ask nothing of each piece
template <typename T, int N>
__device__ __forceinline__ void tl_load_turns(const TlRow<T>& row, int p0, int lane, int step, int p_hi, uint4 (&q)[N]) {
  if (p0 > lane && row.first(p0 - lane + (N - 1) * step + 32) <= row.V && p0 - lane + (N - 1) * step + 32 <= p_hi) {
    const uint4* at = reinterpret_cast<const uint4*>(row.row + row.first(p0));
#pragma unroll
    for (int j = 0; j < N; ++j) q[j] = at[j * step];
  } else {
    tl_load(row, p0, step, p_hi, q);
  }
}

__device__ __forceinline__ void tl_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void tl_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// the address of the first block's variable of the same place
__device__ __forceinline__ uint32_t tl_of_first(const void* p) {
  uint32_t at = (uint32_t)__cvta_generic_to_shared(p);
  asm volatile("mapa.shared::cluster.u32 %0, %0, 0;" : "+r"(at));
  return at;
}

// AHEAD: pieces a thread has on their way while it works on as many.  LONG: rows whose parts have more than TL_SLOTS times 512 bytes
template <typename T, int THREADS, int AHEAD, bool LONG>
__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(TokenLogprobs a) {
  qb_follow();
  __shared__ TlShared sh;
  constexpr int PER = TlRow<T>::PER, WARPS = THREADS / 32;
  const int rank = a.cut > 1 ? (int)(blockIdx.x % a.cut) : 0, r = blockIdx.x / a.cut;
  if (a.cut > 1) tl_cluster_arrive();      // all blocks of the cluster run before one writes to the first's memory
  const TlRow<T> row(a.logits, a.stride, r, a.V);
  const int share = (row.pieces + a.cut - 1) / a.cut, p_lo = min(row.pieces, rank * share), p_hi = min(row.pieces, p_lo + share);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float x_token = 0.f;
  int token = -1;
  if (threadIdx.x == 0) {
    sh.n_cand = sh.n_hits = 0;
    if (rank == 0 && a.logprob != nullptr) token = a.tokens[r];
  }

  // ---- the one pass ----
  float my_top = -INFINITY;      // NaN aside
  float2 s2 = make_float2(0.f, 0.f), u2 = s2;
  uint4 q[AHEAD], q_next[AHEAD];
  // slot (b >> shift) * WARPS + warp: the pieces of the warp's turns (b >> shift) << shift and on, a turn being 32 pieces.  (The shift of every row's
  // slots, long or not, took 8% of the time in float32, 12% in bfloat16, which are bound by the issue of instructions as much as by memory.)
  const int turns = (p_hi - p_lo + THREADS - 1) / THREADS;
  int shift = 0, turn = 0;
  if (LONG)
    while (((turns - 1) >> shift) * WARPS + WARPS > TL_SLOTS) ++shift;
  {
    for (int k = lane; k <= (turns - 1) >> shift; k += 32) sh.slots[k * WARPS + warp] = -INFINITY;
    __syncwarp();
  }
  tl_load_turns(row, p_lo + (int)threadIdx.x, lane, THREADS, p_hi, q_next);
  // (whole warps take part in each turn)
#pragma unroll 2
  for (int p0 = p_lo + (int)threadIdx.x; p0 - lane < p_hi; p0 += AHEAD * THREADS, turn += AHEAD) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) q[j] = q_next[j];
    tl_load_turns(row, p0 + AHEAD * THREADS, lane, THREADS, p_hi, q_next);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const float of_piece = TlRow<T>::largest(q[j]), of_turn = tl_warp_max(of_piece);
      top = fmaxf(top, of_piece);
      if (lane == 0) {      // (turns behind the last have slots that nobody looks at)
        float* slot = &sh.slots[((turn + j) >> shift) * WARPS + warp];
        *slot = !LONG ? of_turn : tl_max_nan(*slot, of_turn);
      }
    }
    if (top > my_top) {
      const float d = my_top - top;
      if (d < -200.f) {      // nothing yet, or nothing that still has a weight, or a NaN that has to be seen
        s2.x *= 0.f, s2.y *= 0.f;
        u2 = s2;
      } else {
        const float f = tl_exp2(d * TL_LOG2E);
        u2 = make_float2((u2.x + s2.x * d) * f, (u2.y + s2.y * d) * f);
        s2 = make_float2(s2.x * f, s2.y * f);
      }
      my_top = top;
    }
    const float base = my_top == -INFINITY ? 0.f : -my_top, least = TlRow<T>::floor_of(-base);
    const float2 base2 = make_float2(base, base), log2e = make_float2(TL_LOG2E, TL_LOG2E);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      float v[PER];
      TlRow<T>::numbers_above(q[j], least, v);
#pragma unroll
      for (int e = 0; e < PER; e += 2) {
        const float2 d = tl_add2(make_float2(v[e], v[e + 1]), base2);
        const float2 w = tl_mul2(d, log2e), p = make_float2(tl_exp2(w.x), tl_exp2(w.y));
        s2 = tl_add2(s2, p);
        u2 = tl_fma2(p, d, u2);
      }
    }
  }
  if (token >= 0 && token < a.V) x_token = qb_to_float<T>(row.row[token]);
  if (a.top > 0) {
    float g = my_top;
#pragma unroll
    for (int o = 1; o < THREADS / TL_GROUPS; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (threadIdx.x % (THREADS / TL_GROUPS) == 0) sh.groups[threadIdx.x / (THREADS / TL_GROUPS)] = g;
  }
  const TlSum mine = tl_join<32>(TlSum{my_top, s2.x + s2.y, u2.x + u2.y});
  if (lane == 0) sh.sums[warp] = mine;
  __syncthreads();
  if (warp == WARPS - 1) {
    const TlSum total = tl_join<WARPS>(sh.sums[lane % WARPS]);
    if (lane == 0) sh.total = total;
  }

  // ---- the largest ----
  if (a.top > 0) {
    {
      // a group's place among all: THREADS / TL_GROUPS threads count a part each
      constexpr int PARTS = THREADS / TL_GROUPS;
      const int mine = threadIdx.x / PARTS, from = threadIdx.x % PARTS * 4;
      const float me = sh.groups[mine];
      int above = 0;
#pragma unroll 8
      for (int j = from; j < TL_GROUPS; j += 4 * PARTS) {
        const float4 g = *reinterpret_cast<const float4*>(&sh.groups[j]);
        above += (g.x > me || (g.x == me && j < mine)) + (g.y > me || (g.y == me && j + 1 < mine)) + (g.z > me || (g.z == me && j + 2 < mine)) +
                 (g.w > me || (g.w == me && j + 3 < mine));
      }
#pragma unroll
      for (int o = 1; o < PARTS; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
      if (from == 0 && above == a.top - 1) sh.threshold = me;
    }
    __syncthreads();
    const float threshold = sh.threshold;
    const int n_slots = ((turns - 1) >> shift) * WARPS + WARPS;
    for (int k = threadIdx.x; k < n_slots; k += THREADS)      // (a slot of nothing but NaN is looked at too)
      if (!(sh.slots[k] < threshold)) sh.hits[atomicAdd(&sh.n_hits, 1)] = (unsigned short)k;
    __syncthreads();
    // the pieces of the slots that reach the threshold, shared out over all
    const int pairs = sh.n_hits << (5 + shift);
    volatile int* n_cand = &sh.n_cand;
    constexpr int LOOK = 4;
    for (int k0 = threadIdx.x; k0 < pairs && *n_cand <= TL_CAND; k0 += LOOK * THREADS) {
      uint4 found[LOOK];
      int piece[LOOK];
#pragma unroll
      for (int j = 0; j < LOOK; ++j) {
        const int k = k0 + j * THREADS;
        piece[j] = p_hi;
        if (k < pairs) {
          const int slot = sh.hits[k >> (5 + shift)], of = (k >> 5) & ((1 << shift) - 1);
          piece[j] = p_lo + ((slot / WARPS << shift) + of) * THREADS + slot % WARPS * 32 + (k & 31);
        }
        found[j] = TlRow<T>::nothing();
        if (piece[j] < p_hi) found[j] = row.whole(piece[j]) ? row.load_whole(piece[j]) : row.load_edge(piece[j]);
      }
#pragma unroll
      for (int j = 0; j < LOOK; ++j) {
        float v[PER];
        TlRow<T>::numbers(found[j], v);
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const int i = row.first(piece[j]) + e;
          if ((v[e] >= threshold || v[e] != v[e]) && piece[j] < p_hi && i >= 0 && i < a.V) {
            const int at = atomicAdd(&sh.n_cand, 1);
            if (at < TL_CAND) sh.cand[at] = tl_entry(v[e], i);
          }
        }
      }
    }
    __syncthreads();
    const int n = sh.n_cand;
    if (n <= TL_CAND) {
      tl_rank<THREADS>(sh.cand, n, a.top, sh.sorted);
    } else {
      // one by one: every thread holds the largest of its elements that is still to come
      unsigned long long last = ~0ull, best = 0ull;
      bool look = true;
      for (int k = 0; k < a.top; ++k) {
        if (look) {
          best = 0ull;
          for (int p0 = p_lo + (int)threadIdx.x; p0 < p_hi; p0 += LOOK * THREADS) {
            uint4 found[LOOK];
            tl_load(row, p0, THREADS, p_hi, found);
#pragma unroll
            for (int j = 0; j < LOOK; ++j) {
              float v[PER];
              TlRow<T>::numbers(found[j], v);
#pragma unroll
              for (int e = 0; e < PER; ++e) {
                const int p = p0 + j * THREADS, i = row.first(p) + e;
                const unsigned long long x = p < p_hi && i >= 0 && i < a.V ? tl_entry(v[e], i) : 0ull;
                if (x < last && x > best) best = x;
              }
            }
          }
        }
        const unsigned long long top = tl_block_max<THREADS>(best, sh.warp_best);
        if (threadIdx.x == 0) sh.sorted[k] = top;
        look = best == top;      // entries are all different: one thread's
        last = top;
      }
    }
  }
  __syncthreads();

  // ---- the blocks of a cluster joined: all write to the first's memory ----
  if (a.cut > 1) {
    tl_cluster_wait();
    for (int k = threadIdx.x; k < a.top; k += THREADS)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(tl_of_first(&sh.joined[rank * a.top + k])), "l"(sh.sorted[k]) : "memory");
    if (threadIdx.x < 3) {
      const float v = threadIdx.x == 0 ? sh.total.m : threadIdx.x == 1 ? sh.total.s : sh.total.u;
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(tl_of_first(&sh.totals[rank]) + 4u * threadIdx.x), "f"(v) : "memory");
    }
    tl_cluster_arrive();
    tl_cluster_wait();
    if (rank != 0) return;
    if (warp == WARPS - 1) {
      const TlSum total = tl_join<TL_MAX_CUT>(lane < a.cut ? sh.totals[lane] : TlSum{-INFINITY, 0.f, 0.f});
      if (lane == 0) sh.total = total;
    }
    if (warp == 0) {
      // the lists are sorted: a lane holds the head of one and the entry behind it, the largest head is taken each time
      const unsigned long long* list = &sh.joined[min(lane, a.cut - 1) * a.top];
      unsigned long long head = lane < a.cut ? list[0] : 0ull, behind = lane < a.cut && a.top > 1 ? list[1] : 0ull;
      int at = 2;
      for (int k = 0; k < a.top; ++k) {
        const uint32_t key = __reduce_max_sync(0xffffffffu, (uint32_t)(head >> 32));
        const uint32_t place = __reduce_max_sync(0xffffffffu, (uint32_t)(head >> 32) == key ? (uint32_t)head : 0u);
        if (lane == 0) sh.sorted[k] = (unsigned long long)key << 32 | place;
        if (head == ((unsigned long long)key << 32 | place)) {
          head = behind;
          behind = lane < a.cut && at < a.top ? list[at] : 0ull;
          ++at;
        }
      }
    }
    __syncthreads();
  }

  const TlSum total = sh.total;
  const float none = __int_as_float(0x7fffffff);
  const bool is_one = total.m > -INFINITY && total.m < INFINITY;      // and s is NaN where an element is
  const float log_s = is_one ? logf(total.s) : none;
  if (threadIdx.x == 0) {
    if (a.logprob != nullptr) {
      const bool known = token >= 0 && token < a.V;
      if (!known) qb_set_status(a.status, QB_STATUS_BAD_TOKEN, token, 12);
      a.logprob[r] = known ? x_token - total.m - log_s : none;
    }
    if (a.entropy != nullptr) a.entropy[r] = log_s - total.u / total.s;
  }
  for (int k = threadIdx.x; k < a.top; k += THREADS) {
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
  // Few rows: blocks of 512 threads, as many a row as there are SMs for.  More: blocks of 256, four an SM, which go through some 2,750 float32 or 3,900
  // bfloat16 numbers a microsecond and take 5 us behind their part (measured); a row is cut so that the waves of blocks take the least
  // (rows of 200,064: 150 rows 44 us in four parts, 34 in three; 300 rows 72 in two, 63 in five).  Rows for two waves or more are not cut.
  const int threads = 5ll * n < 3 * sms ? 512 : 256;
  if (threads == 512) {
    while (a.cut < TL_MAX_CUT && (long long)n * a.cut < sms && V / a.cut >= 4096) a.cut *= 2;
  } else if (n < 8 * sms) {
    double least = 0.;
    for (int cut = 1; cut <= 8 && (cut == 1 || V / cut >= 4096); ++cut) {
      const double waves = (double)(((long long)n * cut + 4 * sms - 1) / (4 * sms));
      const double us = waves * ((double)V / cut / (dtype == QB_F32 ? 2750. : 3900.) + 5.);
      if (cut == 1 || us < least) {
        least = us;
        a.cut = cut;
      }
    }
  }
  if ((long long)n * a.cut > 0x7fffffffll) return QB_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = (unsigned)(n * a.cut);
  cfg.blockDim = threads;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.cut;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  QB_DISPATCH_DTYPE(dtype, T, {
    // (a block's slots: its pieces, a turn of its threads at a time)
    const long long share = ((long long)V / (16 / (int)sizeof(T)) + 2 + a.cut - 1) / a.cut;
    const bool is_long = (share + threads - 1) / threads * (threads / 32) > TL_SLOTS;
    auto kern = threads == 512 ? (is_long ? token_logprobs_kernel<T, 512, 4, true> : token_logprobs_kernel<T, 512, 4, false>)
                               : (is_long ? token_logprobs_kernel<T, 256, 4, true> : token_logprobs_kernel<T, 256, 4, false>);
    if (a.cut > 8) err = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (err == cudaSuccess) err = cudaLaunchKernelEx(&cfg, kern, a);
  });
  if (err != cudaSuccess) return (int)err;
  QB_LAUNCH_CHECK();
  return 0;
}
