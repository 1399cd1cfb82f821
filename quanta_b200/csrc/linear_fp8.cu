// y[t, n] = sum_b xs[b, t] ws[n / 128, b] sum_{k in block b} x[t, k] w[n, k]: the product of two e4m3 matrices with a scale for every 128 columns
// of a row of x and for every 128 x 128 block of w, on the 5th-generation tensor cores.
//
// The scales change every 128 k, so what the tensor cores sum over one block of k is taken out of TMEM, scaled and added in float32 registers
// (one rounding a block); several accumulators take turns, so that the tensor cores work on the next block meanwhile.  That addition has as
// many elements as the tile and has to keep up with the products (512 cycles for 128 x 256 and 128 k), which decides the forms:
//
//  * 8 tokens or fewer, but for matrices of very many short rows, and more where the matrix is small: linear_fp8_few.cu, without tensor memory (its
//    rule and both sides' times stand there).
//  * up to 32 tokens, or 64 of a matrix of few rows (linear_fp8_few_kernel): the weights are the 128-row operand and the tokens the N operand, so that few tokens use the full
//    height of the MMA and the weights are read once.  A TMEM lane is a weight row, a column a token; the columns' scales come from shared memory.
//  * more (linear_fp8_kernel): the tokens are the rows, the weights the columns.  A lane has its token's scale in a register and one weight
//    scale for all of its columns, so the addition is one packed multiply-add for two numbers and reads nothing.  (With the tokens as columns the
//    scales' way from shared memory to the registers, 128 KB a k block of 256 tokens, took 1,024 cycles: 8,192 x 4,096 x 22,016 1,175 us.)
//    Steps of many tokens: two blocks on neighbouring SMs take 256 tokens x 256 weight rows together (cta_group::2), each fetching its own 128
//    tokens and half of the weight tile.
//
// Measured on a B200, one product after another in a graph: 8,192 tokens, 4,096 x 22,016 650 to 680 us (2.2 PFLOP/s; 775 where products follow one another
// for seconds and the clock falls under the power limit), which is the power limit's and the issue's, the tensor cores being active 64% of the
// cycles; 1,024 x 4,096 x 4,096 20 us; 512 x 4,096 x 4,096 14.7 us and, in two parts along k, 317 x 5,648 x 2,000 16.2 us, which are bound by what an SM takes
// from L2 (some 50 bytes a cycle; a 128 x 128 tile reads 256 bytes for every 128 x 128 products); 128 x 4,096 x 22,016 23.7 us, the bytes 14; 32 x 11,008 x 4,096
// 13.4 us, the bytes 7.
//
// A product of few tiles is cut along k over the blocks of a cluster; each leaves its sums in shared memory, and every block adds one share of
// them, the blocks' parts in order, so the result is the same in every run.
//
// Every wait on an mbarrier is bounded; when one runs out the block records it in the status words, its outputs are NaN, it lets its copies in
// flight land, frees its TMEM and returns.  The wait for tensor memory (tcgen05.alloc) has no bound, so nothing that holds tensor memory waits for another block:
// it is given back before the cluster's barriers.  A pair's blocks do wait for one another with it, but where they ask for it nobody else can have it:
// they take an SM's registers (64,512 of 65,536) for themselves.
#include "fp8.cuh"
#include "tensor_core.cuh"

namespace {

constexpr int L8_M = 128, L8_BK = 128;      // weight rows of a tile; k of a stage: 128 bytes, one swizzle row
constexpr int L8_A = L8_M * L8_BK;          // bytes of a weight tile
constexpr int L8_MAX_STAGES = 8;
constexpr int L8_SCALES = 4, L8_AHEAD = 3;      // slots of the scales' ring, blocks they are fetched ahead of it
constexpr int L8_FIRST = 4;                 // the first adding warp
constexpr int L8_FEW_THREADS = 256, L8_THREADS = 384;

struct LinearFp8 {
  const float *xs, *ws;
  void* out;
  int T, K, N;
  int blocks, per;            // k blocks, k blocks a block of the cluster takes
  int stages, cut, t_tiles;
  int* status;
  int early;
};

struct L8Shared {
  uint64_t full[L8_MAX_STAGES], acc_full[L8_MAX_STAGES], acc_empty[L8_MAX_STAGES], sc_full[L8_SCALES], sc_empty[L8_SCALES];
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ void l8_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// c += a * b, two numbers at a time
__device__ __forceinline__ void l8_fma2(float2& c, float ax, float ay, float bx, float by) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%0, %1};\n\tfma.rn.f32x2 c, a, b, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "+f"(c.x), "+f"(c.y) : "f"(ax), "f"(ay), "f"(bx), "f"(by));
}

template <typename O>
__device__ __forceinline__ O l8_staged(uint32_t at) {
  if constexpr (sizeof(O) == 4) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return __uint_as_float(v);
  } else {
    unsigned short v;
    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
    return __ushort_as_bfloat16(v);
  }
}
// a map of a tensor on its way before the first copy needs it
__device__ __forceinline__ void l8_fetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

__device__ __forceinline__ float l8_remote(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

constexpr int L8_NONE = 0x7fffffff;         // a NaN's bits

// For a block that gave up: time (0.1 ms) for what it cannot wait on, copies or MMAs that are on their way
__device__ __forceinline__ void l8_give_time() {
  const uint64_t since = global_ns();
  for (uint32_t it = 0; it < TC_SPIN_LIMIT && global_ns() - since < 100000ull; ++it) __nanosleep(1000);
}

// Eight parts of four neighbours, from the blocks of the cluster at this address, added in the order of the blocks.
__device__ __forceinline__ float4 l8_sum_parts(uint32_t at, int cut) {
  float4 v[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    v[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < cut)
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v[r].x), "=f"(v[r].y), "=f"(v[r].z), "=f"(v[r].w) : "r"(mapa_u32(at, (uint32_t)r)) : "memory");
  }
  float4 s = v[0];
#pragma unroll
  for (int r = 1; r < 8; ++r)
    if (r < cut) s = make_float4(s.x + v[r].x, s.y + v[r].y, s.z + v[r].z, s.w + v[r].w);
  return s;
}
// whether a block of the cluster gave up
__device__ __forceinline__ bool l8_missing(int* flag, int cut) {
  int missing = 0;
  for (int r = 0; r < cut; ++r) missing |= __float_as_int(l8_remote(mapa_u32(smem_u32(flag), (uint32_t)r)));
  return missing != 0;
}
template <typename O>
__device__ __forceinline__ void l8_store4(O* row, int n, int N, float4 v) {
  if (N % 4 == 0 && ((uintptr_t)row & (4 * sizeof(O) - 1)) == 0) {      // (n is a multiple of 4)
    if (n >= N) return;
    if constexpr (sizeof(O) == 4) {
      *reinterpret_cast<float4*>(row + n) = v;
    } else {
      __nv_bfloat162 q[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
      *reinterpret_cast<uint2*>(row + n) = *reinterpret_cast<const uint2*>(q);
    }
    return;
  }
  const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < N) row[n + i] = qb_from_float<O>(f[i]);
}

//   warp 0     : TMA producer: per k block the weight tile [128 x 128] and the token tile [NT x 128], 128-byte swizzle, into a ring of stages
//   warp 1     : MMA issuer: 4 x tcgen05.mma (32 k each) a stage; the commit hands the accumulator over and frees the stage
//   warp 2     : scales: xs[b, t] * ws[n / 128, b] of the tile's tokens into a ring in shared memory, fetched several blocks ahead
//   warps 4-7  : one TMEM lane quadrant each: add, then store
// NT: tokens of a tile (the MMA's N)
template <int NT, typename O>
__global__ void __launch_bounds__(L8_FEW_THREADS)
linear_fp8_few_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, LinearFp8 a) {
  constexpr int ADDERS = 4, COLS = NT;
  constexpr uint32_t STAGE = L8_A + NT * L8_BK;
  constexpr int ACC = NT <= 32 ? 8 : 4;
  constexpr uint32_t TMEM = ACC * NT;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  __shared__ L8Shared sh;
  __shared__ __align__(16) float scales[L8_SCALES][NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = a.cut > 1 ? (int)cluster_ctarank() : 0, tile = blockIdx.x / a.cut;
  const int n0 = tile / a.t_tiles * L8_M, t0 = tile % a.t_tiles * NT;
  const int k_first = rank * a.per, k_blocks = max(0, min(a.per, a.blocks - k_first));
  volatile int* abort_flag = &sh.abort_flag;
  // weights that one token tile reads leave L2 first; tokens, and weights that others read too, stay
  const uint64_t pol_w = a.t_tiles > 1 ? l2_policy_evict_last() : l2_policy_evict_first(), pol_x = l2_policy_evict_last();

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) mbar_init(smem_u32(&sh.full[s]), 1);
    for (int s = 0; s < ACC; ++s) {
      mbar_init(smem_u32(&sh.acc_full[s]), 1);
      mbar_init(smem_u32(&sh.acc_empty[s]), ADDERS);
    }
    for (int s = 0; s < L8_SCALES; ++s) {
      mbar_init(smem_u32(&sh.sc_full[s]), 1);
      mbar_init(smem_u32(&sh.sc_empty[s]), ADDERS);
    }
    sh.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    l8_fetch_map(&tm_w);
    l8_fetch_map(&tm_x);
    // the first weights may be asked for before the launch ahead has ended; its tokens are not there yet
    for (int kb = 0; a.early && kb < min(a.stages, k_blocks); ++kb) {
      mbar_expect_tx(smem_u32(&sh.full[kb]), STAGE);
      tma_load_2d(smem_u32(tiles) + (uint32_t)kb * STAGE, &tm_w, (k_first + kb) * L8_BK, n0, smem_u32(&sh.full[kb]), pol_w);
    }
  }
  // (no tensor memory before it: a block of the launch ahead may still have to get its own)
  qb_follow();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = sh.tmem_base;

  O* out = reinterpret_cast<O*>(a.out);

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, armed = 0;
#pragma unroll 1
      for (int kb = 0; kb < k_blocks; ++kb) {
        // a stage is free when the products of the k block that it held are there (no more stages than accumulators: their barrier is then at that phase)
        const int past = kb - a.stages;
        if (past >= 0 && !mbar_wait(smem_u32(&sh.acc_full[past % ACC]), (uint32_t)(past / ACC) & 1u, abort_flag)) break;
        const uint32_t full = smem_u32(&sh.full[s]), st = smem_u32(tiles) + (uint32_t)s * STAGE;
        if (!a.early || kb >= a.stages) {
          mbar_expect_tx(full, STAGE);
          tma_load_2d(st, &tm_w, (k_first + kb) * L8_BK, n0, full, pol_w);
        }
        tma_load_2d(st + L8_A, &tm_x, (k_first + kb) * L8_BK, t0, full, pol_x);
        armed = kb + 1;
        if (++s == a.stages) s = 0;
      }
      if (*abort_flag && a.early && armed < min(a.stages, k_blocks)) {
        // weights are on their way whose tokens were not asked for, so that their barriers do not complete: give them time
        l8_give_time();
      }
      if (*abort_flag) {
        // let the copies that were issued land before this block's shared memory is given away
        for (int kb = max(0, armed - a.stages); kb < armed; ++kb) {
          const uint64_t since = global_ns();
          for (uint32_t it = 0; it < TC_SPIN_LIMIT && !mbar_try_wait(smem_u32(&sh.full[kb % a.stages]), (uint32_t)(kb / a.stages) & 1u); ++it)
            if ((it & 63u) == 63u && global_ns() - since > TC_WAIT_NS) break;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_e4m3(L8_M, NT);
      uint32_t parity = 0u;
      int s = 0;
#pragma unroll 1
      for (int kb = 0; kb < k_blocks; ++kb) {
        const int half = kb % ACC;
        if (!mbar_wait(smem_u32(&sh.acc_empty[half]), (uint32_t)(kb / ACC & 1) ^ 1u, abort_flag)) break;
        if (!mbar_wait(smem_u32(&sh.full[s]), parity, abort_flag)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t st = smem_u32(tiles) + (uint32_t)s * STAGE;
        const uint64_t a_desc = umma_desc_sw128(st), b_desc = umma_desc_sw128(st + L8_A);
#pragma unroll
        for (int k = 0; k < L8_BK / 32; ++k)      // 32 bytes further along the swizzled row: +2 in the 16-byte address field
          umma_e4m3(tmem_base + (uint32_t)(half * NT), a_desc + 2 * k, b_desc + 2 * k, idesc, k != 0);
        umma_commit(smem_u32(&sh.acc_full[half]));
        if (++s == a.stages) { s = 0; parity ^= 1u; }
      }
    }
  } else if (warp == 2) {
    constexpr int PER = (NT + 31) / 32;
    float ahead[L8_AHEAD][PER], w_ahead[L8_AHEAD];
    auto fetch = [&](int kb, float (&v)[PER], float& w) {
      const bool in = kb < k_blocks;
      w = in ? a.ws[(size_t)(n0 / L8_M) * a.blocks + k_first + kb] : 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int t = t0 + i * 32 + lane;
        v[i] = in && t < a.T && i * 32 + lane < NT ? a.xs[(size_t)(k_first + kb) * a.T + t] : 0.f;
      }
    };
#pragma unroll
    for (int d = 0; d < L8_AHEAD; ++d) fetch(d, ahead[d], w_ahead[d]);
    bool ok = true;
#pragma unroll 1
    for (int k0 = 0; k0 < k_blocks && ok; k0 += L8_AHEAD) {
#pragma unroll
      for (int d = 0; d < L8_AHEAD; ++d) {
        const int kb = k0 + d, slot = kb % L8_SCALES;
        if (kb >= k_blocks || !ok) break;
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.sc_empty[slot]), (uint32_t)(kb / L8_SCALES & 1) ^ 1u, abort_flag) ? 1 : 0) != 0;
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (i * 32 + lane < NT) scales[slot][i * 32 + lane] = ahead[d][i] * w_ahead[d];
        __syncwarp();
        if (lane == 0) l8_arrive(smem_u32(&sh.sc_full[slot]));
        fetch(kb + L8_AHEAD, ahead[d], w_ahead[d]);
      }
    }
  } else if (warp >= L8_FIRST) {
    float2 acc[COLS / 2];
  #pragma unroll
    for (int i = 0; i < COLS / 2; ++i) acc[i] = make_float2(0.f, 0.f);
    const int quad = warp & 3;
    const uint32_t from = tmem_base + ((uint32_t)(quad * 32) << 16);
    bool ok = true;
#pragma unroll 1
    for (int kb = 0; kb < k_blocks; ++kb) {
      const int half = kb % ACC, slot = kb % L8_SCALES;
      // tcgen05.ld is .sync.aligned: the lanes vote on the waits' answers
      ok = mbar_wait(smem_u32(&sh.sc_full[slot]), (uint32_t)(kb / L8_SCALES & 1), abort_flag);
      ok = ok && mbar_wait(smem_u32(&sh.acc_full[half]), (uint32_t)(kb / ACC & 1), abort_flag);
      ok = __all_sync(0xffffffffu, ok ? 1 : 0) != 0;
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      uint32_t v[2][16];
      tmem_ld16(from + (uint32_t)(half * NT), v[0]);
#pragma unroll
      for (int c = 0; c < COLS; c += 16) {
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (c + 16 < COLS) tmem_ld16(from + (uint32_t)(half * NT + c + 16), v[(c / 16 + 1) & 1]);
        const uint32_t(&u)[16] = v[(c / 16) & 1];
        const float4* sc = reinterpret_cast<const float4*>(&scales[slot][c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 f = sc[i];
          l8_fma2(acc[c / 2 + 2 * i], __uint_as_float(u[4 * i]), __uint_as_float(u[4 * i + 1]), f.x, f.y);
          l8_fma2(acc[c / 2 + 2 * i + 1], __uint_as_float(u[4 * i + 2]), __uint_as_float(u[4 * i + 3]), f.z, f.w);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        l8_arrive(smem_u32(&sh.acc_empty[half]));
        l8_arrive(smem_u32(&sh.sc_empty[slot]));
      }
    }
    if (a.cut == 1) {
      const int n = n0 + quad * 32 + lane;
      if (n < a.N) {
        O* dst = out + (size_t)t0 * a.N + n;
#pragma unroll
        for (int i = 0; i < COLS; ++i)
          if (t0 + i < a.T) dst[(size_t)i * a.N] = qb_from_float<O>(!ok ? __int_as_float(L8_NONE) : i & 1 ? acc[i / 2].y : acc[i / 2].x);
      }
    } else if (ok) {
      // all products are done, so the ring is free: this block's sums [NT][128]
      float* part = reinterpret_cast<float*>(tiles);
#pragma unroll
      for (int i = 0; i < COLS; ++i) part[i * L8_M + quad * 32 + lane] = i & 1 ? acc[i / 2].y : acc[i / 2].x;
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  // Given back before the cluster's barriers: a block that still waits for tensor memory reaches them only once it has some, and those it waits
  // for may be of its own cluster, or of another that holds columns here and waits for them on another SM (at 64 tokens, 1,024 x 4,096, shared memory
  // places four blocks on an SM, tensor memory two).
  if (warp == 1) {
    if (*abort_flag) l8_give_time();      // (MMAs whose accumulators nobody waited for)
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM) : "memory");
  }
  if (a.cut > 1) {
    cluster_sync_all();
    // a share of the columns; without the parts of a block that gave up it is no number
    const bool missing = l8_missing(&sh.abort_flag, a.cut);
    const uint32_t part = smem_u32(tiles);
    const int share = (NT + a.cut - 1) / a.cut, c_end = min(min(NT, (rank + 1) * share), a.T - t0);
    for (int i = rank * share * L8_M + (int)threadIdx.x * 4; i < c_end * L8_M; i += blockDim.x * 4) {
      float4 sum = l8_sum_parts(part + 4u * i, a.cut);
      if (missing) sum.x = sum.y = sum.z = sum.w = __int_as_float(L8_NONE);
      l8_store4(out + (size_t)(t0 + i / L8_M) * a.N, n0 + i % L8_M, a.N, sum);
    }
    cluster_sync_all();      // the parts stay until all have read them
  }
  if (threadIdx.x == 0 && sh.abort_flag) qb_set_status(a.status, QB_STATUS_WAIT_TIMEOUT, tile, 11);
}

// ---------------------------------------------------------------------------------------------
// More tokens.  A tile is 128 tokens x SIDE_N weight rows (128 or 256), or, for a PAIR of blocks, 256 tokens x SIDE_N weight rows (256 or 128), of which each block
// fetches its own 128 tokens and half of the weights and holds the sums of its own tokens.
//   warp 0     : TMA producer
//   warps 1, 2 : MMA issuers (of a pair's first block), 4 x tcgen05.mma a job, N = 128.  A k block of 256 weight rows is two jobs, the rows' halves, with
//                accumulators of their own (four in all), so that the addition of one half runs under the products of the other.  An MMA is
//                taken when the tensor cores are ready for it, and the waits and commits of a k block cost an issuer some 400 cycles besides the
//                512 of its products, so two take the k blocks in turn.  (One issuer, N = 256, two accumulators: 984 cycles a k block, of which
//                the tensor cores worked 512.)  The number of stages is even, so that a stage and an accumulator belong to one issuer, which
//                waits for every phase of their barriers in order.
//   warps 4-11 : a TMEM lane quadrant and half the columns (64 or 128) each: add, then store. They hold up to 128 sums a thread, more registers than
//                a block of 384 threads can give every one, so the other warps hand some of theirs over; what all have then is at most
//                what the block was launched with.
// Pairs walk over the tiles (a block an SM), so that the copies of the next tile run under the stores of the last; a block of a cut product has one.
// Tiles go by groups of L8_GROUP token tiles, whose tokens and the weights that pass meanwhile stay in L2.
constexpr int L8_REGS_ADD = 224, L8_REGS_OTHER = 56, L8_REGS_LAUNCH = 168, L8_GROUP = 8;
static_assert(256 * L8_REGS_ADD + 128 * L8_REGS_OTHER <= L8_THREADS * L8_REGS_LAUNCH, "registers of the launch");
constexpr int L8_BOX = 32 * 128;            // bytes of a warp's staged part of the output: 32 rows of 128 bytes
struct L8Big {
  uint64_t full[8], empty[8], acc_full[2][4], acc_empty[2][4];      // [half][accumulator]
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ void l8_arrive_at(uint32_t bar_cluster) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}
__device__ __forceinline__ void l8_store_box(const CUtensorMap* map, uint32_t from, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(c0), "r"(c1), "r"(from) : "memory");
}

template <bool PAIR, int SIDE_N, typename O>
__global__ void __launch_bounds__(L8_THREADS, 1)
linear_fp8_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_out,
                  LinearFp8 a, int boxes) {
  static_assert(SIDE_N == 128 || SIDE_N == 256, "weight rows of a tile");
  constexpr int SIDE_T = PAIR ? 256 : 128, HALVES = PAIR ? SIDE_N / 128 : 1, MMA_N = PAIR ? 128 : SIDE_N, COLS = SIDE_N / 2;
  constexpr int ACC = SIDE_N == 128 ? 4 : 2;      // accumulators a half
  constexpr int B_ROWS = PAIR ? SIDE_N / 2 : SIDE_N;      // weight rows that a block fetches
  constexpr uint32_t STAGE = L8_A + B_ROWS * L8_BK;
  constexpr uint32_t TMEM = 512;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  __shared__ L8Big sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR || a.cut > 1 ? (int)cluster_ctarank() : 0, width = PAIR ? 2 : a.cut;      // blocks of the cluster
  const int k_first = PAIR ? 0 : rank * a.per, k_blocks = max(0, min(a.per, a.blocks - k_first));
  const int n_tiles = (a.N + SIDE_N - 1) / SIDE_N, tiles_all = n_tiles * a.t_tiles;
  const int tile_first = blockIdx.x / width, tile_step = gridDim.x / width;
  volatile int* abort_flag = &sh.abort_flag;
  // a tile's first weight row and this block's first token
  auto place = [&](int tile, int& n0, int& t0) {
    const int per_group = L8_GROUP * n_tiles, group = tile / per_group, in = tile - group * per_group;
    const int high = min(L8_GROUP, a.t_tiles - group * L8_GROUP);
    n0 = in / high * SIDE_N;
    t0 = (group * L8_GROUP + in % high) * SIDE_T + (PAIR ? rank * 128 : 0);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(smem_u32(&sh.full[s]), 1);
      mbar_init(smem_u32(&sh.empty[s]), 1);
    }
    for (int s = 0; s < HALVES * ACC; ++s) {
      mbar_init(smem_u32(&sh.acc_full[s / ACC][s % ACC]), 1);
      mbar_init(smem_u32(&sh.acc_empty[s / ACC][s % ACC]), (PAIR ? 16 : 8) / HALVES);      // the warps that add it, of each block of a pair
    }
    sh.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    l8_fetch_map(&tm_w);
    l8_fetch_map(&tm_x);
    if (!PAIR && a.early) {      // a block alone: its first weights, as above
      int n0, t0;
      place(tile_first, n0, t0);
      const uint64_t pol = l2_policy_evict_last();
      for (int kb = 0; kb < min(a.stages, k_blocks); ++kb) {
        mbar_expect_tx(smem_u32(&sh.full[kb]), STAGE);
        tma_load_2d(smem_u32(tiles) + (uint32_t)kb * STAGE + L8_A, &tm_w, (k_first + kb) * L8_BK, n0, smem_u32(&sh.full[kb]), pol);
      }
    }
  }
  qb_follow();      // (no tensor memory before it: a block of the launch ahead may still have to get its own)
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(TMEM) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(TMEM) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (PAIR) cluster_sync_all();      // both blocks' barriers exist before either counts on the other's
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = sh.tmem_base;
  O* out = reinterpret_cast<O*>(a.out);

  if (warp < L8_FIRST) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L8_REGS_OTHER));
  if (warp == 0) {
    if (lane == 0) {
      const uint64_t pol = l2_policy_evict_last();
      const uint32_t full0 = smem_u32(&sh.full[0]), bars = PAIR ? mapa_u32(full0, 0u) : full0;
      uint32_t parity = 1u;
      int s = 0, armed = 0;
      bool ok = true;
#pragma unroll 1
      for (int tile = tile_first; tile < tiles_all && ok; tile += tile_step) {
        int n0, t0;
        place(tile, n0, t0);
        if (PAIR) n0 += rank * B_ROWS;
#pragma unroll 1
        for (int kb = 0; kb < k_blocks; ++kb) {
          ok = mbar_wait(smem_u32(&sh.empty[s]), parity, abort_flag);
          if (!ok) break;
          const uint32_t st = smem_u32(tiles) + (uint32_t)s * STAGE;
          // (a pair: every copy of either block counts on the first block's barrier, which expects both blocks' bytes)
          const bool ahead = !PAIR && a.early && kb < a.stages;
          if (!ahead && (rank == 0 || !PAIR)) mbar_expect_tx(full0 + 8u * s, (PAIR ? 2 : 1) * STAGE);
          if constexpr (PAIR) {
            tma_load_2d_pair(st, &tm_x, kb * L8_BK, t0, bars + 8u * s, pol);
            tma_load_2d_pair(st + L8_A, &tm_w, kb * L8_BK, n0, bars + 8u * s, pol);
          } else {
            tma_load_2d(st, &tm_x, (k_first + kb) * L8_BK, t0, full0 + 8u * s, pol);
            if (!ahead) tma_load_2d(st + L8_A, &tm_w, (k_first + kb) * L8_BK, n0, full0 + 8u * s, pol);
          }
          ++armed;
          if (++s == a.stages) { s = 0; parity ^= 1u; }
        }
      }
      const bool unarmed = !PAIR && a.early && armed < min(a.stages, k_blocks);
      if (*abort_flag && ((PAIR && rank != 0) || unarmed)) {
        // this block's copies count on the other block's barriers, which it cannot wait on, or on some that do not complete: give them time
        l8_give_time();
      } else if (*abort_flag) {
        // let the copies that were issued land before this block's shared memory is given away
        for (int i = max(0, armed - a.stages); i < armed; ++i) {
          const uint64_t since = global_ns();
          for (uint32_t it = 0; it < TC_SPIN_LIMIT && !mbar_try_wait(full0 + 8u * (i % a.stages), (uint32_t)(i / a.stages) & 1u); ++it)
            if ((it & 63u) == 63u && global_ns() - since > TC_WAIT_NS) break;
        }
      }
    }
  } else if (warp < 3) {
    if (lane == 0 && (rank == 0 || !PAIR)) {
      const uint32_t idesc = umma_idesc_e4m3(PAIR ? 256 : 128, MMA_N), first = (uint32_t)warp - 1u;
      const uint64_t a_first = umma_desc_sw128(smem_u32(tiles)), b_first = umma_desc_sw128(smem_u32(tiles) + L8_A);
      const int mine = tile_first < tiles_all ? (tiles_all - tile_first + tile_step - 1) / tile_step : 0;
      const int turns = mine * k_blocks;
      uint32_t full_parity = 0u, empty_parity = 1u;
      int s = (int)first;
      uint32_t buf = first;
      bool ok = true;
#pragma unroll 1
      for (int turn = (int)first; turn < turns && ok; turn += 2) {
        ok = mbar_wait(smem_u32(&sh.full[s]), full_parity, abort_flag);
        const uint64_t a_desc = a_first + (uint64_t)(s * (int)(STAGE >> 4)), b_desc = b_first + (uint64_t)(s * (int)(STAGE >> 4));
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          ok = ok && mbar_wait(smem_u32(&sh.acc_empty[h][buf]), empty_parity, abort_flag);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t to = tmem_base + ((uint32_t)(h * ACC) + buf) * (uint32_t)MMA_N;
#pragma unroll
          for (int k = 0; k < L8_BK / 32; ++k) {      // 32 bytes further along the swizzled row: +2 in the 16-byte address field
            // (a pair's half: 64 weight rows of each block)
            if (PAIR) umma_e4m3_pair(to, a_desc + 2 * k, b_desc + (uint64_t)(h * (64 * L8_BK >> 4) + 2 * k), idesc, k != 0);
            else umma_e4m3(to, a_desc + 2 * k, b_desc + 2 * k, idesc, k != 0);
          }
          if (PAIR) umma_commit_pair(smem_u32(&sh.acc_full[h][buf])); else umma_commit(smem_u32(&sh.acc_full[h][buf]));
        }
        if (!ok) break;
        if (PAIR) umma_commit_pair(smem_u32(&sh.empty[s])); else umma_commit(smem_u32(&sh.empty[s]));
        if ((buf += 2u) >= ACC) { buf = first; empty_parity ^= 1u; }
        if ((s += 2) >= a.stages) { s -= a.stages; full_parity ^= 1u; }
      }
    }
  } else if (warp >= L8_FIRST) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L8_REGS_ADD));
    constexpr int AHEAD = 4, WS = HALVES;
    const int quad = warp & 3, group = (warp - L8_FIRST) / 4, h = HALVES == 2 ? group : 0;
    // column i of the warp's sums: weight row n0 + col0 + i, or, of a pair's 256, n0 + col0 + i / 64 * 128 + i % 64
    constexpr int SPAN = HALVES == 2 ? 64 : COLS, STRIDE = HALVES == 2 ? 128 : COLS;
    const int col0 = group * SPAN;
    const uint32_t from = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(HALVES == 2 ? h * ACC * 128 : group * COLS);
    const uint32_t full0 = smem_u32(&sh.acc_full[h][0]), empty0 = PAIR ? mapa_u32(smem_u32(&sh.acc_empty[h][0]), 0u) : smem_u32(&sh.acc_empty[h][0]);
    // (a block alone has one tile, and the ring is free behind its products)
    const uint32_t staged = smem_u32(tiles) + (PAIR ? (uint32_t)a.stages * STAGE : 0u) + (uint32_t)(warp - L8_FIRST) * 2 * L8_BOX;
    float x_ahead[AHEAD], w_ahead[WS][AHEAD];
    const float *xs = a.xs, *ws = a.ws;
    bool has_x = false, has_w[WS];
    auto scales_of = [&](int tile) {      // of a tile's first blocks
      if (tile >= tiles_all) return;
      int n0, t0;
      place(tile, n0, t0);
      const int t = t0 + quad * 32 + lane;
      has_x = t < a.T;
      xs = a.xs + (size_t)k_first * a.T + (has_x ? t : 0);
      if (!PAIR && SIDE_N == 256) n0 += col0;
      ws = a.ws + (size_t)(n0 / L8_BK) * a.blocks + k_first;
#pragma unroll
      for (int i = 0; i < WS; ++i) has_w[i] = n0 + i * 128 < a.N;
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) {
        x_ahead[d] = has_x && d < k_blocks ? xs[(size_t)d * a.T] : 0.f;
#pragma unroll
        for (int i = 0; i < WS; ++i) w_ahead[i][d] = has_w[i] && d < k_blocks ? ws[i * a.blocks + d] : 0.f;
      }
    };
    scales_of(tile_first);
    uint32_t turn = 0u, at_box = 0u;
    bool ok = true;
#pragma unroll 1
    for (int tile = tile_first; tile < tiles_all; tile += tile_step) {
      float2 acc[COLS / 2];
#pragma unroll
      for (int i = 0; i < COLS / 2; ++i) acc[i] = make_float2(0.f, 0.f);
#pragma unroll 1
      for (int k0 = 0; k0 < k_blocks && ok; k0 += AHEAD) {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
          const int kb = k0 + d;
          if (kb >= k_blocks || !ok) break;
          const uint32_t buf = turn % ACC, at = from + buf * (uint32_t)MMA_N;
          float f[WS];
#pragma unroll
          for (int i = 0; i < WS; ++i) f[i] = x_ahead[d] * w_ahead[i][d];
          if (kb + AHEAD < k_blocks) {
            const int next = kb + AHEAD;
            if (has_x) x_ahead[d] = xs[(size_t)next * a.T];
#pragma unroll
            for (int i = 0; i < WS; ++i)
              if (has_w[i]) w_ahead[i][d] = ws[i * a.blocks + next];
          }
          // tcgen05.ld is .sync.aligned: the lanes vote on the wait's answer
          ok = __all_sync(0xffffffffu, mbar_wait(full0 + 8u * buf, turn / ACC & 1u, abort_flag) ? 1 : 0) != 0;
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          uint32_t v[2][16];
          tmem_ld16(at, v[0]);
#pragma unroll
          for (int c = 0; c < COLS; c += 16) {
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if (c + 16 < COLS) {
              tmem_ld16(at + (uint32_t)(c + 16), v[(c / 16 + 1) & 1]);
            } else {
              // all are read: the accumulator is free while the last of them are added
              asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
              __syncwarp();
              if (lane == 0) {
                if (PAIR) l8_arrive_at(empty0 + 8u * buf); else l8_arrive(empty0 + 8u * buf);
              }
            }
            const uint32_t(&u)[16] = v[(c / 16) & 1];
#pragma unroll
            for (int i = 0; i < 8; ++i) l8_fma2(acc[c / 2 + i], __uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]), f[c / SPAN], f[c / SPAN]);
          }
          ++turn;
        }
      }
      int n0, t0;
      place(tile, n0, t0);
      scales_of(tile + tile_step);
      if (!ok) {
#pragma unroll
        for (int i = 0; i < COLS / 2; ++i) acc[i].x = acc[i].y = __int_as_float(L8_NONE);
      }
      const int row = quad * 32 + lane;
      if (!PAIR && SIDE_N == 128 && a.cut > 1) {
        // all products are done, so the ring is free: this block's sums [128 tokens][128 + 4]
        if (ok) {
          float* part = reinterpret_cast<float*>(tiles) + row * (128 + 4) + col0;
#pragma unroll
          for (int i = 0; i < COLS / 4; ++i) *reinterpret_cast<float4*>(part + 4 * i) = make_float4(acc[2 * i].x, acc[2 * i].y, acc[2 * i + 1].x, acc[2 * i + 1].y);
        }
      } else if (PAIR || ok) {
        // 32 rows of 128 bytes at a time, laid out as the copy's swizzle has them; two boxes take turns.  Rows that do not lie on 16 bytes are written
        // by the warp, a row after the other (by its own thread each, two bytes of 32 rows at a time, 1,054 x 1,280 x 3,207 took 52 us).
        constexpr int PER = 128 / (int)sizeof(O);
#pragma unroll
        for (int b = 0; b < COLS / PER; ++b) {
          if (boxes && lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");      // the copy out of this box, two ago
          __syncwarp();
          const uint32_t box = staged + at_box, to = box + (uint32_t)lane * 128;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (sizeof(O) == 4) {
                const int i = b * PER + c * 4 + e;
                w[e] = __float_as_uint(i & 1 ? acc[i / 2].y : acc[i / 2].x);
              } else {
                const float2 p = acc[(b * PER + c * 8) / 2 + e];
                const __nv_bfloat162 q = __floats2bfloat162_rn(p.x, p.y);
                w[e] = *reinterpret_cast<const uint32_t*>(&q);
              }
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + (uint32_t)((c ^ (lane & 7)) * 16)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
          }
          const int n = n0 + col0 + b * PER / SPAN * STRIDE + b * PER % SPAN;
          if (!boxes) {
            __syncwarp();
            const int rows = min(32, a.T - t0 - quad * 32);
            O* dst = out + (size_t)(t0 + quad * 32) * a.N + n;
#pragma unroll 4
            for (int r = 0; r < rows; ++r, dst += a.N)
#pragma unroll
              for (int i = lane; i < PER; i += 32)
                if (n + i < a.N) dst[i] = l8_staged<O>(box + (uint32_t)(r * 128 + (i * (int)sizeof(O) ^ (r & 7) * 16)));
            at_box ^= (uint32_t)L8_BOX;
            continue;
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            if (t0 + quad * 32 < a.T && n < a.N) l8_store_box(&tm_out, box, n, t0 + quad * 32);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          at_box ^= (uint32_t)L8_BOX;
        }
      } else if (t0 + row < a.T) {
        O* dst = out + (size_t)(t0 + row) * a.N;
#pragma unroll
        for (int i = 0; i < COLS; ++i) {
          const int n = n0 + col0 + i / SPAN * STRIDE + i % SPAN;
          if (n < a.N) dst[n] = qb_from_float<O>(i & 1 ? acc[i / 2].y : acc[i / 2].x);
        }
      }
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1 && *abort_flag) l8_give_time();
  if constexpr (!PAIR) {      // before the cluster's barriers, as above
    if (warp == 1) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM) : "memory");
    }
  }
  if (!PAIR && SIDE_N == 128 && a.cut > 1) {
    cluster_sync_all();
    // a share of the rows; without the parts of a block that gave up they are no numbers
    const bool missing = l8_missing(&sh.abort_flag, a.cut);
    const uint32_t part = smem_u32(tiles);
    int n0, t0;
    place(tile_first, n0, t0);
    const int share = 128 / a.cut, r_end = min((rank + 1) * share, a.T - t0);
    for (int i = rank * share * 32 + (int)threadIdx.x; i < r_end * 32; i += L8_THREADS) {
      const int row = i / 32, col = i % 32 * 4;
      float4 sum = l8_sum_parts(part + 4u * (uint32_t)(row * (128 + 4) + col), a.cut);
      if (missing) sum.x = sum.y = sum.z = sum.w = __int_as_float(L8_NONE);
      l8_store4(out + (size_t)(t0 + row) * a.N, n0 + col, a.N, sum);
    }
  }
  // no block leaves while another reads its parts, and none of a pair, whose blocks have got their tensor memory together, gives it back while the other's
  // MMAs or sums may use it
  if (PAIR || a.cut > 1) cluster_sync_all();
  if constexpr (PAIR) {
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM) : "memory");
  }
  if (threadIdx.x == 0 && sh.abort_flag) qb_set_status(a.status, QB_STATUS_WAIT_TIMEOUT, tile_first, 11);
}

// [rows, cols] row-major, boxes of [box_rows] rows of 128 bytes
int l8_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint32_t size, uint32_t box_rows, CUtensorMapDataType type) {
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {cols * size};
  const cuuint32_t box[2] = {128 / size, box_rows};
  return make_map(map, base, 2, dims, strides, box, type);
}

int l8_cluster_launch(const void* kern, void** args, unsigned grid, unsigned threads, unsigned width, size_t smem, cudaStream_t stream) {
  cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (err != cudaSuccess) return (int)err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = width;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return (int)cudaLaunchKernelExC(&cfg, kern, args);
}

template <int NT, typename O>
int l8_few(CUtensorMap& tm_w, CUtensorMap& tm_x, LinearFp8& a, unsigned grid, size_t smem, cudaStream_t stream) {
  void* args[] = {&tm_w, &tm_x, &a};
  return l8_cluster_launch((const void*)linear_fp8_few_kernel<NT, O>, args, grid, L8_FEW_THREADS, (unsigned)a.cut, smem, stream);
}
template <bool PAIR, int SIDE_N, typename O>
int l8_many(CUtensorMap& tm_w, CUtensorMap& tm_x, CUtensorMap& tm_out, LinearFp8& a, int boxes, unsigned grid, size_t smem, cudaStream_t stream) {
  // the registers that the block's warps share out are those of the launch
  const void* kern = (const void*)linear_fp8_kernel<PAIR, SIDE_N, O>;
  cudaFuncAttributes attr;
  const cudaError_t err = cudaFuncGetAttributes(&attr, kern);
  if (err != cudaSuccess) return (int)err;
  if (attr.numRegs != L8_REGS_LAUNCH) return QB_ERR_UNSUPPORTED;
  void* args[] = {&tm_w, &tm_x, &tm_out, &a, &boxes};
  return l8_cluster_launch(kern, args, grid, L8_THREADS, PAIR ? 2u : (unsigned)a.cut, smem, stream);
}

}  // namespace

// linear_fp8_few.cu
bool qb_linear_fp8_tokens_takes(int T, int K, int N);
int qb_linear_fp8_tokens(const void* x, const float* xs, const void* w, const float* ws, void* out, int out_dtype, int T, int K, int N, int early,
                         int sms, cudaStream_t stream);

// early: w and ws were written two launches before this one at the latest (or by the host); all but pairs of blocks then ask for their
// first pieces before the launch ahead has ended.
extern "C" int qb_linear_fp8(const void* x, const float* xs, const void* w, const float* ws, void* out, int out_dtype, int T, int K, int N,
                             int early, int* status, cudaStream_t stream) {
  if (T <= 0 || N <= 0) return 0;
  if (K <= 0 || K % 16 || (((uintptr_t)x | (uintptr_t)w) & 15)) return QB_ERR_BAD_ARG;
  if (out_dtype != QB_F32 && out_dtype != QB_BF16) return QB_ERR_BAD_ARG;
  int sms = 0;
  int rc = sm_count(sms);
  if (rc) return rc;
  if (qb_linear_fp8_tokens_takes(T, K, N)) return qb_linear_fp8_tokens(x, xs, w, ws, out, out_dtype, T, K, N, early, sms, stream);
  LinearFp8 a{xs, ws, out, T, K, N};
  a.early = early;
  a.blocks = (K + L8_BK - 1) / L8_BK;
  a.status = status;
  const CUtensorMapDataType bytes = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  CUtensorMap tm_w, tm_x, tm_out;
  // Weights as rows up to 32 tokens, and up to 64 where their tiles are half the SMs at most, so that eight k blocks and more are cut along k (64 tokens,
  // 8,192 x 8,192: 19.2 us, tokens as rows 20.1; 4,096 x 4,096: 9.7 and 10.2; 4,096 x 11,008, 86 tiles: 16.9 and 14.6).  With a short k that is the slower
  // side (64 tokens, 512 x 8,000, uncut: 5.9 and 5.0; 1,024 x 5,000, in two parts: 7.1 and 5.8; 2,048 x 9,000: 9.8 and 9.0).
  const long long tiles_128 = (N + L8_M - 1) / L8_M;
  if (T <= 32 || (T <= 64 && 2 * tiles_128 <= sms)) {
    const int NT = T <= 16 ? 16 : T <= 32 ? 32 : 64;
    a.t_tiles = 1;
    const long long tiles = tiles_128;
    // Along k as long as the parts are at most one an SM (a k block takes some 0.3 us, joining the parts some 2.5: 32 tokens, 16 tiles, 16 k blocks
    // 8.4 us uncut, 5.7 in four parts, 5.9 in eight), and once more where a part is still long (86 tiles, 32 k blocks, 32 tokens: 14.8 us, 14.0 in two).
    a.cut = 1;
    while (a.cut < 8 && tiles * a.cut * 2 <= sms && a.blocks >= (a.cut < 4 ? 8 : 32)) a.cut *= 2;
    if (a.cut < 8 && tiles * a.cut < sms && a.blocks / a.cut * NT >= 20 * 32) a.cut *= 2;
    a.per = (a.blocks + a.cut - 1) / a.cut;
    const size_t stage = L8_A + (size_t)NT * L8_BK, need = a.cut > 1 ? (size_t)NT * L8_M * 4 : 0;
    int stages = (int)(100 * 1024 / stage);
    if (stages > (NT <= 32 ? 8 : 4)) stages = NT <= 32 ? 8 : 4;      // (accumulators)
    if (stages > a.per) stages = a.per;
    a.stages = stages;
    const size_t ring = stage * stages, smem = (ring > need ? ring : need) + 1024;
    rc = l8_map(&tm_w, w, (uint64_t)N, (uint64_t)K, 1, L8_M, bytes);
    if (!rc) rc = l8_map(&tm_x, x, (uint64_t)T, (uint64_t)K, 1, (uint32_t)NT, bytes);
    if (rc) return rc;
    const unsigned grid = (unsigned)(tiles * a.cut);
    QB_DISPATCH_DTYPE(out_dtype, O, {
      if (NT == 16) rc = l8_few<16, O>(tm_w, tm_x, a, grid, smem, stream);
      else if (NT == 32) rc = l8_few<32, O>(tm_w, tm_x, a, grid, smem, stream);
      else rc = l8_few<64, O>(tm_w, tm_x, a, grid, smem, stream);
    });
    if (rc) return rc;
    QB_LAUNCH_CHECK();
    return 0;
  }
  // Pairs of blocks where tiles of 128 x 128 would be more than one for every SM (768 tokens, 4,096 x 4,096: 21 us, 27 with single blocks; 512, one tile an
  // SM: 19 and 14), but for tokens that fill half a pair's tile at most.  256 weight rows a pair or 128, whichever makes the shorter waves: a tile of
  // 128 takes some 0.65 of one of 256 (256 tokens, 4,096 x 22,016: 39 us in two waves of the one, 35 in three of the other; 1,024: 92 and 115).
  // Else single blocks, cut along k where they are few, or, where they are not cut and k is long, pairs with 128 rows, which fetch three quarters
  // of the bytes (512 tokens, 11,008 x 4,096: 30.4 us, single blocks 29.9, which took 35 before their ring had six stages; 4,096 x 4,096: 14.7 and 13.7).
  const long long singles = (T + 127) / 128 * tiles_128, t_pairs = (T + 255) / 256;
  const long long waves_256 = (t_pairs * ((N + 255) / 256) * 2 + sms - 1) / sms, waves_128 = (t_pairs * ((N + 127) / 128) * 2 + sms - 1) / sms;
  // Along k where that saves more than the joining takes (256 tokens, 4,096 x 4,096, 32 k blocks: 13.3 us uncut, 12.2 in two parts; 16 k blocks and 32 tiles:
  // 8.2 us, 8.7 in four parts).
  a.cut = 1;
  if (a.blocks > 16)
    while (a.cut < 4 && singles * a.cut * 2 <= sms) a.cut *= 2;
  const bool pair = T > 128 && (singles > sms || (a.cut == 1 && a.blocks >= 32));
  // Up to 128 tokens: tiles of 256 weight rows, by the bytes of their waves (128 tokens, 4,096 x 22,016: 29.5 us in two waves of 128 rows, 23.6 in one).
  const long long wide_waves = ((N + 255) / 256 + sms - 1) / sms, plain_waves = (singles + sms - 1) / sms;
  const int side = (pair ? singles > sms && waves_256 * 20 <= waves_128 * 13 : T <= 128 && wide_waves * (128 + 256) < plain_waves * (128 + 128)) ? 256 : 128;
  const int w_rows = pair ? side / 2 : side;      // weight rows of a block's stage
  const size_t size = out_dtype == QB_F32 ? 4 : 2;
  const int boxes = N * size % 16 == 0 && ((uintptr_t)out & 15) == 0;
  a.t_tiles = (T + (pair ? 255 : 127)) / (pair ? 256 : 128);
  const long long tiles = (long long)((N + side - 1) / side) * a.t_tiles;
  a.per = (a.blocks + a.cut - 1) / a.cut;
  if (tiles * a.cut > 0x7fffffffll) return QB_ERR_UNSUPPORTED;
  const size_t stage = L8_A + (size_t)w_rows * L8_BK, staged = pair ? 8 * 2 * L8_BOX : 0;
  a.stages = side == 128 ? 6 : 4;
  const size_t smem = stage * a.stages + staged + 1024;
  rc = l8_map(&tm_w, w, (uint64_t)N, (uint64_t)K, 1, (uint32_t)w_rows, bytes);
  if (!rc) rc = l8_map(&tm_x, x, (uint64_t)T, (uint64_t)K, 1, 128, bytes);
  if (!rc && boxes)
    rc = l8_map(&tm_out, out, (uint64_t)T, (uint64_t)N, (uint32_t)size, 32, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
  if (rc) return rc;
  if (!boxes) tm_out = tm_x;      // not used
  const unsigned grid = pair ? (unsigned)(tiles * 2 < sms / 2 * 2 ? tiles * 2 : sms / 2 * 2) : (unsigned)(tiles * a.cut);
  QB_DISPATCH_DTYPE(out_dtype, O, {
    if (pair && side == 256) rc = l8_many<true, 256, O>(tm_w, tm_x, tm_out, a, boxes, grid, smem, stream);
    else if (pair) rc = l8_many<true, 128, O>(tm_w, tm_x, tm_out, a, boxes, grid, smem, stream);
    else if (side == 256) rc = l8_many<false, 256, O>(tm_w, tm_x, tm_out, a, boxes, grid, smem, stream);
    else rc = l8_many<false, 128, O>(tm_w, tm_x, tm_out, a, boxes, grid, smem, stream);
  });
  if (rc) return rc;
  QB_LAUNCH_CHECK();
  return 0;
}
