// y[t, n] = sum_b xs[b, t] ws[n / 128, b] sum_{k in block b} x[t, k] w[n, k]: the product of two e4m3 matrices with a scale for every 128 columns
// of a row of x and for every 128 x 128 block of w, on the 5th-generation tensor cores.
//
// The scales change every 128 k, so what the tensor cores sum over one block of k is taken out of TMEM, scaled and added in float32 registers
// (one rounding a block); two accumulators take turns, so that the tensor cores work on the next block meanwhile.  The weights are the
// 128-row operand and the tokens the N operand: a block of 128 weight rows has one scale per k block, a token's scale belongs to a column, and a
// step of few tokens still uses the full height of the MMA and reads its weights once.  A thread of the adding warps owns one weight row (a
// TMEM lane) and up to 128 tokens.
//
//   warp 0     : TMA producer: per k block the weight tile [128 x 128] and the token tile [NT x 128], 128-byte swizzle, into a ring of stages
//   warp 1     : MMA issuer: 4 x tcgen05.mma (32 k each) a stage; commits free the stage and hand the accumulator over
//   warp 2     : scales: xs[b, t] * ws[n / 128, b] of the tile's tokens into a ring in shared memory, fetched several blocks ahead
//   warps 4-...: one TMEM lane quadrant each (two warps a quadrant where a tile has 128 tokens or more): add, then store
//
// A matrix of few tiles is cut along k over the blocks of a cluster; each leaves its sums in shared memory, and every block adds one share of the
// columns, the blocks' parts in order, so the result is the same in every run.
//
// Every wait on an mbarrier is bounded; when one runs out the block records it in the status words, its outputs are NaN, it lets its copies in
// flight land, frees its TMEM and returns.
#include "fp8.cuh"
#include "tensor_core.cuh"

namespace {

constexpr int L8_M = 128, L8_BK = 128;      // weight rows of a tile; k of a stage: 128 bytes, one swizzle row
constexpr int L8_A = L8_M * L8_BK;          // bytes of a weight tile
constexpr int L8_MAX_STAGES = 12, L8_SCALES = 4, L8_AHEAD = 3;      // slots of the scales' ring, blocks they are fetched ahead of it
constexpr int L8_FIRST = 4;                 // the first adding warp (a warpgroup of its own: it has other numbers of registers)

struct LinearFp8 {
  const float *xs, *ws;
  void* out;
  int T, K, N;
  int blocks, per;            // k blocks, k blocks a block of the cluster takes
  int stages, cut, t_tiles;
  int* status;
};

struct L8Shared {
  uint64_t full[L8_MAX_STAGES], empty[L8_MAX_STAGES], acc_full[2], acc_empty[2], sc_full[L8_SCALES], sc_empty[L8_SCALES];
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

__device__ __forceinline__ float l8_remote(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

constexpr int l8_adders(int NT) { return NT >= 128 ? 8 : 4; }
constexpr int l8_threads(int NT) { return (L8_FIRST + l8_adders(NT)) * 32; }
// Tiles of 256 tokens: the adding threads hold 128 sums each, more registers than a block of 384 threads can give every one of them, so
// the other warps hand some of theirs over.  What all have afterwards is what the block was launched with, at most.
constexpr int L8_REGS_ADD = 216, L8_REGS_OTHER = 56, L8_REGS_LAUNCH = 168;
static_assert(256 * L8_REGS_ADD + 128 * L8_REGS_OTHER <= 384 * L8_REGS_LAUNCH, "registers of the launch");

// NT: tokens of a tile (the MMA's N)
template <int NT, typename O>
__global__ void __launch_bounds__(l8_threads(NT))
linear_fp8_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, LinearFp8 a) {
  qb_follow();
  constexpr int ADDERS = l8_adders(NT), COLS = NT / (ADDERS / 4);      // columns an adding warp owns
  constexpr uint32_t STAGE = L8_A + NT * L8_BK;
  constexpr uint32_t TMEM = 2 * NT < 32 ? 32 : 2 * NT;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  __shared__ L8Shared sh;
  __shared__ __align__(16) float scales[L8_SCALES][NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = a.cut > 1 ? (int)cluster_ctarank() : 0, tile = blockIdx.x / a.cut;
  const int n0 = tile / a.t_tiles * L8_M, t0 = tile % a.t_tiles * NT;
  const int k_first = rank * a.per, k_blocks = max(0, min(a.per, a.blocks - k_first));
  volatile int* abort_flag = &sh.abort_flag;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(smem_u32(&sh.full[s]), 1);
      mbar_init(smem_u32(&sh.empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&sh.acc_full[s]), 1);
      mbar_init(smem_u32(&sh.acc_empty[s]), ADDERS);
    }
    for (int s = 0; s < L8_SCALES; ++s) {
      mbar_init(smem_u32(&sh.sc_full[s]), 1);
      mbar_init(smem_u32(&sh.sc_empty[s]), ADDERS);
    }
    sh.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = sh.tmem_base;

  O* out = reinterpret_cast<O*>(a.out);

  if (warp < L8_FIRST) {
    if constexpr (NT == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L8_REGS_OTHER));
  }
  if (warp == 0) {
    if (lane == 0) {
      // weights that one token tile reads leave L2 first; tokens, and weights that others read too, stay
      const uint64_t pol_w = a.t_tiles > 1 ? l2_policy_evict_last() : l2_policy_evict_first(), pol_x = l2_policy_evict_last();
      uint32_t parity = 1u;
      int s = 0, armed = 0;
#pragma unroll 1
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (!mbar_wait(smem_u32(&sh.empty[s]), parity, abort_flag)) break;
        const uint32_t full = smem_u32(&sh.full[s]), st = smem_u32(tiles) + (uint32_t)s * STAGE;
        mbar_expect_tx(full, STAGE);
        tma_load_2d(st, &tm_w, (k_first + kb) * L8_BK, n0, full, pol_w);
        tma_load_2d(st + L8_A, &tm_x, (k_first + kb) * L8_BK, t0, full, pol_x);
        armed = kb + 1;
        if (++s == a.stages) { s = 0; parity ^= 1u; }
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
        const int half = kb & 1;
        if (!mbar_wait(smem_u32(&sh.acc_empty[half]), (uint32_t)(kb >> 1 & 1) ^ 1u, abort_flag)) break;
        if (!mbar_wait(smem_u32(&sh.full[s]), parity, abort_flag)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t st = smem_u32(tiles) + (uint32_t)s * STAGE;
        const uint64_t a_desc = umma_desc_sw128(st), b_desc = umma_desc_sw128(st + L8_A);
#pragma unroll
        for (int k = 0; k < L8_BK / 32; ++k)      // 32 bytes further along the swizzled row: +2 in the 16-byte address field
          umma_e4m3(tmem_base + (uint32_t)(half * NT), a_desc + 2 * k, b_desc + 2 * k, idesc, k != 0);
        umma_commit(smem_u32(&sh.empty[s]));
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
    if constexpr (NT == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L8_REGS_ADD));
    float2 acc[COLS / 2];
  #pragma unroll
    for (int i = 0; i < COLS / 2; ++i) acc[i] = make_float2(0.f, 0.f);
    const int quad = warp & 3, col0 = (warp - L8_FIRST) / 4 * COLS;
    const uint32_t from = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)col0;
    bool ok = true;
#pragma unroll 1
    for (int kb = 0; kb < k_blocks; ++kb) {
      const int half = kb & 1, slot = kb % L8_SCALES;
      // tcgen05.ld is .sync.aligned: the lanes vote on the waits' answers
      ok = mbar_wait(smem_u32(&sh.sc_full[slot]), (uint32_t)(kb / L8_SCALES & 1), abort_flag);
      ok = ok && mbar_wait(smem_u32(&sh.acc_full[half]), (uint32_t)(kb >> 1 & 1), abort_flag);
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
        const float4* sc = reinterpret_cast<const float4*>(&scales[slot][col0 + c]);
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
        O* dst = out + (size_t)(t0 + col0) * a.N + n;
#pragma unroll
        for (int i = 0; i < COLS; ++i)
          if (t0 + col0 + i < a.T) dst[(size_t)i * a.N] = qb_from_float<O>(!ok ? __int_as_float(0x7fffffff) : i & 1 ? acc[i / 2].y : acc[i / 2].x);
      }
    } else if (ok) {
      // all products are done, so the ring is free: this block's sums [NT][128]
      float* part = reinterpret_cast<float*>(tiles);
#pragma unroll
      for (int i = 0; i < COLS; ++i) part[(col0 + i) * L8_M + quad * 32 + lane] = i & 1 ? acc[i / 2].y : acc[i / 2].x;
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (a.cut > 1) {
    cluster_sync_all();
    // a share of the columns, the blocks' parts in order; without the parts of a block that gave up it is no number
    int missing = 0;
    for (int r = 0; r < a.cut; ++r) missing |= __float_as_int(l8_remote(mapa_u32(smem_u32(&sh.abort_flag), (uint32_t)r)));
    const uint32_t part = smem_u32(tiles);
    const int share = (NT + a.cut - 1) / a.cut, c_end = min(min(NT, (rank + 1) * share), a.T - t0);
    for (int i = rank * share * L8_M + (int)threadIdx.x; i < c_end * L8_M; i += blockDim.x) {
      float sum = 0.f;
      for (int r = 0; r < a.cut; ++r) sum += l8_remote(mapa_u32(part + 4u * i, (uint32_t)r));
      const int n = n0 + i % L8_M;
      if (n < a.N) out[(size_t)(t0 + i / L8_M) * a.N + n] = qb_from_float<O>(missing ? __int_as_float(0x7fffffff) : sum);
    }
    cluster_sync_all();      // the parts stay until all have read them
  }
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM) : "memory");
  if (threadIdx.x == 0 && sh.abort_flag) qb_set_status(a.status, QB_STATUS_WAIT_TIMEOUT, tile, 11);
}

// [rows, K] e4m3, boxes of [box_rows, 128]
int map_e4m3(CUtensorMap* map, const void* base, uint64_t rows, uint64_t K, uint32_t box_rows) {
  const cuuint64_t dims[2] = {K, rows}, strides[1] = {K};
  const cuuint32_t box[2] = {L8_BK, box_rows};
  return make_map(map, base, 2, dims, strides, box, CU_TENSOR_MAP_DATA_TYPE_UINT8);
}

template <int NT, typename O>
int l8_launch(const CUtensorMap& tm_w, const CUtensorMap& tm_x, const LinearFp8& a, unsigned grid, size_t smem, cudaStream_t stream) {
  auto kern = linear_fp8_kernel<NT, O>;
  cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (err != cudaSuccess) return (int)err;
  if (NT == 256) {
    // the registers that the block's warps share out are those of the launch
    cudaFuncAttributes attr;
    err = cudaFuncGetAttributes(&attr, kern);
    if (err != cudaSuccess) return (int)err;
    if (attr.numRegs != L8_REGS_LAUNCH) return QB_ERR_UNSUPPORTED;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = l8_threads(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.cut;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  err = cudaLaunchKernelEx(&cfg, kern, tm_w, tm_x, a);
  return (int)err;
}

}  // namespace

extern "C" int qb_linear_fp8(const void* x, const float* xs, const void* w, const float* ws, void* out, int out_dtype, int T, int K, int N,
                             int* status, cudaStream_t stream) {
  if (T <= 0 || N <= 0) return 0;
  if (K <= 0 || K % 16 || (((uintptr_t)x | (uintptr_t)w) & 15)) return QB_ERR_BAD_ARG;
  int sms = 0;
  int rc = sm_count(sms);
  if (rc) return rc;
  const int NT = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : T <= 128 ? 128 : 256;
  LinearFp8 a{xs, ws, out, T, K, N};
  a.blocks = (K + L8_BK - 1) / L8_BK;
  a.t_tiles = (T + NT - 1) / NT;
  const long long tiles = (long long)((N + L8_M - 1) / L8_M) * a.t_tiles;
  a.cut = 1;
  while (a.cut < 8 && tiles * a.cut < sms && a.blocks >= 4 * a.cut) a.cut *= 2;
  a.per = (a.blocks + a.cut - 1) / a.cut;
  if (tiles * a.cut > 0x7fffffffll) return QB_ERR_UNSUPPORTED;
  a.status = status;
  const size_t stage = L8_A + (size_t)NT * L8_BK, need = a.cut > 1 ? (size_t)NT * L8_M * 4 : 0;
  // one block an SM where the accumulators fill half of the TMEM or more
  size_t room = NT >= 128 ? 200 * 1024 : 100 * 1024;
  int stages = (int)(room / stage);
  if (stages > L8_MAX_STAGES) stages = L8_MAX_STAGES;
  if (stages > a.per) stages = a.per;
  if (stages < 1) stages = 1;
  a.stages = stages;
  const size_t ring = stage * stages;
  const size_t smem = (ring > need ? ring : need) + 1024;
  CUtensorMap tm_w, tm_x;
  rc = map_e4m3(&tm_w, w, (uint64_t)N, (uint64_t)K, L8_M);
  if (rc) return rc;
  rc = map_e4m3(&tm_x, x, (uint64_t)T, (uint64_t)K, (uint32_t)NT);
  if (rc) return rc;
  const unsigned grid = (unsigned)(tiles * a.cut);
  QB_DISPATCH_DTYPE(out_dtype, O, {
    if (NT == 16) rc = l8_launch<16, O>(tm_w, tm_x, a, grid, smem, stream);
    else if (NT == 32) rc = l8_launch<32, O>(tm_w, tm_x, a, grid, smem, stream);
    else if (NT == 64) rc = l8_launch<64, O>(tm_w, tm_x, a, grid, smem, stream);
    else if (NT == 128) rc = l8_launch<128, O>(tm_w, tm_x, a, grid, smem, stream);
    else rc = l8_launch<256, O>(tm_w, tm_x, a, grid, smem, stream);
  });
  if (rc) return rc;
  QB_LAUNCH_CHECK();
  return 0;
}
