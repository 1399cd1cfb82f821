// Rows that leave a norm, an activation or another kernel in e4m3 with a scale for every 128 columns (fp8.cuh): what a product in 8 bits reads.
//
// All of them are bound by memory; what 8 bits save is that the row passes it once, with one byte a number on the way out.  Measured on a B200, one
// after another in a graph: norm of 8,192 x 4,096 with two float32 slots 88 us (6.5 TB/s), one row 2.4 us, of 6,311 x 2,434 (rows that do not lie on 16 bytes) with a bfloat16 addend 34 us (5.0 TB/s);
// plain rows of 8,192 x 11,008 bfloat16 42 us (6.5 TB/s), one row 1.3 us; activation of 8,192 x 11,008 bfloat16, clamped with
// biases 82 us (5.5 TB/s), silu without 70 (6.5 TB/s), one row 1.6 us.
#include "fp8.cuh"

namespace {

// ---------------------------------------------------------------------------------------------
// Row r (token tok = rows[r] if rows != null, else r):
//   x = h[tok, :] + sum_s delta[tok, s, :]  (float32, s ascending), or, with a gain g, h[tok, :] + g * (z * rsqrt(mean(z^2) + eps_d)) of their sum z;  if store_h: h[tok, :] = x
//   out[r, :], scales[:, r] = e4m3 of w * (x * rsqrt(mean(x^2) + eps))
// A tok outside the T rows of h gives a row of NaN.
// ---------------------------------------------------------------------------------------------
struct NormFp8 {
  float* h;
  const void* delta;
  const float *w, *g;
  uint8_t* out;
  float* scales;
  const int* rows;
  int S, n, T, H;
  float eps, eps_d;
  int store_h;
};

// Sum over the block, warps in index order; `scratch` (32 floats) is used by no other sum.
__device__ __forceinline__ float fp8_row_sum(float v, float* scratch) {
  const int lane = threadIdx.x & 31, n = blockDim.x >> 5;
  v = qb_warp_sum(v);
  if (lane == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  return qb_warp_sum(lane < n ? scratch[lane] : 0.f);
}

__device__ __forceinline__ void fp8_no_row(const NormFp8& a, int r) {
  for (int i = threadIdx.x; i < a.H; i += blockDim.x) {
    a.out[(size_t)r * a.H + i] = 0x7f;
    if (i % FP8_BLOCK == 0) a.scales[(size_t)(i / FP8_BLOCK) * a.n + r] = __int_as_float(0x7fffffff);
  }
}

// A thread's eight numbers of a row: eight neighbours from column i on, or (rows of no whole, aligned pieces) every sixteenth of a block from i on, of
// which `left` exist, 16 apart.
template <bool VEC, typename D>
__device__ __forceinline__ void fp8_load8(const D* row, int i, int left, float (&v)[8]) {
  if constexpr (VEC) {
    QbVec8<D>::load(row + i, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e * 16 < left ? qb_to_float<D>(row[i + e * 16]) : 0.f;
  }
}
// x += the slots' eight numbers, slots in order
template <bool VEC, typename D>
__device__ __forceinline__ void fp8_add_slots(const NormFp8& a, int tok, int i, float (&x)[8]) {
  const D* d = (const D*)a.delta + (size_t)tok * a.S * a.H;
#pragma unroll 2
  for (int s = 0; s < a.S; ++s) {
    float dv[8];
    fp8_load8<VEC, D>(d + (size_t)s * a.H, i, a.H - i, dv);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += dv[e];
  }
}

// Rows of at most 8,192 numbers: a thread keeps its 8 in registers from the load to the store, 16 threads hold a block of 128 and find its largest
// among themselves.  VEC: rows of whole 32-byte pieces.
// MOST: threads at most.  Without a gain the registers are held down to 32, so that an SM has the bytes of four rows on their way (8,192 rows of 4,096,
// two float32 slots: 97 us with 40, 88 with 32; with a gain, and 40 instead of 56, they spill: 45 -> 59 us at 2,048).
template <typename D, bool GAIN, int MOST, bool VEC>
__global__ void __launch_bounds__(MOST, (GAIN || !VEC) && MOST == 1024 ? 1 : 2) norm_fp8_rows_kernel(NormFp8 a) {
  qb_follow();
  __shared__ float scratch[2][32];
  const int r = blockIdx.x, tok = a.rows != nullptr ? a.rows[r] : r, i = VEC ? threadIdx.x * 8 : threadIdx.x / 16 * FP8_BLOCK + threadIdx.x % 16;
  const bool in = i < a.H;
  if (tok < 0 || tok >= a.T) {
    fp8_no_row(a, r);
    return;
  }
  float x[8], w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  if (GAIN) {
    float z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = w[e] = 0.f;
    if (in) {
      fp8_load8<VEC, float>(a.h + (size_t)tok * a.H, i, a.H - i, x);
      fp8_load8<VEC, float>(a.g, i, a.H - i, w);
      fp8_add_slots<VEC, D>(a, tok, i, z);
    }
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += z[e] * z[e];
    const float inv = rsqrtf(fp8_row_sum(ss, scratch[0]) / (float)a.H + a.eps_d);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += w[e] * (z[e] * inv);
  } else if (in) {
    fp8_load8<VEC, float>(a.h + (size_t)tok * a.H, i, a.H - i, x);
    if (a.delta != nullptr) fp8_add_slots<VEC, D>(a, tok, i, x);
  }
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
  if (in && a.store_h && a.delta != nullptr) {
    float* h = a.h + (size_t)tok * a.H + i;
    if constexpr (VEC) {
      QbVec8<float>::store(h, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e * 16 < a.H) h[e * 16] = x[e];
    }
  }
  // the gains are every block's, so they are near; asked for before the sum
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = 0.f;
  if (in) fp8_load8<VEC, float>(a.w, i, a.H - i, w);
  const float inv = rsqrtf(fp8_row_sum(ss, scratch[1]) / (float)a.H + a.eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = w[e] * (x[e] * inv);
  const float top = fp8_block_largest(fp8_largest(x));
  if (!in) return;
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(a.out + (size_t)r * a.H + i) = fp8_eight(x, fp8_up(top));
  } else {
    const float up = fp8_up(top);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e * 16 < a.H) a.out[(size_t)r * a.H + i + e * 16] = fp8_one(x[e] * up);
  }
  if ((threadIdx.x & 15) == 0) a.scales[(size_t)(i / FP8_BLOCK) * a.n + r] = fp8_scale(top);
}

// Longer rows: held in shared memory between the passes, a warp a block of 128.  Number by number, so some 2.3 times the bytes' time (one float32
// addend, 4,096 x 12,288: 233 us, the bytes 100; 2,048 x 20,000: 249 and 81; one row of 8,200 9.4 us): no model here is as wide.
template <typename D>
__global__ void __launch_bounds__(512) norm_fp8_any_kernel(NormFp8 a) {
  extern __shared__ float row[];      // H floats
  __shared__ float scratch[2][32];
  const int r = blockIdx.x, tok = a.rows != nullptr ? a.rows[r] : r;
  if (tok < 0 || tok >= a.T) {
    fp8_no_row(a, r);
    return;
  }
  float* h = a.h + (size_t)tok * a.H;
  const D* d = a.delta != nullptr ? (const D*)a.delta + (size_t)tok * a.S * a.H : nullptr;
  auto sum_of = [&](int i) {
    float z = 0.f;
    for (int s = 0; s < a.S; ++s) z += qb_to_float<D>(d[(size_t)s * a.H + i]);
    return z;
  };
  float ss = 0.f;
  if (a.g != nullptr) {
    for (int i = threadIdx.x; i < a.H; i += blockDim.x) {
      row[i] = sum_of(i);
      ss += row[i] * row[i];
    }
    const float inv = rsqrtf(fp8_row_sum(ss, scratch[0]) / (float)a.H + a.eps_d);
    ss = 0.f;
    for (int i = threadIdx.x; i < a.H; i += blockDim.x) {
      row[i] = h[i] + a.g[i] * (row[i] * inv);
      ss += row[i] * row[i];
    }
  } else {
    for (int i = threadIdx.x; i < a.H; i += blockDim.x) {
      row[i] = d != nullptr ? h[i] + sum_of(i) : h[i];
      ss += row[i] * row[i];
    }
  }
  if (a.store_h && d != nullptr)
    for (int i = threadIdx.x; i < a.H; i += blockDim.x) h[i] = row[i];
  const float inv = rsqrtf(fp8_row_sum(ss, scratch[1]) / (float)a.H + a.eps);
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int b = threadIdx.x >> 5; b * FP8_BLOCK < a.H; b += blockDim.x >> 5) {
    float v[4], top = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = b * FP8_BLOCK + e * 32 + lane;
      v[e] = i < a.H ? a.w[i] * (row[i] * inv) : 0.f;
      top = fp8_max(top, fabsf(v[e]));
    }
    top = fp8_max(top, __shfl_xor_sync(0xffffffffu, top, 16));
    top = fp8_block_largest(top);
    const float up = fp8_up(top);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = b * FP8_BLOCK + e * 32 + lane;
      if (i < a.H) a.out[(size_t)r * a.H + i] = fp8_one(v[e] * up);
    }
    if (lane == 0) a.scales[(size_t)b * a.n + r] = fp8_scale(top);
  }
}

// ---------------------------------------------------------------------------------------------
// v = act(x[r, c] + bias[c]) * (x[r, I + c] + bias[I + c])  (the activations of glu_act), or, kind 3, v = x[r, c]; out, scales = e4m3 of v.
// ---------------------------------------------------------------------------------------------
constexpr int ACT_SILU = 0, ACT_CLAMPED = 1, ACT_GELU = 2, ACT_NONE = 3;
struct ActFp8 {
  const void* x;
  const float* bias;
  uint8_t* out;
  float* scales;
  int n, I;
  float limit, alpha;
};

__device__ __forceinline__ float fp8_min(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The exponential and the reciprocal are the fast ones (some 2 ulp, and 2^-23 of the argument; a sigmoid below 2^-126 is zero): what follows is rounded to
// four bits.
__device__ __forceinline__ float2 fp8_sigmoid2(float2 g, float by) {      // 1 / (1 + e^(-g by / log2 e))
  const float2 z = fp8_mul2(g, make_float2(-by, -by));
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(z.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(z.y));
  e = fp8_add2(e, make_float2(1.f, 1.f));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e.x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e.y));
  return e;
}
// Two numbers at a time: the kernel is bound by the issue of instructions (an activation with biases and clamps) as much as by memory.
template <int KIND>
__device__ __forceinline__ float2 act_two(float2 g, float2 u, float limit, float alpha) {
  constexpr float LOG2E = 1.4426950408889634f;
  if (KIND == ACT_CLAMPED) {
    g = make_float2(fp8_min(g.x, limit), fp8_min(g.y, limit));      // (a NaN stays one)
    u = make_float2(fp8_max(fp8_min(u.x, limit), -limit), fp8_max(fp8_min(u.y, limit), -limit));
    const float2 t = fp8_mul2(g, fp8_sigmoid2(g, alpha * LOG2E));
    return fp8_fma2(u, t, t);
  }
  if (KIND == ACT_GELU) {      // as qb_gelu_tanh
    const float2 t = fp8_fma2(fp8_mul2(g, g), fp8_mul2(g, make_float2(0.044715f, 0.044715f)), g);
    return fp8_mul2(fp8_mul2(g, fp8_sigmoid2(t, 1.5957691216057308f * LOG2E)), u);
  }
  if (KIND == ACT_SILU) return fp8_mul2(fp8_mul2(g, fp8_sigmoid2(g, LOG2E)), u);
  return g;
}

// Sixteen threads hold a block of 128 columns, eight numbers each, and take the same columns of neighbouring rows: the biases stay in registers,
// the numbers of several rows (128 bytes a thread) are on their way together, and the rows' scales of a block are neighbours.  VEC: whole 16-byte
// pieces; else neighbouring threads take neighbouring numbers of the block (8,192 x 11,007 bfloat16, silu 113 us, 69 on whole pieces; two or four rows on
// their way 118 and 170).  A block spans 2,048 columns, so in narrower rows threads have nothing to do (8,192 rows bfloat16, silu: 512 columns 14.5 us, the
// bytes 3.2; 1,408 15.5 and 8.8; 2,056 21.3 and 12.9; plain rows of 512 9.4 and 1.9).
constexpr int ACT_THREADS = 256, ACT_COLS = ACT_THREADS * 8, ACT_ROWS = 8;
template <typename T, int KIND, bool BIAS, bool VEC>
__global__ void __launch_bounds__(ACT_THREADS) act_fp8_kernel(ActFp8 a, int rows_each) {
  qb_follow();
  constexpr int AHEAD = !VEC ? 1 : sizeof(T) == 2 ? 4 : 2, PIECES = VEC ? (int)sizeof(T) / 2 : 1;
  const int c = blockIdx.x * ACT_COLS + threadIdx.x * 8, c0 = c / FP8_BLOCK * FP8_BLOCK + (threadIdx.x & 15);
  const bool in = c < a.I;
  const size_t width = KIND == ACT_NONE ? a.I : 2 * (size_t)a.I;
  auto column = [&](int e) { return VEC ? c + e : c0 + e * 16; };
  float bg[8], bu[8];
  if (BIAS) {
    if (VEC && in) {
      QbVec8<float>::load(a.bias + c, bg);
      QbVec8<float>::load(a.bias + a.I + c, bu);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool has = !VEC && column(e) < a.I;
        bg[e] = has ? a.bias[column(e)] : 0.f;
        bu[e] = has ? a.bias[a.I + column(e)] : 0.f;
      }
    }
  }
  const int r_end = min(a.n, ((int)blockIdx.y + 1) * rows_each);
#pragma unroll 1
  for (int r0 = blockIdx.y * rows_each; r0 < r_end; r0 += AHEAD) {
    uint4 raw[AHEAD][2][PIECES];
    if (VEC) {
#pragma unroll
      for (int d = 0; d < AHEAD; ++d)
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
          raw[d][0][p] = raw[d][1][p] = make_uint4(0u, 0u, 0u, 0u);
          if (!in || r0 + d >= r_end) continue;
          const uint4* row = reinterpret_cast<const uint4*>((const T*)a.x + (size_t)(r0 + d) * width + c);
          raw[d][0][p] = row[p];
          if (KIND != ACT_NONE) raw[d][1][p] = row[(size_t)a.I * sizeof(T) / 16 + p];
        }
    }
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {
      const int r = r0 + d;
      if (r >= r_end) break;
      float g[8], u[8];
      if (VEC) {
        QbVec8<T>::load(reinterpret_cast<const T*>(raw[d][0]), g);
        QbVec8<T>::load(reinterpret_cast<const T*>(raw[d][1]), u);
      } else {
        // (all are asked for before the first is looked at)
        const T* row = (const T*)a.x + (size_t)r * width;
        T one[2][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = column(e);
          one[0][e] = one[1][e] = qb_from_float<T>(0.f);
          if (i < a.I) {
            one[0][e] = row[i];
            if (KIND != ACT_NONE) one[1][e] = row[a.I + i];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          g[e] = qb_to_float<T>(one[0][e]);
          u[e] = qb_to_float<T>(one[1][e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float2 g2 = make_float2(g[e], g[e + 1]), u2 = make_float2(u[e], u[e + 1]);
        if (BIAS) {
          g2 = fp8_add2(g2, make_float2(bg[e], bg[e + 1]));
          u2 = fp8_add2(u2, make_float2(bu[e], bu[e + 1]));
        }
        g2 = act_two<KIND>(g2, u2, a.limit, a.alpha);
        g[e] = g2.x;
        g[e + 1] = g2.y;
      }
      const float top = fp8_block_largest(fp8_largest(g)), up = fp8_up(top);
      if (VEC) {
        if (in) *reinterpret_cast<uint2*>(a.out + (size_t)r * a.I + c) = fp8_eight(g, up);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (column(e) < a.I) a.out[(size_t)r * a.I + column(e)] = fp8_one(g[e] * up);
      }
      if ((threadIdx.x & 15) == 0 && in) a.scales[(size_t)(c / FP8_BLOCK) * a.n + r] = fp8_scale(top);
    }
  }
}

template <typename T, int KIND, bool BIAS>
void act_fp8_launch(const ActFp8& a, bool vec, cudaStream_t stream) {
  // few rows: one a block, so that more SMs take part; a grid has 65,535 rows of blocks at most
  const int across = (a.I + ACT_COLS - 1) / ACT_COLS;
  int rows = (long long)a.n * across >= 148 * 8 * ACT_ROWS ? ACT_ROWS : 1;
  while ((a.n + rows - 1) / rows > 65535) rows *= 2;
  const dim3 grid(across, (a.n + rows - 1) / rows);
  if (vec) qb_launch(act_fp8_kernel<T, KIND, BIAS, true>, grid, ACT_THREADS, 0, stream, a, rows);
  else qb_launch(act_fp8_kernel<T, KIND, BIAS, false>, grid, ACT_THREADS, 0, stream, a, rows);
}
template <typename T, int KIND>
void act_fp8_launch(const ActFp8& a, bool vec, cudaStream_t stream) {
  if (KIND != ACT_NONE && a.bias != nullptr) act_fp8_launch<T, KIND, KIND != ACT_NONE>(a, vec, stream);
  else act_fp8_launch<T, KIND, false>(a, vec, stream);
}

}  // namespace

extern "C" int qb_add_rmsnorm_fp8(float* h, const void* delta, int delta_dtype, int S, const float* w, const float* g, void* out, float* scales,
                                  const int* rows, int n_rows, int T, int H, float eps, float eps_d, int store_h, cudaStream_t stream) {
  if (n_rows <= 0 || H <= 0) return 0;
  if (g != nullptr && delta == nullptr) return QB_ERR_BAD_ARG;
  const NormFp8 a{h, delta, w, g, (uint8_t*)out, scales, rows, S, n_rows, T, H, eps, eps_d, store_h};
  if (H <= 8192) {
    const bool vec = H % 8 == 0 && (((uintptr_t)h | (uintptr_t)delta | (uintptr_t)w | (uintptr_t)g) & 15) == 0 && ((uintptr_t)out & 7) == 0;
    const int threads = ((H + FP8_BLOCK - 1) / FP8_BLOCK * 16 + 31) / 32 * 32;
    QB_DISPATCH_DTYPE(delta_dtype, D, {
      if (!vec && g != nullptr) qb_launch(norm_fp8_rows_kernel<D, true, 1024, false>, n_rows, threads, 0, stream, a);
      else if (!vec) qb_launch(norm_fp8_rows_kernel<D, false, 1024, false>, n_rows, threads, 0, stream, a);
      else if (g != nullptr && threads <= 512) qb_launch(norm_fp8_rows_kernel<D, true, 512, true>, n_rows, threads, 0, stream, a);
      else if (g != nullptr) qb_launch(norm_fp8_rows_kernel<D, true, 1024, true>, n_rows, threads, 0, stream, a);
      else qb_launch(norm_fp8_rows_kernel<D, false, 1024, true>, n_rows, threads, 0, stream, a);
    });
    QB_LAUNCH_CHECK();
    return 0;
  }
  const size_t smem = (size_t)H * sizeof(float);
  if (smem > 200 * 1024) return QB_ERR_UNSUPPORTED;
  QB_DISPATCH_DTYPE(delta_dtype, D, {
    auto kern = norm_fp8_any_kernel<D>;
    if (smem + 1024 > 48 * 1024) {      // (the kernel also has some static shared memory)
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return (int)e;
    }
    kern<<<n_rows, 512, smem, stream>>>(a);
  });
  QB_LAUNCH_CHECK();
  return 0;
}

extern "C" int qb_act_fp8(const void* x, int dtype, const float* bias, void* out, float* scales, int n_rows, int I, int kind, float limit,
                          float alpha, cudaStream_t stream) {
  if (n_rows <= 0 || I <= 0) return 0;
  if (kind < 0 || kind > ACT_NONE) return QB_ERR_BAD_ARG;
  const ActFp8 a{x, bias, (uint8_t*)out, scales, n_rows, I, limit, alpha};
  const bool vec = I % 8 == 0 && (((uintptr_t)x | (uintptr_t)bias) & 15) == 0 && ((uintptr_t)out & 7) == 0;
  QB_DISPATCH_DTYPE(dtype, T, {
    if (kind == ACT_SILU) act_fp8_launch<T, ACT_SILU>(a, vec, stream);
    else if (kind == ACT_CLAMPED) act_fp8_launch<T, ACT_CLAMPED>(a, vec, stream);
    else if (kind == ACT_GELU) act_fp8_launch<T, ACT_GELU>(a, vec, stream);
    else act_fp8_launch<T, ACT_NONE>(a, vec, stream);
  });
  QB_LAUNCH_CHECK();
  return 0;
}
