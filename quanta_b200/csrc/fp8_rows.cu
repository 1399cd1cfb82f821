// Rows that leave a norm, an activation or another kernel in e4m3 with a scale for every 128 columns (fp8.cuh): what a product in 8 bits reads.
//
// All of them are bound by memory; what 8 bits save is that the row passes it once, with one byte a number on the way out.
#include "fp8.cuh"

namespace {

// ---------------------------------------------------------------------------------------------
// Row r (token tok = rows[r] if rows != null, else r):
//   z = sum_s delta[tok, s, :]  (float32, s ascending);  with a gain g:  z = g * (z * rsqrt(mean(z^2) + eps_d))
//   x = h[tok, :] + z;  if store_h: h[tok, :] = x
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

// Rows of whole 32-byte pieces of at most 8,192 numbers: a thread keeps its 8 in registers from the load to the store, 16 threads hold a block
// of 128 and find its largest among themselves.
template <typename D, bool GAIN>
__global__ void __launch_bounds__(1024) norm_fp8_rows_kernel(NormFp8 a) {
  qb_follow();
  __shared__ float scratch[2][32];
  const int r = blockIdx.x, tok = a.rows != nullptr ? a.rows[r] : r, i = threadIdx.x * 8;
  const bool in = i < a.H;
  if (tok < 0 || tok >= a.T) {
    fp8_no_row(a, r);
    return;
  }
  float x[8], z[8], w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = z[e] = w[e] = 0.f;
  if (in) {
    QbVec8<float>::load(a.h + (size_t)tok * a.H + i, x);
    QbVec8<float>::load(a.w + i, w);
    if (a.delta != nullptr) {
      const D* d = (const D*)a.delta + (size_t)tok * a.S * a.H + i;
#pragma unroll 8
      for (int s = 0; s < a.S; ++s) {
        float dv[8];
        QbVec8<D>::load(d + (size_t)s * a.H, dv);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] += dv[e];
      }
    }
  }
  if (GAIN) {
    float g[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = 0.f;
    if (in) QbVec8<float>::load(a.g + i, g);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += z[e] * z[e];
    const float inv = rsqrtf(fp8_row_sum(ss, scratch[0]) / (float)a.H + a.eps_d);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = g[e] * (z[e] * inv);
  }
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] += z[e];
    ss += x[e] * x[e];
  }
  if (in && a.store_h && a.delta != nullptr) QbVec8<float>::store(a.h + (size_t)tok * a.H + i, x);
  const float inv = rsqrtf(fp8_row_sum(ss, scratch[1]) / (float)a.H + a.eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = w[e] * (x[e] * inv);
  const float top = fp8_block_largest(fp8_largest(x));
  if (!in) return;
  *reinterpret_cast<uint2*>(a.out + (size_t)r * a.H + i) = fp8_eight(x, FP8_TOP / top);
  if ((threadIdx.x & 15) == 0) a.scales[(size_t)(i / FP8_BLOCK) * a.n + r] = top / FP8_TOP;
}

// Any other row: held in shared memory between the passes, a warp a block of 128.
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
    const float up = FP8_TOP / top;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = b * FP8_BLOCK + e * 32 + lane;
      if (i < a.H) a.out[(size_t)r * a.H + i] = fp8_one(v[e] * up);
    }
    if (lane == 0) a.scales[(size_t)b * a.n + r] = top / FP8_TOP;
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

template <int KIND>
__device__ __forceinline__ float act_one(float g, float u, float limit, float alpha) {
  if (KIND == ACT_CLAMPED) {
    g = g > limit ? limit : g;                                        // (a NaN stays one)
    u = u > limit ? limit : u < -limit ? -limit : u;
    return g / (1.f + expf(-alpha * g)) * (u + 1.f);
  }
  if (KIND == ACT_GELU) return qb_gelu_tanh(g) * u;
  if (KIND == ACT_SILU) return g / (1.f + expf(-g)) * u;
  return g;
}

constexpr int ACT_THREADS = 256, ACT_COLS = ACT_THREADS * 8;
// VEC: whole 16-byte pieces.  Sixteen threads hold a block of 128 columns, eight numbers each; a thread takes the same columns of several rows.
template <typename T, int KIND, bool VEC>
__global__ void __launch_bounds__(ACT_THREADS) act_fp8_kernel(ActFp8 a) {
  qb_follow();
  const int c = blockIdx.x * ACT_COLS + threadIdx.x * 8;
  const int width = KIND == ACT_NONE ? a.I : 2 * a.I;
  const T* x = (const T*)a.x;
  for (int r = blockIdx.y; r < a.n; r += gridDim.y) {
    float g[8], u[8];
    const T* row = x + (size_t)r * width;
    if (VEC) {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = u[e] = 0.f;
      if (c < a.I) {
        QbVec8<T>::load(row + c, g);
        if (KIND != ACT_NONE) QbVec8<T>::load(row + a.I + c, u);
        if (KIND != ACT_NONE && a.bias != nullptr) {
          float bg[8], bu[8];
          QbVec8<float>::load(a.bias + c, bg);
          QbVec8<float>::load(a.bias + a.I + c, bu);
#pragma unroll
          for (int e = 0; e < 8; ++e) { g[e] += bg[e]; u[e] += bu[e]; }
        }
      }
    } else {
      // neighbouring threads take neighbouring numbers of the block
      const int c0 = c / FP8_BLOCK * FP8_BLOCK + (threadIdx.x & 15);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = c0 + e * 16;
        g[e] = i < a.I ? qb_to_float<T>(row[i]) : 0.f;
        u[e] = KIND != ACT_NONE && i < a.I ? qb_to_float<T>(row[a.I + i]) : 0.f;
        if (KIND != ACT_NONE && a.bias != nullptr && i < a.I) { g[e] += a.bias[i]; u[e] += a.bias[a.I + i]; }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = act_one<KIND>(g[e], u[e], a.limit, a.alpha);
    const float top = fp8_block_largest(fp8_largest(g)), up = FP8_TOP / top;
    if (VEC) {
      if (c < a.I) *reinterpret_cast<uint2*>(a.out + (size_t)r * a.I + c) = fp8_eight(g, up);
    } else {
      const int c0 = c / FP8_BLOCK * FP8_BLOCK + (threadIdx.x & 15);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c0 + e * 16 < a.I) a.out[(size_t)r * a.I + c0 + e * 16] = fp8_one(g[e] * up);
    }
    if ((threadIdx.x & 15) == 0 && c < a.I) a.scales[(size_t)(c / FP8_BLOCK) * a.n + r] = top / FP8_TOP;
  }
}

template <typename T, int KIND>
void act_fp8_launch(const ActFp8& a, bool vec, cudaStream_t stream) {
  const dim3 grid((a.I + ACT_COLS - 1) / ACT_COLS, a.n < 32768 ? a.n : 32768);
  if (vec) qb_launch(act_fp8_kernel<T, KIND, true>, grid, ACT_THREADS, 0, stream, a);
  else qb_launch(act_fp8_kernel<T, KIND, false>, grid, ACT_THREADS, 0, stream, a);
}

}  // namespace

extern "C" int qb_add_rmsnorm_fp8(float* h, const void* delta, int delta_dtype, int S, const float* w, const float* g, void* out, float* scales,
                                  const int* rows, int n_rows, int T, int H, float eps, float eps_d, int store_h, cudaStream_t stream) {
  if (n_rows <= 0 || H <= 0) return 0;
  if (g != nullptr && delta == nullptr) return QB_ERR_BAD_ARG;
  const NormFp8 a{h, delta, w, g, (uint8_t*)out, scales, rows, S, n_rows, T, H, eps, eps_d, store_h};
  if (H % 8 == 0 && H <= 8192 && (((uintptr_t)h | (uintptr_t)delta | (uintptr_t)w | (uintptr_t)g) & 15) == 0 && ((uintptr_t)out & 7) == 0) {
    const int threads = (H / 8 + 31) / 32 * 32;
    QB_DISPATCH_DTYPE(delta_dtype, D, {
      if (g != nullptr) qb_launch(norm_fp8_rows_kernel<D, true>, n_rows, threads, 0, stream, a);
      else qb_launch(norm_fp8_rows_kernel<D, false>, n_rows, threads, 0, stream, a);
    });
    QB_LAUNCH_CHECK();
    return 0;
  }
  const size_t smem = (size_t)H * sizeof(float);
  if (smem > 200 * 1024) return QB_ERR_UNSUPPORTED;
  QB_DISPATCH_DTYPE(delta_dtype, D, {
    auto kern = norm_fp8_any_kernel<D>;
    if (smem > 48 * 1024) {
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
