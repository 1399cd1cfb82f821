// The product of linear_fp8.cu for few tokens, of a small matrix for more: bound by the bytes of w, and by what a launch costs besides them.
//
// A block takes 16 rows of w, its warps blocks of 128 k (one scale each) in turn.  A lane loads the 32 numbers of a row's 128 that it
// then multiplies (the order of k inside an mma is free as long as both operands have it), 32 bytes a load, so that weights go from memory to
// registers without shared memory, a barrier or tensor memory.  The four mma.sync of a block of 128 sum its products (of 8 bits each) in
// float32, the sum is scaled by token and weight block and added in float32; the warps' parts are added in the order of the warps, so a
// row's bits are the same in every step of as many warps a block.
//
// Measured on a B200, one product after another in a graph, weights from memory, microseconds (bytes at 6.5 TB/s / this / tcgen05):
//   one token    4,096 x 22,016 13.8 / 18.5 / 18.5, 512 x 29,000 2.3 / 6.1 / 5.9, 1,024 x 200,000 (4 tokens) 31.3 / 40.8 / 39.9, 16 x 200,000 0.5 / 20.3 / 11.9
//   8 tokens     4,096 x 4,096 2.6 / 5.5 / 7.8, 2,048 x 2,048 0.6 / 2.1 / 5.1, 1,024 x 1,024 0.2 / 1.7 / 4.4
//   16           4,096 x 4,096 2.6 / 6.6 / 7.9, 2,048 x 11,264 3.5 / 9.1 / 8.9, 4,096 x 22,016 13.8 / 22.4 / 18.7
//   32           2,048 x 2,048 0.6 / 3.4 / 5.6, 4,096 x 2,048 1.3 / 5.2 / 7.0, 2,048 x 4,096 1.3 / 6.5 / 5.9, 4,096 x 4,096 2.6 / 10.7 / 8.2
//   64           1,024 x 1,024 0.2 / 2.4 / 5.7, 2,048 x 2,048 0.6 / 6.4 / 6.6, 2,048 x 4,096 1.3 / 10.8 / 7.0
//   128          1,024 x 1,024 0.2 / 4.3 / 6.0, 1,024 x 2,048 0.3 / 7.4 / 6.0;   256: 2,048 x 512 0.2 / 6.3 / 8.0;   1,000: 512 x 64 0 / 2.0 / 4.6
// What tcgen05 takes more of a small matrix are the barriers, the tensor memory, the maps and a cluster's parts before and behind the bytes.  One token of a
// large matrix is bound by the bytes, waves of blocks at a time: 4,096 x 9,472 (592 blocks, four an SM) 9.3 us, 18,944 16.0, 28,416 22.3, 37,888 28.3, 56,832 40.3,
// so 3.1 us of start and end and 6.2 a full wave (38.8 MB, 0.96 of the rate of a copy); 22,016 is 2.3 waves and pays 1.2 us for the part (18.7).  With more
// tokens it is the issue of instructions (154 a warp for 2 KB and 8 tokens: e4m3 operands of mma.sync are converted to fp16 first).  Blocks that walk over the rows, with the next rows' weights on their way, took the same time; four pieces ahead instead of two a
// longer one in blocks of four warps (fewer of them).  Weights asked for before the launch ahead has ended (`early`): norm, product, activation and product of 4,096 x 11,008 for
// one token 33.0 -> 32.2 us, for 32 38.1 -> 35.8, of 2,048 x 5,632 15.0 -> 13.7 and 22.5 -> 21.1.
#include "fp8.cuh"

namespace {

struct LinearFp8Few {
  const uint8_t *x, *w;
  const float *xs, *ws;
  void* out;
  int T, K, N, blocks, early;
};
struct alignas(16) L8Piece {
  uint32_t u[8];
};

// 32 bytes of a row, of which `left` (a multiple of 16) exist; WIDE: on 32 bytes and all there.  Weights are read once: not kept in L1.
template <bool WIDE, bool ONCE>
__device__ __forceinline__ L8Piece l8f_load(const uint8_t* p, int left) {
  L8Piece v = {};
  if (WIDE) {
    if (left > 0) {
      if (ONCE)
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v.u[0]), "=r"(v.u[1]), "=r"(v.u[2]), "=r"(v.u[3]), "=r"(v.u[4]), "=r"(v.u[5]), "=r"(v.u[6]), "=r"(v.u[7]) : "l"(p));
      else
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v.u[0]), "=r"(v.u[1]), "=r"(v.u[2]), "=r"(v.u[3]), "=r"(v.u[4]), "=r"(v.u[5]), "=r"(v.u[6]), "=r"(v.u[7]) : "l"(p));
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (left > 16 * h)
        asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.u[4 * h]), "=r"(v.u[4 * h + 1]), "=r"(v.u[4 * h + 2]), "=r"(v.u[4 * h + 3]) : "l"(p + 16 * h));
  }
  return v;
}

__device__ __forceinline__ void l8f_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: tiles of 8 tokens.  D, XD: pieces of w and of x (with the scales) a warp holds ahead.
template <int NT, int D, int XD, int WARPS, int MINB, bool WIDE, typename O>
__global__ void __launch_bounds__(WARPS * 32, MINB) linear_fp8_tokens_kernel(LinearFp8Few a) {
  static_assert(D % XD == 0, "the ring of x divides the ring of w");
  if (!a.early) qb_follow();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, t0 = blockIdx.y * NT * 8;
  const uint8_t* wr[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) wr[h] = a.w + (size_t)min(n0 + h * 8 + g, a.N - 1) * a.K + t * 32;
  const uint8_t* xr[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) xr[n] = a.x + (size_t)min(t0 + n * 8 + g, a.T - 1) * a.K + t * 32;
  const float* ws = a.ws + (size_t)(n0 / FP8_BLOCK) * a.blocks;
  L8Piece wb[D][2], xb[XD][NT];
  float xsb[XD][NT][2], wsb[XD];
  auto fetch_w = [&](int kb, L8Piece (&b)[2]) {
    const int left = kb < a.blocks ? a.K - kb * FP8_BLOCK - t * 32 : 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) b[h] = l8f_load<WIDE, true>(wr[h] + kb * FP8_BLOCK, left);
  };
  auto fetch_x = [&](int kb, int at) {
    const int left = kb < a.blocks ? a.K - kb * FP8_BLOCK - t * 32 : 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      xb[at][n] = l8f_load<WIDE, false>(xr[n] + kb * FP8_BLOCK, left);
      // the scales of the tokens whose sums this lane has
#pragma unroll
      for (int i = 0; i < 2; ++i) xsb[at][n][i] = kb < a.blocks ? a.xs[(size_t)kb * a.T + min(t0 + n * 8 + 2 * t + i, a.T - 1)] : 0.f;
    }
    wsb[at] = kb < a.blocks ? ws[kb] : 0.f;
  };
#pragma unroll
  for (int d = 0; d < D; ++d) fetch_w(warp + d * WARPS, wb[d]);
  if (a.early) qb_follow();
#pragma unroll
  for (int d = 0; d < XD; ++d) fetch_x(warp + d * WARPS, d);
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  for (int k0 = warp; k0 < a.blocks; k0 += D * WARPS) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int kb = k0 + d * WARPS;
      if (kb >= a.blocks) break;
      float c[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[n][i] = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          l8f_mma(c[n], wb[d][0].u[2 * s], wb[d][1].u[2 * s], wb[d][0].u[2 * s + 1], wb[d][1].u[2 * s + 1], xb[d % XD][n].u[2 * s], xb[d % XD][n].u[2 * s + 1]);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = fmaf(c[n][i], xsb[d % XD][n][i & 1] * wsb[d % XD], acc[n][i]);
      fetch_w(kb + D * WARPS, wb[d]);
      fetch_x(kb + XD * WARPS, d % XD);
    }
  }
  // the warps' parts, added in the order of the warps
  constexpr int PAD = 20, TOK = NT * 8;
  __shared__ float part[WARPS][TOK][PAD];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][n * 8 + 2 * t + (i & 1)][g + 8 * (i >> 1)] = acc[n][i];
  __syncthreads();
  for (int v = threadIdx.x; v < TOK * 16; v += WARPS * 32) {
    const int tok = t0 + v / 16, row = v % 16;
    if (tok >= a.T || n0 + row >= a.N) continue;
    float s = part[0][v / 16][row];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) s += part[w][v / 16][row];
    reinterpret_cast<O*>(a.out)[(size_t)tok * a.N + n0 + row] = qb_from_float<O>(s);
  }
}

template <int NT, int D, int XD, int WARPS, int MINB, typename O>
void l8f_launch(const LinearFp8Few& a, cudaStream_t stream) {
  const dim3 grid((a.N + 15) / 16, (a.T + NT * 8 - 1) / (NT * 8));
  if (a.K % 32 == 0 && (((uintptr_t)a.x | (uintptr_t)a.w) & 31) == 0) qb_launch(linear_fp8_tokens_kernel<NT, D, XD, WARPS, MINB, true, O>, grid, WARPS * 32, 0, stream, a);
  else qb_launch(linear_fp8_tokens_kernel<NT, D, XD, WARPS, MINB, false, O>, grid, WARPS * 32, 0, stream, a);
}

}  // namespace

// Whether products of T tokens and a [N, K] matrix are this kernel's.  Up to 8 tokens all but those of very many short rows; more as long as its
// blocks are few for their length, blocks x (K + 4,096) at most 3 x 2^20, by the times above and those of some 200 sizes (K 256 to 11,008, N 512 to 10,000, 9 to 256
// tokens), of which none is off by more than some tenth (32 tokens, 2,048 x 4,096, which lies on the line: 6.5 us, tcgen05 5.9).
bool qb_linear_fp8_tokens_takes(int T, int K, int N) {
  if (T <= 8) return K >= 1024 || N <= 30000;
  const long long blocks = (long long)((N + 15) / 16) * ((T + 15) / 16);
  return blocks * (K + 4096ll) <= 3 << 20;
}

// K a multiple of 16, x and w on 16 bytes (linear_fp8.cu has looked).  Blocks of four warps where there are two for every SM or
// more, else of eight, so that few blocks have as many bytes on their way, and three pieces ahead
// (one token, 5,632 x 2,048 4.3 -> 3.8 us, 16,384 x 2,048 12.0 -> 10.5).  Four blocks an SM, or five, with less ahead, where that is one wave instead of two (4,096 x
// 11,008 12.3 -> 10.9 us; 4,096 x 14,336 13.6 and 15.8, 4,096 x 22,016 18.7 and 19.0).  More than 16 tokens: tiles of 16, two blocks an SM; of 32, one an SM, where
// those are one wave and tiles of 16 would be more than a block an SM (32 tokens, 2,048 x 2,048: 3.4 us, with 16 3.7; 4,096 x 1,024: 4.5 and 3.6).
int qb_linear_fp8_tokens(const void* x, const float* xs, const void* w, const float* ws, void* out, int out_dtype, int T, int K, int N, int early,
                         int sms, cudaStream_t stream) {
  const LinearFp8Few a{(const uint8_t*)x, (const uint8_t*)w, xs, ws, out, T, K, N, (K + FP8_BLOCK - 1) / FP8_BLOCK, early};
  const int across = (N + 15) / 16;
  const bool many = across >= 2 * sms, wide = (long long)across * ((T + 15) / 16) > sms && (long long)across * ((T + 31) / 32) <= sms;
  QB_DISPATCH_DTYPE(out_dtype, O, {
    if (T <= 8 && many && across > 4 * sms && across <= 5 * sms) l8f_launch<1, 2, 1, 4, 5, O>(a, stream);
    else if (T <= 8 && many) l8f_launch<1, 2, 2, 4, 4, O>(a, stream);
    else if (T <= 8) l8f_launch<1, 3, 3, 8, 2, O>(a, stream);
    else if (T <= 16 && many) l8f_launch<2, 2, 2, 4, 4, O>(a, stream);
    else if (T <= 16 || !wide) l8f_launch<2, 2, 2, 8, 2, O>(a, stream);
    else l8f_launch<4, 2, 2, 8, 1, O>(a, stream);
  });
  QB_LAUNCH_CHECK();
  return 0;
}
