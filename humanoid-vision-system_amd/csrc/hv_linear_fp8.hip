// c = act(a_scale w_scale (a . w^T) + bias) for rows of e4m3 codes with one fp32 scale per row of a and of w
// (nn.Linear on 8-bit rows, e.g. the MLP of vit_encoder_decoder.py:146-152).
//
// The codes go to the matrix cores as they are (32x32x64 tiles of 8-bit floats, unit block scales, fp32 sums); both
// scales, the bias and the activation are applied to the fp32 sums before the one rounding to the output type.
#include "hv_common.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int NT = 256;
constexpr int UNIT = 0x7f7f7f7f;                          // block scales 2^0

struct LinArgs {
  const unsigned char *a, *w;
  long lda, ldw, m, ldc;
  int n, k, act;
  const float *as, *ws, *bias;
  void* c;
};

__device__ __forceinline__ f32x16 mma(i32x8 a, i32x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, UNIT, 0, UNIT);
}

// an LDS tile has rows of 128 codes; the 16-byte chunk c of a row lies at c ^ (row & 7)
constexpr int BK = 128;
__device__ __forceinline__ u32x4 chunk(const unsigned char* tile, int row, int c) {
  return *(const u32x4*)(tile + row * BK + ((c ^ (row & 7)) << 4));
}
// operand of k-step ks (64 codes): lane (row = lane & 31, half = lane >> 5) holds chunks 4 ks + 2 half, + 1.  Any
// numbering of the contraction index serves that a and w share.
__device__ __forceinline__ i32x8 operand(const unsigned char* tile, int row, int ks, int half) {
  union { u32x4 q[2]; i32x8 v; } u;
  u.q[0] = chunk(tile, row, 4 * ks + 2 * half);
  u.q[1] = chunk(tile, row, 4 * ks + 2 * half + 1);
  return u.v;
}

template <typename T>
__global__ void __launch_bounds__(NT) k_linear_fp8(const LinArgs p) {
  constexpr int BM = 128, BN = 128;
  __shared__ __align__(16) unsigned char sm[(BM + BN) * BK];
  unsigned char *ta = sm, *tw = sm + BM * BK;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, r31 = lane & 31;
  const long m0 = (long)blockIdx.y * BM;
  const int n0 = blockIdx.x * BN, wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[i][j][x] = 0.f;
  u32x4 ra[4], rw[4];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int id = threadIdx.x + i * NT, row = id >> 3, k = k0 + (id & 7) * 16;
      ra[i] = m0 + row < p.m && k < p.k ? *(const u32x4*)(p.a + (m0 + row) * p.lda + k) : u32x4{0, 0, 0, 0};
      rw[i] = n0 + row < p.n && k < p.k ? *(const u32x4*)(p.w + (long)(n0 + row) * p.ldw + k) : u32x4{0, 0, 0, 0};
    }
  };
  fetch(0);
  for (int k0 = 0; k0 < p.k; k0 += BK) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int id = threadIdx.x + i * NT, row = id >> 3, c = id & 7;
      *(u32x4*)(ta + row * BK + ((c ^ (row & 7)) << 4)) = ra[i];
      *(u32x4*)(tw + row * BK + ((c ^ (row & 7)) << 4)) = rw[i];
    }
    __syncthreads();
    if (k0 + BK < p.k) fetch(k0 + BK);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      i32x8 fa[2], fw[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = operand(ta, wm + 32 * i + r31, ks, half);
        fw[i] = operand(tw, wn + 32 * i + r31, ks, half);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mma(fa[i], fw[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int n = n0 + wn + 32 * j + r31;
    if (n >= p.n) continue;
    const float ws = p.ws[n], b = p.bias ? p.bias[n] : 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const long m = m0 + wm + 32 * i + 8 * (x >> 2) + 4 * half + (x & 3);
        if (m < p.m) Elem<T>::store((T*)p.c + m * p.ldc, n, hv_act(acc[i][j][x] * p.as[m] * ws + b, p.act));
      }
  }
}

}  // namespace

extern "C" size_t hv_linear_fp8_work_bytes(long, int, int) { return 0; }

extern "C" int hv_linear_fp8(const void* a, long lda, const float* a_scale, const void* w, long ldw, const float* w_scale,
                             const float* bias, int act, long m, int n, int k, int c_dtype, void* c, long ldc, void* work,
                             hv_stream_t stream) {
  if (m < 0 || n < 0 || k <= 0 || lda < k || ldw < k || ldc < n || act < HV_ACT_NONE || act > HV_ACT_SIGMOID) return HV_EINVAL;
  if (k % 16 || lda % 16 || ldw % 16 || m > (1L << 31)) return HV_EUNSUPPORTED;
  if (c_dtype != HV_F32 && c_dtype != HV_BF16) return HV_EINVAL;
  if (m == 0 || n == 0) return HV_OK;
  if (!a || !w || !c || !a_scale || !w_scale || ((uintptr_t)a & 15) || ((uintptr_t)w & 15)) return HV_EINVAL;
  const LinArgs p{(const unsigned char*)a, (const unsigned char*)w, lda, ldw, m, ldc, n, k, act, a_scale, w_scale, bias, c};
  const dim3 g(hv_cdiv(n, 128), hv_cdiv(m, 128));
  if (g.y > 65535) return HV_EUNSUPPORTED;
  HV_DISPATCH(c_dtype, (k_linear_fp8<T><<<g, NT, 0, (hipStream_t)stream>>>(p)));
  HV_CHECK_LAUNCH();
  hv_diag_count(HV_KF_LINEAR_FP8);
  return HV_OK;
}
