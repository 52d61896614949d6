// Residual addition + RMS norm in one pass over the rows (RMSNorm.forward, manifold_layers.py:449-456, after the
// residual addition of vit_encoder_decoder.py:190-208): s = x + residual, y = s / sqrt(mean(s^2) + eps) * w, y in fp32,
// bf16 or e4m3 with one scale per row; its backward; and the plain row quantiser that lays 8-bit weights out.
//
// Bytes bound it: every value is read once, kept in registers through the row's sums, and written once.  TPR threads
// own a row, each VW-wide chunks (VW = 8: 16 bytes of bf16; VW = 1 where cols is no multiple of 8), so a row of up to
// TPR * V * VW columns needs no second read.  Sums, the row maximum and the weight's gradient are fp32.
// (16384 x 4096 bf16 rows on a bf16 residual to e4m3: 90 us, 5.2 TB/s; 16400 x 1024 bf16 on fp32: forward 38 us, backward 54 + 4.)
#include "hv_common.h"

namespace {

constexpr float E4M3_MAX = 448.f;
constexpr float SCALE_FLOOR = 7.52316384526264e-37f;     // 2^-120: keeps 1 / scale finite, an all-zero row gets codes 0

template <int VW> struct Vec { float v[VW]; };

template <int VW, typename T> __device__ __forceinline__ Vec<VW> load_vec(const T* p) {
  Vec<VW> r;
  if constexpr (VW == 1) {
    r.v[0] = Elem<T>::load(p, 0);
  } else if constexpr (sizeof(T) == 2) {
    const u16x8 u = *(const u16x8*)p;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = bf2f(u[e]);
  } else {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { r.v[e] = a[e]; r.v[4 + e] = b[e]; }
  }
  return r;
}

template <int VW, typename T> __device__ __forceinline__ void store_vec(T* p, const Vec<VW>& r) {
  if constexpr (VW == 1) {
    Elem<T>::store(p, 0, r.v[0]);
  } else if constexpr (sizeof(T) == 2) {
    *(uint4*)p = make_uint4(pack_bf16x2(r.v[0], r.v[1]), pack_bf16x2(r.v[2], r.v[3]), pack_bf16x2(r.v[4], r.v[5]),
                            pack_bf16x2(r.v[6], r.v[7]));
  } else {
    *(float4*)p = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
    *(float4*)(p + 4) = make_float4(r.v[4], r.v[5], r.v[6], r.v[7]);
  }
}

template <int VW> __device__ __forceinline__ void store_e4m3(unsigned char* p, const Vec<VW>& r) {
  if constexpr (VW == 1) {
    *p = (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(r.v[0], 0.f, 0, false) & 0xff);
  } else {
    int a = __builtin_amdgcn_cvt_pk_fp8_f32(r.v[0], r.v[1], 0, false);
    int b = __builtin_amdgcn_cvt_pk_fp8_f32(r.v[4], r.v[5], 0, false);
    a = __builtin_amdgcn_cvt_pk_fp8_f32(r.v[2], r.v[3], a, true);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(r.v[6], r.v[7], b, true);
    *(uint2*)p = make_uint2(a, b);
  }
}

// the larger one, NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) { return a != a || a > b ? a : b; }

// sum / maximum over the TPR threads of a row; red: one float per wave
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += red[i];
  }
  return v;
}
template <int TPR> __device__ __forceinline__ float row_max(float v, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max_nan(v, __shfl_xor(v, o, 64));
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < TPR / 64; ++i) v = max_nan(v, red[i]);
  }
  return v;
}

struct NormArgs {
  const void* x;
  long ldx;
  const void* residual;
  long rows, first;               // this launch: rows first .. rows - 1
  int cols, x_dtype, r_dtype;
  float eps;
  const float* w;                 // null: rows are quantised as they are
  void* sum;
  void* y;
  float* y_scale;
  float* rstd;
};

// threads of a block: TPR threads per row, at least 256
template <int TPR> constexpr int threads_of() { return TPR < 256 ? 256 : TPR; }

template <typename TY, int VW, int TPR, int V>
__global__ void __launch_bounds__(threads_of<TPR>()) k_add_rmsnorm(const NormArgs a) {
  __shared__ float red[16];
  constexpr int RPB = threads_of<TPR>() / TPR;           // rows of a block
  const long row = a.first + (long)blockIdx.x * RPB + threadIdx.x / TPR;
  const int t = threadIdx.x % TPR;
  if (row >= a.rows) return;                             // whole waves, and whole blocks where the row spans waves
  const long base = row * a.cols;
  Vec<VW> s[V];
  auto in = [&](int i) { return (t + i * TPR) * VW < a.cols; };
  auto read = [&](auto* p) {
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = in(i) ? load_vec<VW>(p + (t + i * TPR) * VW) : Vec<VW>{};
  };
  auto add = [&](auto* p) {
    Vec<VW> r[V];
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = in(i) ? load_vec<VW>(p + (t + i * TPR) * VW) : Vec<VW>{};
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < VW; ++e) s[i].v[e] += r[i].v[e];
  };
  auto write = [&](auto* p) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (in(i)) store_vec<VW>(p + (t + i * TPR) * VW, s[i]);
  };
  if (a.x_dtype == HV_BF16) read((const unsigned short*)a.x + row * a.ldx);
  else read((const float*)a.x + row * a.ldx);
  if (a.residual) {
    if (a.r_dtype == HV_BF16) {
      add((const unsigned short*)a.residual + base);
      write((unsigned short*)a.sum + base);
    } else {
      add((const float*)a.residual + base);
      write((float*)a.sum + base);
    }
  }
  if (a.w) {
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < VW; ++e) q = fmaf(s[i].v[e], s[i].v[e], q);
    const float rs = 1.f / sqrtf(row_sum<TPR>(q, red) / a.cols + a.eps);
    if (a.rstd && t == 0) a.rstd[row] = rs;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (in(i)) {
        const Vec<VW> w = load_vec<VW>(a.w + (t + i * TPR) * VW);
#pragma unroll
        for (int e = 0; e < VW; ++e) s[i].v[e] = s[i].v[e] * rs * w.v[e];
      }
  }
  if constexpr (sizeof(TY) == 1) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < VW; ++e) top = max_nan(fabsf(s[i].v[e]), top);
    top = row_max<TPR>(top, red);
    const float scale = max_nan(top / E4M3_MAX, SCALE_FLOOR);
    if (t == 0) a.y_scale[row] = scale;
    const float inv = 1.f / scale;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < VW; ++e) s[i].v[e] *= inv;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (in(i)) store_e4m3<VW>((unsigned char*)a.y + base + (t + i * TPR) * VW, s[i]);
  } else {
    write((TY*)a.y + base);
  }
}

struct NormBackArgs {
  const void *x, *residual;       // the sum's operands, or the sum and null
  const float *rstd, *w;
  const void *dy, *dsum;
  long rows;
  int cols, x_dtype, r_dtype, dy_dtype, dx_dtype;
  void *dx, *dresidual;
  float* part;                    // [blocks, cols] column sums of dy s rstd
};

// n = s rstd, g = w dy:  ds = dsum + rstd (g - n mean(g n));  dw = sum_rows dy n.  A block walks over rows with a
// fixed stride and keeps its columns' share of dw in registers; the shares are summed by k_norm_dw in a fixed order.
template <int VW, int TPR, int V>
__global__ void __launch_bounds__(threads_of<TPR>()) k_add_rmsnorm_back(const NormBackArgs a) {
  constexpr int NTB = threads_of<TPR>(), RPB = NTB / TPR;
  __shared__ float red[16];
  __shared__ float fold[RPB > 1 ? (RPB - 1) * TPR * V * VW : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  auto in = [&](int i) { return (t + i * TPR) * VW < a.cols; };
  Vec<VW> w[V], dw[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    w[i] = in(i) ? load_vec<VW>(a.w + (t + i * TPR) * VW) : Vec<VW>{};
    dw[i] = Vec<VW>{};
  }
  for (long row = (long)blockIdx.x * RPB + sub; row < a.rows; row += (long)gridDim.x * RPB) {
    const long base = row * a.cols;
    Vec<VW> n[V], g[V], d[V];
    auto read = [&](Vec<VW>* to, const void* from, int dtype) {
      if (dtype == HV_BF16) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          to[i] = in(i) ? load_vec<VW>((const unsigned short*)from + base + (t + i * TPR) * VW) : Vec<VW>{};
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          to[i] = in(i) ? load_vec<VW>((const float*)from + base + (t + i * TPR) * VW) : Vec<VW>{};
      }
    };
    read(n, a.x, a.x_dtype);
    read(g, a.dy, a.dy_dtype);
    if (a.residual) {
      read(d, a.residual, a.r_dtype);
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int e = 0; e < VW; ++e) n[i].v[e] += d[i].v[e];
    }
    if (a.dsum) {
      read(d, a.dsum, a.r_dtype);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = Vec<VW>{};
    }
    const float rs = a.rstd[row];
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        n[i].v[e] *= rs;
        dw[i].v[e] = fmaf(g[i].v[e], n[i].v[e], dw[i].v[e]);
        g[i].v[e] *= w[i].v[e];
        q = fmaf(g[i].v[e], n[i].v[e], q);
      }
    q = row_sum<TPR>(q, red) / a.cols;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < VW; ++e) d[i].v[e] = fmaf(rs, fmaf(-n[i].v[e], q, g[i].v[e]), d[i].v[e]);
    auto write = [&](void* to, int dtype) {
      if (to == nullptr) return;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (in(i)) {
          if (dtype == HV_BF16) store_vec<VW>((unsigned short*)to + base + (t + i * TPR) * VW, d[i]);
          else store_vec<VW>((float*)to + base + (t + i * TPR) * VW, d[i]);
        }
    };
    write(a.dx, a.dx_dtype);
    write(a.dresidual, a.r_dtype);
  }
  if constexpr (RPB > 1) {                               // the block's rows of one column set
    if (sub > 0) {
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int e = 0; e < VW; ++e) fold[((sub - 1) * V * VW + i * VW + e) * TPR + t] = dw[i].v[e];
    }
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < VW; ++e)
        for (int o = 0; o < RPB - 1; ++o) dw[i].v[e] += fold[(o * V * VW + i * VW + e) * TPR + t];
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (in(i)) store_vec<VW>(a.part + (long)blockIdx.x * a.cols + (t + i * TPR) * VW, dw[i]);
}

// dw[c] = sum_b part[b, c]: 16 columns x 64 shares of the blocks per workgroup
__global__ void __launch_bounds__(1024) k_norm_dw(const float* __restrict__ part, int nb, int cols, float* __restrict__ dw) {
  __shared__ float red[64][17];
  const int cl = threadIdx.x & 15, share = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float v = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int b = share; b < nb; b += 64) v += part[(long)b * cols + c];
  }
  red[share][cl] = v;
  __syncthreads();
  if (share < 16) {
    v = red[share][cl] + red[share + 16][cl] + red[share + 32][cl] + red[share + 48][cl];
    red[share][cl] = v;                                   // read and written by this thread only
  }
  __syncthreads();
  if (share == 0 && c < cols) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += red[i][cl];
    dw[c] = v;
  }
}

constexpr int MAX_COLS = 32768;

// threads per row and chunks per thread for a row length: the smallest group whose registers hold the row
#define HV_ROW_SHAPE(cols, wide, CALL)                     \
  do {                                                     \
    if (wide) {                                            \
      if ((cols) <= 512) CALL(8, 64, 1);                   \
      else if ((cols) <= 1024) CALL(8, 64, 2);             \
      else if ((cols) <= 2048) CALL(8, 256, 1);            \
      else if ((cols) <= 4096) CALL(8, 256, 2);            \
      else if ((cols) <= 8192) CALL(8, 256, 4);            \
      else CALL(8, 1024, 4);                               \
    } else {                                               \
      if ((cols) <= 512) CALL(1, 64, 8);                   \
      else if ((cols) <= 4096) CALL(1, 256, 16);           \
      else CALL(1, 1024, 32);                              \
    }                                                      \
  } while (0)

constexpr long LAUNCH_ROWS = 1L << 21;                   // of one launch: a grid stays below 2^32 threads

template <typename TY> int launch_norm(NormArgs a, bool wide, hipStream_t s) {
#define HV_NORM_CALL(VW, TPR, V)                                                                    \
  k_add_rmsnorm<TY, VW, TPR, V><<<hv_cdiv(a.rows - a.first, threads_of<TPR>() / TPR), threads_of<TPR>(), 0, s>>>(a)
  for (const long rows = a.rows; a.first < rows; a.first += LAUNCH_ROWS) {
    a.rows = rows < a.first + LAUNCH_ROWS ? rows : a.first + LAUNCH_ROWS;
    HV_ROW_SHAPE(a.cols, wide, HV_NORM_CALL);
    HV_CHECK_LAUNCH();
  }
#undef HV_NORM_CALL
  return HV_OK;
}

bool a16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int norm_blocks(long rows, int cols) {
  const int rpb = cols <= 512 || (cols <= 1024 && cols % 8 == 0) ? 4 : 1;
  const long b = (rows + rpb - 1) / rpb;
  return (int)(b < 1024 ? (b > 0 ? b : 1) : 1024);
}

bool is_float(int dt) { return dt == HV_F32 || dt == HV_BF16; }

}  // namespace

extern "C" int hv_add_rmsnorm(int x_dtype, const void* x, int r_dtype, const void* residual, long rows, int cols,
                              float eps, const float* scale, void* sum, int y_dtype, void* y, float* y_scale,
                              float* rstd, hv_stream_t stream) {
  if (!is_float(x_dtype) || (residual && !is_float(r_dtype)) || rows < 0 || cols <= 0 || !(eps >= 0.f)) return HV_EINVAL;
  if (!(is_float(y_dtype) || y_dtype == HV_E4M3)) return HV_EINVAL;
  if (cols > MAX_COLS) return HV_EUNSUPPORTED;
  if (rows == 0) return HV_OK;
  if (!x || !scale || !y || (residual && !sum) || (y_dtype == HV_E4M3 && !y_scale)) return HV_EINVAL;
  const bool wide = cols % 8 == 0 && a16(x) && a16(residual) && a16(scale) && a16(sum) && a16(y);
  const NormArgs a{x, cols, residual, rows, 0, cols, x_dtype, r_dtype, eps, scale, sum, y, y_scale, rstd};
  hipStream_t s = (hipStream_t)stream;
  hv_diag_count(HV_KF_ADD_RMSNORM);
  if (y_dtype == HV_E4M3) return launch_norm<unsigned char>(a, wide, s);
  HV_DISPATCH(y_dtype, return launch_norm<T>(a, wide, s));
  return HV_EINVAL;
}

extern "C" int hv_quantize_rows_fp8(int dtype, const void* x, long ld, long rows, int cols, void* codes, float* scale,
                                    hv_stream_t stream) {
  if (!is_float(dtype) || rows < 0 || cols <= 0 || ld < cols) return HV_EINVAL;
  if (cols > MAX_COLS) return HV_EUNSUPPORTED;
  if (rows == 0) return HV_OK;
  if (!x || !codes || !scale) return HV_EINVAL;
  const bool wide = cols % 8 == 0 && ld % 8 == 0 && a16(x) && ((uintptr_t)codes & 7) == 0;
  const NormArgs a{x, ld, nullptr, rows, 0, cols, dtype, dtype, 0.f, nullptr, nullptr, codes, scale, nullptr};
  return launch_norm<unsigned char>(a, wide, (hipStream_t)stream);
}

extern "C" size_t hv_add_rmsnorm_backward_work_floats(long rows, int cols) {
  return rows <= 0 || cols <= 0 ? 0 : (size_t)norm_blocks(rows, cols) * cols;
}

extern "C" int hv_add_rmsnorm_backward(int x_dtype, const void* x, int r_dtype, const void* residual, const float* rstd,
                                       const float* scale, int dy_dtype, const void* dy, const void* dsum, long rows, int cols,
                                       int dx_dtype, void* dx, void* dresidual, float* dscale, float* work,
                                       hv_stream_t stream) {
  if (!is_float(x_dtype) || !is_float(r_dtype) || !is_float(dy_dtype) || (dx && !is_float(dx_dtype)) || rows < 0 || cols <= 0)
    return HV_EINVAL;
  if (cols > MAX_COLS) return HV_EUNSUPPORTED;
  if (!dscale || (rows > 0 && (!x || !rstd || !scale || !dy || !work))) return HV_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  const int nb = rows > 0 ? norm_blocks(rows, cols) : 0;
  if (rows > 0) {
    const bool wide = cols % 8 == 0 && a16(x) && a16(residual) && a16(scale) && a16(dy) && a16(dsum) && a16(dx) &&
                      a16(dresidual) && a16(work);
    const NormBackArgs a{x,    residual, rstd,    scale,    dy,       dsum, rows,
                         cols, x_dtype,  r_dtype, dy_dtype, dx_dtype, dx,   dresidual, work};
#define HV_NORM_CALL(VW, TPR, V) k_add_rmsnorm_back<VW, TPR, V><<<nb, threads_of<TPR>(), 0, s>>>(a)
    HV_ROW_SHAPE(cols, wide, HV_NORM_CALL);
#undef HV_NORM_CALL
  }
  k_norm_dw<<<hv_cdiv(cols, 16), 1024, 0, s>>>(work, nb, cols, dscale);
  HV_CHECK_LAUNCH();
  hv_diag_count(HV_KF_ADD_RMSNORM);
  return HV_OK;
}
