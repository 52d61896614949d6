// Attention over packed sequences of different lengths: causal or not, grouped heads, head dims up to
// 128, bf16 and fp32, forward and backward (reference core: manifold_layers.py:404-427).
//
// Rows.  The G = hq / hkv query heads that share a key / value head are packed into the rows of one
// tile: packed row r of a sequence is (token r / G, head r % G), so a key / value tile is read once for
// the whole group and the gradient of a shared head is summed in registers.
//
// Orientation.  Scores are formed transposed, S^T = K Q^T, with 32x32 matrix tiles: a lane then holds
// 16 scores of ONE query (column lane & 31; keys 8 (r / 4) + 4 (lane >> 5) + r % 4 for register r), so a
// softmax row is 16 registers and one exchange between the two lane halves, and the running maximum and
// sums are one register each.  The contraction index of the second product may be numbered freely: with
// key slot (h, e) = key 16 s + 8 (e / 4) + 4 h + e % 4 the accumulator registers 8 s .. 8 s + 7 ARE the
// second operand of O^T += V^T P^T (no lane exchange), and V is read from LDS with the transposing load.
// The backward uses the same two moves for dQ^T += K^T dS^T, dV^T += dO^T P and dK^T += Q^T dS.
//
// LDS tiles are rows of DP elements (DP = d rounded up to 32 / 64 / 128, columns >= d zero) whose 16-byte
// chunks are permuted by a function of the row (Lay::f), so that the row reads (16 rows of one chunk) and the
// transposing reads (4 rows of four chunks) spread over the banks.
#include "hv_common.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// division by a number fixed on the host: x / d for 0 <= x < 2^31 is (mulhi(x, mul) + x) >> shift
struct FastDiv {
  uint32_t mul, shift, d;
  explicit FastDiv(uint32_t v) : shift(0), d(v) {
    while ((1ull << shift) < v) ++shift;
    mul = (uint32_t)((((1ull << 32) * ((1ull << shift) - v)) / v) + 1);
  }
  __device__ __forceinline__ int div(int x) const { return (int)((__umulhi((uint32_t)x, mul) + (uint32_t)x) >> shift); }
  __device__ __forceinline__ int mod(int x, int q) const { return x - q * (int)d; }
};

// what the kernels get: the call's arguments, the query heads per key / value head and the key / value heads
struct Args : hv_attn_packed_args {
  FastDiv group, heads;
  explicit Args(const hv_attn_packed_args& a) : hv_attn_packed_args(a), group(a.hq / a.hkv), heads(a.hkv) {}
};

constexpr float LOG2E = 1.4426950408889634f;
constexpr int NT = 256;         // threads of every block: 4 waves
constexpr int KEYS = 64;        // keys of a dK / dV block
constexpr float NEG_INF = -__builtin_inff();

template <typename T> struct Frag;                       // 8 values of a lane: one operand over 16 columns
template <> struct Frag<unsigned short> { bf16x8 v; };
template <> struct Frag<float> { float v[8]; };

__device__ __forceinline__ f32x16 mma16(const Frag<unsigned short>& a, const Frag<unsigned short>& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma16(const Frag<float>& a, const Frag<float>& b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
  return c;
}

template <typename T, int DP> struct Lay {               // an LDS tile
  static constexpr int ROWB = DP * (int)sizeof(T);       // bytes of a row
  static constexpr int CH = ROWB / 16;                   // its 16-byte chunks
  static constexpr int EPC = 16 / (int)sizeof(T);        // elements of a chunk
  static constexpr int NS = DP / 16, NDT = DP / 32;      // 16-column steps, 32-column tiles
  // chunk permutation of a row (a row of 0 mod 16: none).  CH >= 16: 16 rows' equal chunks, and 4 rows' aligned groups of
  // 4, lie in 256 different bytes, the width of an LDS access (permuted over 128 bytes only: half the LDS rate, 127 against
  // 228 bytes a clock and CU; the forward gains 2 %).  Shorter rows: over 128 bytes, so that a row and the row 8 below it
  // are permuted alike and share an address (64 columns: 92 us, over 256 bytes 98 us, causal ragged batch of 8569 rows).
  static constexpr __device__ __forceinline__ int f(int row) {
    return CH >= 16 ? ((row & 3) << 2) | ((row >> 2) & 3)
                    : CH == 8 ? ((row & 3) << 1) | ((row >> 2) & 1) : (row & 2) | ((row >> 2) & 1);
  }
};

// a wave's view of a tile: lane constants of the two kinds of operand reads
template <typename T, int DP> struct View {
  using L = Lay<T, DP>;
  int row_base, row_x, tr_base, tr_x;
  __device__ __forceinline__ View(int lane) {
    const int h = lane >> 5, m = lane & 31;
    row_base = m * L::ROWB;
    if constexpr (sizeof(T) == 2) {
      row_x = (h ^ L::f(m)) << 4;
      const int i = lane & 15, rl = 4 * h + (i >> 2);
      tr_base = rl * L::ROWB + (i & 1) * 8;
      tr_x = ((2 * ((lane >> 4) & 1) + ((i >> 1) & 1)) ^ L::f(rl)) << 4;
    } else {
      row_x = ((2 * h) ^ L::f(m)) << 4;
      tr_base = 4 * h * L::ROWB + (m & 3) * 4;
      tr_x = ((m >> 2) ^ h) << 4;                        // f(4 h) = h here, the rest of the row per element
    }
  }
  // operand over columns 16 s .. 16 s + 15 of the 32 rows from `tile` (a multiple of 32 rows into the tile)
  __device__ __forceinline__ Frag<T> rows(const char* tile, int s) const {
    Frag<T> r;
    if constexpr (sizeof(T) == 2) {
      r.v = *(const bf16x8*)(tile + row_base + (row_x ^ (s << 5)));
    } else {
      const f32x4 a = *(const f32x4*)(tile + row_base + (row_x ^ (s << 6)));
      const f32x4 b = *(const f32x4*)(tile + row_base + (row_x ^ (s << 6) ^ 16));
#pragma unroll
      for (int e = 0; e < 4; ++e) { r.v[e] = a[e]; r.v[4 + e] = b[e]; }
    }
    return r;
  }
  // transposed operand: columns 32 dt .. 32 dt + 31 as rows, the 16 tile rows from `tile` (a multiple of 16 rows
  // into the tile) as contraction slots
  __device__ __forceinline__ Frag<T> cols(const char* tile, int dt) const {
    Frag<T> r;
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const char* p = tile + tr_base;
      const int x = tr_x ^ (dt << 6);
      union { s16x4 q[2]; bf16x8 v; } u;
      u.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + x));
      u.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 8 * L::ROWB + (x ^ (L::f(8) << 4))));
      r.v = u.v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        r.v[e] = *(const float*)(tile + (8 * (e >> 2) + (e & 3)) * L::ROWB + tr_base +
                                 (tr_x ^ (dt << 7) ^ (L::f(8 * (e >> 2) + (e & 3)) << 4)));
    }
    return r;
  }
};

// accumulator registers 8 s .. 8 s + 7 as the second operand of the next product
template <typename T> __device__ __forceinline__ Frag<T> from_acc(const f32x16& c, int s) {
  Frag<T> r;
  if constexpr (sizeof(T) == 2) {
    u32x4 u;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = pack_bf16x2(c[8 * s + 2 * e], c[8 * s + 2 * e + 1]);
    r.v = __builtin_bit_cast(bf16x8, u);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = c[8 * s + e];
  }
  return r;
}

// sum of the 8 values as the product sees them (rounded to T), added to c
__device__ __forceinline__ float add_sum(const Frag<unsigned short>& p, float c) {
  const u32x4 u = __builtin_bit_cast(u32x4, p.v);
  const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, (uint32_t)u[e]), one, c, false);
  return c;
}
__device__ __forceinline__ float add_sum(const Frag<float>& p, float c) {
  return c + (((p.v[0] + p.v[1]) + (p.v[2] + p.v[3])) + ((p.v[4] + p.v[5]) + (p.v[6] + p.v[7])));
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

// ------------------------------------------------------------------------------------------------
// Which rows a block works on: the sequences (and the rows before the first and behind the last one, two
// more "sequences" without keys) cut into tiles of BM packed rows, numbered through.  Every wave scans the
// offsets by itself, 64 sequences at a time.
struct Tile { int seq, start, len, tile; };              // seq -1: no such tile; start, len: its rows in tokens

__device__ __forceinline__ int clamp_row(int v, int total) { return v < 0 ? 0 : (v > total ? total : v); }

__device__ __forceinline__ Tile find_tile(const int* __restrict__ cu, int nseq, long total_l, int G, int BM, int idx,
                                          bool reverse) {
  const int lane = threadIdx.x & 63, total = (int)total_l;
  Tile t{-1, 0, 0, 0};
  int before = 0;
  for (int s0 = 0; s0 < nseq + 2; s0 += 64) {
    const int s = s0 + lane;
    int a = 0, b = 0;
    if (s < nseq) {
      a = clamp_row(cu[s], total);
      b = clamp_row(cu[s + 1], total);
    } else if (s == nseq) {
      b = clamp_row(cu[0], total);
    } else if (s == nseq + 1) {
      a = clamp_row(cu[nseq], total);
      b = total;
    }
    if (b < a) b = a;
    const int n = (int)(((long)(b - a) * G + BM - 1) / BM);
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
    const unsigned long long hit = __ballot(idx < before + upto);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      t.seq = s0 + src;
      t.start = __builtin_amdgcn_readlane(a, src);
      t.len = __builtin_amdgcn_readlane(b, src) - t.start;
      const int nt = __builtin_amdgcn_readlane(n, src);
      t.tile = idx - before - (__builtin_amdgcn_readlane(upto, src) - nt);
      if (reverse) t.tile = nt - 1 - t.tile;
      return t;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return t;
}

// the sequence that owns row `row` (nseq: none)
__device__ __forceinline__ int find_row(const int* __restrict__ cu, int nseq, long total, int row) {
  for (int s0 = 0; s0 < nseq; s0 += 64) {
    const int s = s0 + (threadIdx.x & 63);
    const bool in = s < nseq && clamp_row(cu[s], (int)total) <= row && row < clamp_row(cu[s + 1], (int)total);
    const unsigned long long hit = __ballot(in);
    if (hit) return s0 + __builtin_ctzll(hit);
  }
  return nseq;
}

// rows of sequence `seq` on the other side (none for the two outside ranges)
__device__ __forceinline__ void seq_rows(const int* __restrict__ cu, int nseq, long total, int seq, int& start, int& len) {
  if (seq >= nseq) { start = len = 0; return; }
  start = clamp_row(cu[seq], (int)total);
  len = clamp_row(cu[seq + 1], (int)total) - start;
  if (len < 0) len = 0;
}

// hv_lds_dma16 from base + off, base the same for the whole wave; arrived() waits for both, once per tile.  The base may come
// from a lane read right before it (a vector instruction that writes a scalar pair): five wait states before a load takes it.
__device__ __forceinline__ void dma16_at(const void* wave_base, unsigned off, unsigned lds) {
  const uint64_t b = (uint64_t)wave_base;
  const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b) |
                        (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32)) << 32;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
#pragma clang diagnostic pop
}
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ unsigned lds_at(const void* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)p;
}

// ROWS tile rows into LDS, by the whole block: 64 chunks a wave instruction, permuted on the source side.  A lane keeps the
// address of its chunk for each of its N instructions and moves it on by 64-bit additions (a multiplication per row and
// tile cost a quarter of the tile's time).  Every address is one that may be read: rows behind the last are read from the
// last (what such rows hold is masked), chunks at columns >= d from column 0 (the other operand is 0 there).
template <typename T, int DP, int ROWS> struct Dma {
  using L = Lay<T, DP>;
  static constexpr int N = ROWS * L::CH / NT;            // instructions of a wave
  static_assert(N * NT == ROWS * L::CH, "whole chunks per thread");
  const T* at[N];
  static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
  static __device__ __forceinline__ int row(int n) { return ((wave() * N + n) * 64 + (int)(threadIdx.x & 63)) / L::CH; }
  static __device__ __forceinline__ int col(int n, int d) {
    const int i = (wave() * N + n) * 64 + (threadIdx.x & 63), c = ((i % L::CH) ^ L::f(i / L::CH)) * L::EPC;
    return c < d ? c : 0;
  }
  static __device__ __forceinline__ void send(const T* src, unsigned lds, int n) { hv_lds_dma16(src, lds + (wave() * N + n) * 1024); }
  __device__ __forceinline__ void issue(unsigned lds) const {
#pragma unroll
    for (int n = 0; n < N; ++n) send(at[n], lds, n);
  }
};

// K or V tiles of BN rows, one after the other; the rows of the last tile are held below `end`
template <typename T, int DP, int BN> struct KeyTiles : Dma<T, DP, BN> {
  using B = Dma<T, DP, BN>;
  const T* base;
  long stride, step;
  int end, d;
  __device__ __forceinline__ KeyTiles(const T* p, long row_stride, int rows, int dim)
      : base(p), stride(row_stride), step(row_stride * BN), end(rows), d(dim) {
#pragma unroll
    for (int n = 0; n < B::N; ++n) B::at[n] = p + B::row(n) * row_stride + B::col(n, dim);
  }
  __device__ __forceinline__ void next(int kt, unsigned lds) {       // tiles 0, 1, 2 ... in order
    if ((kt + 1) * BN <= end) {
      B::issue(lds);
#pragma unroll
      for (int n = 0; n < B::N; ++n) B::at[n] += step;
    } else {
#pragma unroll
      for (int n = 0; n < B::N; ++n)
        B::send(base + (long)min(kt * BN + B::row(n), end - 1) * stride + B::col(n, d), lds, n);
    }
  }
};

// Q or dO tiles of `used` packed rows, the largest multiple of the group G in BR (so that a tile holds whole tokens), from
// the one with the last rows backwards.  A lane's chunks lie at the same 32-bit offsets from the tile's first token in every
// tile, so a tile's address is one scalar addition; only the last tile's rows have to be held below `rows`.
template <typename T, int DP, int BR> struct RowTiles : Dma<T, DP, BR> {
  using B = Dma<T, DP, BR>;
  const T* base;
  unsigned off[B::N];
  __device__ __forceinline__ RowTiles(const T* p, long row, long head, int used, int d, const FastDiv& group) : base(p) {
#pragma unroll
    for (int n = 0; n < B::N; ++n) {
      const int x = min(B::row(n), used - 1), t = group.div(x);
      off[n] = (unsigned)((t * row + group.mod(x, t) * head + B::col(n, d)) * sizeof(T));
    }
  }
  __device__ __forceinline__ void last(long row, long head, int r, int rows, int d, const FastDiv& group, unsigned lds) const {
#pragma unroll
    for (int n = 0; n < B::N; ++n) {
      const int x = min(r + B::row(n), rows - 1), t = group.div(x);
      B::send(base + t * row + group.mod(x, t) * head + B::col(n, d), lds, n);
    }
  }
  __device__ __forceinline__ void send_tile(long token_offset, unsigned lds) const {
    const T* p = base + token_offset;
#pragma unroll
    for (int n = 0; n < B::N; ++n) dma16_at(p, off[n], lds + (B::wave() * B::N + n) * 1024);
  }
};

__device__ __forceinline__ void load8(Frag<unsigned short>& f, const unsigned short* p) { f.v = *(const bf16x8*)p; }
__device__ __forceinline__ void load8(Frag<float>& f, const float* p) {
  const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) { f.v[e] = a[e]; f.v[4 + e] = b[e]; }
}

// a lane's row of 16-column operands straight from memory (null: zeros)
template <typename T, int DP> __device__ __forceinline__ void load_row(Frag<T>* f, const T* p, int d, int h) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int c = 16 * s + 8 * h;
    const bool in = p != nullptr && c < d;
    if constexpr (sizeof(T) == 2) {
      f[s].v = in ? *(const bf16x8*)(p + c) : bf16x8{};
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const f32x4 a = in ? *(const f32x4*)(p + c + e) : f32x4{0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < 4; ++x) f[s].v[e + x] = a[x];
      }
    }
  }
}

// Have the operands in registers from here on.  Without it the compiler places its wait for their loads at the first use
// inside the tile loop, where it would also wait for the tile that is on its way.
template <typename T, int N> __device__ __forceinline__ void settle(Frag<T> (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (sizeof(T) == 2) {
      asm volatile("" : "+v"(f[i].v));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(f[i].v[e]));
    }
  }
}

// four consecutive values of a lane's row
__device__ __forceinline__ void store4(unsigned short* p, float a, float b, float c, float d) {
  *(uint2*)p = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
}
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
  *(float4*)p = make_float4(a, b, c, d);
}

template <typename T, int DP>
__device__ __forceinline__ void store_row(T* p, int d, int h, const f32x16* acc, float mul) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * dt + 8 * g + 4 * h;
      if (c < d)
        store4(p + c, acc[dt][4 * g] * mul, acc[dt][4 * g + 1] * mul, acc[dt][4 * g + 2] * mul, acc[dt][4 * g + 3] * mul);
    }
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// ------------------------------------------------------------------------------------------------
// Forward: 4 waves of 32 packed rows each over tiles of BN keys that the block stages once.  KS > 1, where the rows give
// few blocks: KS waves share 32 rows, wave ks takes every KS-th run of BN keys (a tile is KS runs), and their sums are
// joined through LDS in order.
template <typename T, int DP, bool TRAIN, int KS>
__global__ void __launch_bounds__(NT, DP * sizeof(T) * KS > 256 ? 1 : 2) k_attn_packed(const Args a) {
  using L = Lay<T, DP>;
  constexpr int BM = 128 / KS, BN = L::ROWB > 256 ? 32 : 64, BT = BN * KS, TB = BT * L::ROWB, NJ = BN / 32;
  __shared__ __align__(16) char smem[4 * TB];          // K and V, two buffers
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int G = a.group.d, block = a.heads.div(blockIdx.x), kvh = a.heads.mod(blockIdx.x, block);
  const Tile t = find_tile(a.cu_q, a.nseq, a.total_q, G, BM, block, a.causal != 0);
  if (t.seq < 0) return;
  int k0, lk;
  seq_rows(a.cu_k, a.nseq, a.total_k, t.seq, k0, lk);

  const int ks = wave % KS, r = t.tile * BM + wave / KS * 32 + (lane & 31);
  const bool real = r < t.len * G;
  const int tok = real ? a.group.div(r) : 0, g = real ? a.group.mod(r, tok) : 0;
  const int late = lk - t.len;                           // the last query sees every key
  const int lim = !real ? -1 : (a.causal ? min(tok + late, lk - 1) : lk - 1);     // last key of this row
  // the block's last key, the wave's first row's last key: full tiles need no mask
  const int last_r = min((t.tile + 1) * BM, t.len * G) - 1;
  const int lim_blk = a.causal ? min(a.group.div(last_r) + late, lk - 1) : lk - 1;
  int lim_lo = lim, lim_hi = lim;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    lim_lo = min(lim_lo, __shfl_xor(lim_lo, o, 64));
    lim_hi = max(lim_hi, __shfl_xor(lim_hi, o, 64));
  }
  lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);
  lim_hi = __builtin_amdgcn_readfirstlane(lim_hi);

  const long qrow = (long)t.start + tok;
  const int qh = kvh * G + g;
  Frag<T> q[L::NS];
  load_row<T, DP>(q, real ? (const T*)a.q + qrow * a.q_row + (long)qh * a.q_head : nullptr, a.d, h);
  settle(q);
  const T* kp = (const T*)a.k + (long)k0 * a.k_row + (long)kvh * a.k_head;
  const T* vp = (const T*)a.v + (long)k0 * a.v_row + (long)kvh * a.v_head;

  f32x16 o[L::NDT];
#pragma unroll
  for (int i = 0; i < L::NDT; ++i) o[i] = zero16();
  float m = NEG_INF, l = 0.f, lt = 0.f;                  // running maximum, sum of rounded / of exact weights
  const float c2 = a.scale * LOG2E;
  const View<T, DP> view(lane);
  const int ntile = (lim_blk + BT) / BT;

  const unsigned lds0 = lds_at(smem);
  KeyTiles<T, DP, BT> sk(kp, a.k_row, lim_blk + 1, a.d), sv(vp, a.v_row, lim_blk + 1, a.d);
  auto fetch = [&](int kt) {
    const unsigned at = lds0 + (kt & 1) * 2 * TB;
    sk.next(kt, at);
    sv.next(kt, at + TB);
  };
  if (ntile > 0) fetch(0);
  for (int kt = 0; kt < ntile; ++kt) {
    arrived();
    __syncthreads();                                     // tile kt is here, the other buffer is no longer read
    const char* tk = smem + (kt & 1) * 2 * TB + ks * BN * L::ROWB;
    const char* tv = tk + TB;
    if (kt + 1 < ntile) fetch(kt + 1);
    const int key = kt * BT + ks * BN;                   // this wave's first key of the tile
    if (key > lim_hi) continue;
    f32x16 s[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) s[j] = zero16();
#pragma unroll
    for (int i = 0; i < L::NS; ++i) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) s[j] = mma16(view.rows(tk + j * 32 * L::ROWB, i), q[i], s[j]);
    }
    if (key + BN - 1 > lim_lo) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (key + 32 * j + 8 * (x >> 2) + 4 * h + (x & 3) > lim) s[j][x] = NEG_INF;
    }
    float top = s[0][0];
#pragma unroll
    for (int x = 1; x < 16; ++x) top = fmaxf(top, s[0][x]);
#pragma unroll
    for (int j = 1; j < NJ; ++j)
#pragma unroll
      for (int x = 0; x < 16; ++x) top = fmaxf(top, s[j][x]);
    top = fmaxf(top, other_half(top));
    // the running maximum moves only when a score passes it by 8 powers of two: weights stay below 2^8 and
    // the accumulators are seldom rescaled
    if (__any((top - m) * c2 > 8.f)) {
      const float mn = fmaxf(m, top);
      const float alpha = mn == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c2);
      m = mn;
      l *= alpha;
      lt *= alpha;
#pragma unroll
      for (int i = 0; i < L::NDT; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[i][x] *= alpha;
    }
    const float mc = m == NEG_INF ? 0.f : -m * c2;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int x = 0; x < 16; ++x) s[j][x] = __builtin_amdgcn_exp2f(fmaf(s[j][x], c2, mc));
    if constexpr (TRAIN && sizeof(T) == 2) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int x = 0; x < 16; ++x) lt += s[j][x];
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Frag<T> p = from_acc<T>(s[j], i);
        l = add_sum(p, l);
#pragma unroll
        for (int dt = 0; dt < L::NDT; ++dt)
          o[dt] = mma16(view.cols(tv + (32 * j + 16 * i) * L::ROWB, dt), p, o[dt]);
      }
  }
  l += other_half(l);
  if constexpr (TRAIN && sizeof(T) == 2) lt += other_half(lt); else lt = l;
  if constexpr (KS > 1) {                                // wave ks = 0 joins its rows' sums
    constexpr int W = 16 * L::NDT + 3;
    float* part = (float*)smem + (wave / KS * (KS - 1) + ks - 1) * W * 64 + lane;
    static_assert(4 / KS * (KS - 1) * W * 64 * 4 <= 4 * TB, "the joined sums fit the tiles' LDS");
    __syncthreads();
    if (ks > 0) {
      part[0] = m;
      part[64] = l;
      part[128] = lt;
#pragma unroll
      for (int i = 0; i < L::NDT; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) part[(3 + i * 16 + x) * 64] = o[i][x];
    }
    __syncthreads();
    if (ks > 0) return;
    float mx = m;
    part += W * 64;                                      // of ks = 1
#pragma unroll
    for (int k = 0; k < KS - 1; ++k) mx = fmaxf(mx, part[k * W * 64]);
    const float f0 = m == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((m - mx) * c2);
    l *= f0;
    lt *= f0;
#pragma unroll
    for (int i = 0; i < L::NDT; ++i)
#pragma unroll
      for (int x = 0; x < 16; ++x) o[i][x] *= f0;
#pragma unroll
    for (int k = 0; k < KS - 1; ++k) {
      const float* pk = part + k * W * 64;
      const float f = pk[0] == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((pk[0] - mx) * c2);
      l = fmaf(pk[64], f, l);
      lt = fmaf(pk[128], f, lt);
#pragma unroll
      for (int i = 0; i < L::NDT; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[i][x] = fmaf(pk[(3 + i * 16 + x) * 64], f, o[i][x]);
    }
    m = mx;
  }
  if (!real) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const long orow = (qrow * a.hq + qh) * a.d;
  store_row<T, DP>((T*)a.out + orow, a.d, h, o, inv);
  if constexpr (TRAIN) {
    if (h == 0 && a.lse) a.lse[qrow * a.hq + qh] = lt > 0.f || lt != lt ? m * a.scale + __logf(lt) : NEG_INF;
    if constexpr (sizeof(T) == 2) {
      if (a.out_low) {
#pragma unroll
        for (int dt = 0; dt < L::NDT; ++dt)
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const float v = o[dt][x] * inv;
            o[dt][x] = v - bf2f(f2bf(v));
          }
        store_row<T, DP>((T*)a.out_low + orow, a.d, h, o, 1.f);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Forward with few query rows (new tokens against histories): the keys are cut into parts of a.part and a block
// takes one part for all the rows of its sequence, 32 at a time.  Its four waves own a quarter of the part each, in
// slabs of 32 keys, and never wait for one another: K goes from memory to registers as the first operand, V through a
// wave's own LDS, both a slab ahead, so a wave has 2 * 32 rows in flight and a CU eight such waves.  Bytes bound it.
// Partial sums (fp32, with their maxima) go to the workspace and are joined by k_attn_packed_join in a fixed order.
template <typename T, int DP>
__global__ void __launch_bounds__(NT, sizeof(T) == 4 && DP == 128 ? 1 : 2)
k_attn_packed_keys(const Args a, int part_keys, float* __restrict__ po, float4* __restrict__ pml) {
  using L = Lay<T, DP>;
  constexpr int SB = 32 * L::ROWB;                       // a wave's V slab
  constexpr int JB = 32 * DP * 4;                        // a wave's O at the end, fp32
  constexpr int NV = 32 * L::CH / 64;                    // its 16-byte chunks per lane
  __shared__ __align__(16) char smem[4 * SB > 2 * JB ? 4 * SB : 2 * JB];
  __shared__ float red[3][4][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, c31 = lane & 31;
  const int G = a.group.d, block = a.heads.div(blockIdx.x), kvh = a.heads.mod(blockIdx.x, block);
  const Tile t = find_tile(a.cu_k, a.nseq, a.total_k, 1, part_keys, block, false);
  if (t.seq < 0 || t.seq >= a.nseq) return;
  int q0, lq;
  seq_rows(a.cu_q, a.nseq, a.total_q, t.seq, q0, lq);
  const int lk = t.len, late = lk - lq, quarter = part_keys >> 2;
  const int key0 = t.tile * part_keys + wave * quarter, key1 = min(key0 + quarter, lk);
  const T* kp = (const T*)a.k + (long)t.start * a.k_row + (long)kvh * a.k_head;
  const T* vp = (const T*)a.v + (long)t.start * a.v_row + (long)kvh * a.v_head;
  const float c2 = a.scale * LOG2E;
  const View<T, DP> view(lane);
  char* slab = smem + wave * SB;
  for (int r0 = 0; r0 < lq * G; r0 += 32) {
    const int r = r0 + c31;
    const bool real = r < lq * G;
    const int tok = real ? a.group.div(r) : 0, qh = kvh * G + (real ? a.group.mod(r, tok) : 0);
    const long qrow = (long)q0 + tok;
    const int lim = !real ? -1 : (a.causal ? min(tok + late, lk - 1) : lk - 1);
    Frag<T> q[L::NS], k[L::NS];
    load_row<T, DP>(q, real ? (const T*)a.q + qrow * a.q_row + (long)qh * a.q_head : nullptr, a.d, h);
    u32x4 v[NV];
    auto fetch = [&](int key) {
      load_row<T, DP>(k, key + c31 < key1 ? kp + (long)(key + c31) * a.k_row : nullptr, a.d, h);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int i = lane + n * 64, row = i / L::CH, c = i % L::CH;
        v[n] = key + row < key1 && c * L::EPC < a.d ? *(const u32x4*)(vp + (long)(key + row) * a.v_row + c * L::EPC)
                                                    : u32x4{0, 0, 0, 0};
      }
    };
    f32x16 o[L::NDT];
#pragma unroll
    for (int i = 0; i < L::NDT; ++i) o[i] = zero16();
    float m = NEG_INF, l = 0.f, lt = 0.f;                // maximum, sums of the rounded / the exact weights
    if (key0 < key1) fetch(key0);
    for (int key = key0; key < key1; key += 32) {
      f32x16 s = zero16();
#pragma unroll
      for (int i = 0; i < L::NS; ++i) s = mma16(k[i], q[i], s);
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int i = lane + n * 64, row = i / L::CH, c = i % L::CH;
        *(u32x4*)(slab + row * L::ROWB + ((c ^ L::f(row)) << 4)) = v[n];
      }
      __builtin_amdgcn_wave_barrier();
      if (key + 32 < key1) fetch(key + 32);
      const int last = min(lim, key1 - 1);
      if (__any(key + 31 > last)) {
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (key + 8 * (x >> 2) + 4 * h + (x & 3) > last) s[x] = NEG_INF;
      }
      float top = s[0];
#pragma unroll
      for (int x = 1; x < 16; ++x) top = fmaxf(top, s[x]);
      top = fmaxf(top, other_half(top));
      if (__any((top - m) * c2 > 8.f)) {
        const float mn = fmaxf(m, top);
        const float alpha = mn == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c2);
        m = mn;
        l *= alpha;
        lt *= alpha;
#pragma unroll
        for (int i = 0; i < L::NDT; ++i)
#pragma unroll
          for (int x = 0; x < 16; ++x) o[i][x] *= alpha;
      }
      const float mc = m == NEG_INF ? 0.f : -m * c2;
#pragma unroll
      for (int x = 0; x < 16; ++x) s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], c2, mc));
      if (a.lse) {
#pragma unroll
        for (int x = 0; x < 16; ++x) lt += s[x];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Frag<T> p = from_acc<T>(s, i);
        l = add_sum(p, l);
#pragma unroll
        for (int dt = 0; dt < L::NDT; ++dt) o[dt] = mma16(view.cols(slab + 16 * i * L::ROWB, dt), p, o[dt]);
      }
    }
    l += other_half(l);
    lt += other_half(lt);
    // the four quarters of the part: common maximum, then the sums in the order 0 + 2, 1 + 3, (0 2) + (1 3)
    __syncthreads();
    if (h == 0) { red[0][wave][c31] = m; red[1][wave][c31] = l; red[2][wave][c31] = lt; }
    __syncthreads();
    float mx = NEG_INF, lsum = 0.f, ltsum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, red[0][w][c31]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = red[0][w][c31], f = mw == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((mw - mx) * c2);
      lsum = fmaf(red[1][w][c31], f, lsum);
      ltsum = fmaf(red[2][w][c31], f, ltsum);
    }
    const float f = m == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((m - mx) * c2);
#pragma unroll
    for (int i = 0; i < L::NDT; ++i)
#pragma unroll
      for (int x = 0; x < 16; ++x) o[i][x] *= f;
    float* mine = (float*)(smem + (wave & 1) * JB);
#pragma unroll
    for (int step = 2; step > 0; step >>= 1) {
      if (wave >= step && wave < 2 * step) {
#pragma unroll
        for (int i = 0; i < L::NDT; ++i)
#pragma unroll
          for (int x = 0; x < 16; ++x) ((step == 1 ? (float*)smem : mine))[(i * 16 + x) * 64 + lane] = o[i][x];
      }
      __syncthreads();
      if (wave < step) {
#pragma unroll
        for (int i = 0; i < L::NDT; ++i)
#pragma unroll
          for (int x = 0; x < 16; ++x) o[i][x] += ((step == 1 ? (float*)smem : mine))[(i * 16 + x) * 64 + lane];
      }
      __syncthreads();
    }
    if (wave == 0 && real) {
      const long at = ((long)t.tile * a.total_q + qrow) * a.hq + qh;
      store_row<float, DP>(po + at * a.d, a.d, h, o, 1.f);
      if (h == 0) pml[at] = make_float4(mx, lsum, ltsum, 0.f);
    }
  }
}

// out and lse from the parts: one wave per (token, head)
template <typename T>
__global__ void __launch_bounds__(NT) k_attn_packed_join(const Args a, int part_keys,
                                                         const float* __restrict__ po, const float4* __restrict__ pml) {
  const long i = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= a.total_q * a.hq) return;
  const int lane = threadIdx.x & 63;
  int k0, lk;
  seq_rows(a.cu_k, a.nseq, a.total_k, find_row(a.cu_q, a.nseq, a.total_q, (int)(i / a.hq)), k0, lk);
  const int parts = (lk + part_keys - 1) / part_keys;
  const long step = a.total_q * a.hq;
  const float c2 = a.scale * LOG2E;
  float m = NEG_INF, l = 0.f, lt = 0.f, acc[2] = {0.f, 0.f};
  const bool in0 = lane < a.d, in1 = lane + 64 < a.d;
  for (int z0 = 0; z0 < parts; z0 += 64) {               // 64 parts at a time: a lane holds one part's maximum and sums
    const int n = min(64, parts - z0);
    const float4 ml = lane < n ? pml[(z0 + lane) * step + i] : make_float4(NEG_INF, 0.f, 0.f, 0.f);
    const float mn = fmaxf(m, wave_max(ml.x));
    const float old = m == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c2);
    const float w = ml.x == NEG_INF ? (ml.y == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f((ml.x - mn) * c2);
    m = mn;
    l = l * old + wave_sum(ml.y * w);
    lt = lt * old + wave_sum(ml.z * w);
    acc[0] *= old;
    acc[1] *= old;
    const float* p = po + (z0 * step + i) * a.d + lane;
    int z = 0;
    for (; z + 4 <= n; z += 4) {                         // four parts' loads in flight
      float x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = in0 ? p[(z + j) * step * a.d] : 0.f;
        y[j] = in1 ? p[(z + j) * step * a.d + 64] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float wz = __shfl(w, z + j, 64);
        acc[0] = fmaf(x[j], wz, acc[0]);
        acc[1] = fmaf(y[j], wz, acc[1]);
      }
    }
    for (; z < n; ++z) {
      const float wz = __shfl(w, z, 64);
      if (in0) acc[0] = fmaf(p[z * step * a.d], wz, acc[0]);
      if (in1) acc[1] = fmaf(p[z * step * a.d + 64], wz, acc[1]);
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (lane + 64 * e < a.d) {
      const float v = acc[e] * inv;
      Elem<T>::store((T*)a.out + i * a.d, lane + 64 * e, v);
      if constexpr (sizeof(T) == 2)
        if (a.out_low) Elem<T>::store((T*)a.out_low + i * a.d, lane + 64 * e, v - bf2f(f2bf(v)));
    }
  if (a.lse && lane == 0) a.lse[i] = lt > 0.f || lt != lt ? m * a.scale + __logf(lt) : NEG_INF;
}

// ------------------------------------------------------------------------------------------------
// delta_i = dO_i . O_i = sum_j P_ij dP_ij (the mean that the softmax gradient subtracts): 16 lanes per row.  The log-sum-exp's
// own gradient has the same form, d lse_i / d S_ij = P_ij, so dS = P o (dP - (delta - dlse)): it is taken off here.  A row
// that sees no key has none (its lse is the constant -inf).
template <typename T>
__global__ void __launch_bounds__(NT) k_attn_packed_delta(const Args a, float* __restrict__ delta) {
  const int c = (threadIdx.x & 15) * 8;                  // d <= 128
  const long rows = a.total_q * a.hq;
  for (long i = (long)blockIdx.x * 16 + (threadIdx.x >> 4); i < rows; i += (long)gridDim.x * 16) {
    float s = 0.f;
    if (c < a.d) {
      Frag<T> o, g, low;
      const T* pg = (const T*)a.dout + (i / a.hq) * a.do_row + (i % a.hq) * a.do_head + c;
      load8(o, (const T*)a.out + i * a.d + c);
      load8(g, pg);
      if (a.out_low) load8(low, (const T*)a.out_low + i * a.d + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf((float)o.v[e] + (a.out_low ? (float)low.v[e] : 0.f), (float)g.v[e], s);
    }
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) s += __shfl_xor(s, x, 64);
    if (c == 0) delta[i] = a.dlse && a.lse[i] != NEG_INF ? s - a.dlse[i] : s;
  }
}

// dQ: the forward's walk over the keys with dO beside Q; dQ^T += K^T dS^T.  KS: as in the forward
template <typename T, int DP, int KS>
__global__ void __launch_bounds__(NT, DP * sizeof(T) * KS > 256 ? 1 : 2)
k_attn_packed_dq(const Args a, const float* __restrict__ delta) {
  using L = Lay<T, DP>;
  constexpr int BM = 128 / KS, BN = L::ROWB > 256 ? 32 : 64, BT = BN * KS, TB = BT * L::ROWB;
  __shared__ __align__(16) char smem[4 * TB];          // K and V, two buffers
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int G = a.group.d, block = a.heads.div(blockIdx.x), kvh = a.heads.mod(blockIdx.x, block);
  const Tile t = find_tile(a.cu_q, a.nseq, a.total_q, G, BM, block, a.causal != 0);
  if (t.seq < 0) return;
  int k0, lk;
  seq_rows(a.cu_k, a.nseq, a.total_k, t.seq, k0, lk);
  const int ks = wave % KS, r = t.tile * BM + wave / KS * 32 + (lane & 31);
  const bool real = r < t.len * G;
  const int tok = real ? a.group.div(r) : 0, g = real ? a.group.mod(r, tok) : 0;
  const int late = lk - t.len;
  const int lim = !real ? -1 : (a.causal ? min(tok + late, lk - 1) : lk - 1);
  const int last_r = min((t.tile + 1) * BM, t.len * G) - 1;
  const int lim_blk = a.causal ? min(a.group.div(last_r) + late, lk - 1) : lk - 1;
  int lim_lo = lim, lim_hi = lim;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    lim_lo = min(lim_lo, __shfl_xor(lim_lo, o, 64));
    lim_hi = max(lim_hi, __shfl_xor(lim_hi, o, 64));
  }
  lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);
  lim_hi = __builtin_amdgcn_readfirstlane(lim_hi);
  const long qrow = (long)t.start + tok;
  const int qh = kvh * G + g;
  Frag<T> q[L::NS], go[L::NS];
  load_row<T, DP>(q, real ? (const T*)a.q + qrow * a.q_row + (long)qh * a.q_head : nullptr, a.d, h);
  load_row<T, DP>(go, real ? (const T*)a.dout + qrow * a.do_row + (long)qh * a.do_head : nullptr, a.d, h);
  settle(q);
  settle(go);
  const float c2 = a.scale * LOG2E;
  float le = real ? a.lse[qrow * a.hq + qh] : 0.f;
  le = le == NEG_INF ? 0.f : -le * LOG2E;
  float dl = real ? delta[qrow * a.hq + qh] : 0.f;
  asm volatile("" : "+v"(le), "+v"(dl));
  const T* kp = (const T*)a.k + (long)k0 * a.k_row + (long)kvh * a.k_head;
  const T* vp = (const T*)a.v + (long)k0 * a.v_row + (long)kvh * a.v_head;

  f32x16 dq[L::NDT];
#pragma unroll
  for (int i = 0; i < L::NDT; ++i) dq[i] = zero16();
  const View<T, DP> view(lane);
  const int ntile = (lim_blk + BT) / BT;
  const unsigned lds0 = lds_at(smem);
  KeyTiles<T, DP, BT> sk(kp, a.k_row, lim_blk + 1, a.d), sv(vp, a.v_row, lim_blk + 1, a.d);
  auto fetch = [&](int kt) {
    const unsigned at = lds0 + (kt & 1) * 2 * TB;
    sk.next(kt, at);
    sv.next(kt, at + TB);
  };
  if (ntile > 0) fetch(0);
  for (int kt = 0; kt < ntile; ++kt) {
    arrived();
    __syncthreads();                                     // tile kt is here, the other buffer is no longer read
    const char* tk = smem + (kt & 1) * 2 * TB + ks * BN * L::ROWB;
    const char* tv = tk + TB;
    if (kt + 1 < ntile) fetch(kt + 1);
#pragma unroll 1
    for (int j = 0; j < BN / 32; ++j) {
      const int key = kt * BT + ks * BN + 32 * j;
      if (key > lim_hi) break;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int i = 0; i < L::NS; ++i) {
        s = mma16(view.rows(tk + j * 32 * L::ROWB, i), q[i], s);
        dp = mma16(view.rows(tv + j * 32 * L::ROWB, i), go[i], dp);
      }
      if (key + 31 > lim_lo) {
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (key + 8 * (x >> 2) + 4 * h + (x & 3) > lim) s[x] = NEG_INF;
      }
#pragma unroll
      for (int x = 0; x < 16; ++x) s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], c2, le)) * (dp[x] - dl);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Frag<T> p = from_acc<T>(s, i);
#pragma unroll
        for (int dt = 0; dt < L::NDT; ++dt)
          dq[dt] = mma16(view.cols(tk + (32 * j + 16 * i) * L::ROWB, dt), p, dq[dt]);
      }
    }
  }
  if constexpr (KS > 1) {
    static_assert(KS == 2 && 2 * 16 * L::NDT * 64 * 4 <= 4 * TB, "the second wave's sums fit the tiles' LDS");
    float* half = (float*)smem + wave / KS * 16 * L::NDT * 64 + lane;
    __syncthreads();
    if (ks == 1) {
#pragma unroll
      for (int i = 0; i < L::NDT; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) half[(i * 16 + x) * 64] = dq[i][x];
    }
    __syncthreads();
    if (ks == 1) return;
#pragma unroll
    for (int i = 0; i < L::NDT; ++i)
#pragma unroll
      for (int x = 0; x < 16; ++x) dq[i][x] += half[(i * 16 + x) * 64];
  }
  if (real) store_row<T, DP>((T*)a.dq + (qrow * a.hq + qh) * a.d, a.d, h, dq, a.scale);
}

// dK, dV: a block holds 64 keys and walks over the packed rows of its sequence (all heads of the group), 64 rows a tile:
// waves 0 and 2 own the first 32 keys, 1 and 3 the others; 0 and 1 take a tile's first 32 rows, 2 and 3 the others, and
// the two halves are added through LDS at the end.  (Blocks of 128 keys whose waves all walk over every row: half as many,
// twice as long.)  dK and dV of 32 keys fill 128 registers a lane, so K and V stay in LDS and Q and dO have one buffer each:
// two blocks then share a CU and one computes while the other's tile arrives.  (4096 + 2991 causal tokens, 16 heads of 128 on
// 4: K and V in registers, two buffers, one block a CU 386 us, this 318.)  Where the keys give few blocks, `parts` blocks share
// a key tile's rows and write fp32 parts that k_attn_packed_sum adds in order.
template <typename T, int DP>
__global__ void __launch_bounds__(NT, DP * sizeof(T) > 256 ? 1 : 2)
k_attn_packed_dkv(const Args a, const float* __restrict__ delta, float* __restrict__ part_dk, int parts) {
  using L = Lay<T, DP>;
  constexpr int BK = KEYS, BR = 64, TB = BR * L::ROWB;
  __shared__ __align__(16) char smem[4 * TB];          // Q, dO, K, V
  __shared__ __align__(16) float st[2][BR];           // -lse log2 e and delta of the rows
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int part = blockIdx.x % parts, x = blockIdx.x / parts;          // a tile's parts side by side: long blocks first
  const int G = a.group.d, block = a.heads.div(x), kvh = a.heads.mod(x, block);
  const Tile t = find_tile(a.cu_k, a.nseq, a.total_k, 1, BK, block, false);
  if (t.seq < 0) return;
  int q0, lq;
  seq_rows(a.cu_q, a.nseq, a.total_q, t.seq, q0, lq);
  const int kh = wave & 1, rh = wave >> 1;
  const int key = t.tile * BK + kh * 32 + (lane & 31);
  const bool real = key < t.len;
  const long krow = (long)t.start + key;
  const int late = t.len - lq;
  // causal: row (token i) sees key j iff i >= j - late
  const int first_tok = a.causal ? max(t.tile * BK - late, 0) : 0;
  const int first_mine = a.causal ? key - late : 0;      // first token that sees this lane's key
  const int wave_last = a.causal ? t.tile * BK + kh * 32 + 31 - late : 0;   // token that sees all of the wave's keys
  const int rows = lq * G;
  const float c2 = a.scale * LOG2E;

  f32x16 dk[L::NDT], dv[L::NDT];
#pragma unroll
  for (int i = 0; i < L::NDT; ++i) { dk[i] = zero16(); dv[i] = zero16(); }
  const View<T, DP> view(lane);
  // K and V of the block, zeros behind the last key and column (there the tiles' rows hold copies)
  for (int i = threadIdx.x; i < BK * L::CH; i += NT) {
    const int row = i / L::CH, c = i % L::CH;
    const bool in = t.tile * BK + row < t.len && c * L::EPC < a.d;
    const long at = (long)t.start + t.tile * BK + row;
    const int to = row * L::ROWB + ((c ^ L::f(row)) << 4);
    const T* kp = (const T*)a.k + at * a.k_row + (long)kvh * a.k_head + c * L::EPC;
    const T* vp = (const T*)a.v + at * a.v_row + (long)kvh * a.v_head + c * L::EPC;
    *(u32x4*)(smem + 2 * TB + to) = in ? *(const u32x4*)kp : u32x4{0, 0, 0, 0};
    *(u32x4*)(smem + 3 * TB + to) = in ? *(const u32x4*)vp : u32x4{0, 0, 0, 0};
  }
  const char* tk = smem + 2 * TB + kh * 32 * L::ROWB;    // this wave's keys
  const char* tv = tk + TB;
  const T* qp = (const T*)a.q + (long)q0 * a.q_row + (long)kvh * G * a.q_head;
  const T* gp = (const T*)a.dout + (long)q0 * a.do_row + (long)kvh * G * a.do_head;
  const long sbase = (long)q0 * a.hq + (long)kvh * G;
  const unsigned lds0 = lds_at(smem);
  float stat = 0.f;
  const int used = a.group.div(BR) * G, toks = a.group.div(BR);          // rows and tokens of a tile
  const RowTiles<T, DP, BR> sq(qp, a.q_row, a.q_head, used, a.d, a.group), sg(gp, a.do_row, a.do_head, used, a.d, a.group);
  const int t0 = first_tok / toks, tn = (lq + toks - 1) / toks;          // the tiles that this block needs
  auto stats = [&](int rr) {
    if (threadIdx.x < 2 * BR) {
      const int slot = threadIdx.x & (BR - 1), x = rr + slot;
      stat = 0.f;
      if (x < rows && slot < used) {
        const int tk = a.group.div(x);
        const long at = sbase + (long)tk * a.hq + a.group.mod(x, tk);
        stat = threadIdx.x < BR ? a.lse[at] : delta[at];
      }
    }
  };
  // from the last rows, which every block of the sequence needs, backwards: blocks that run together read the same tiles
  int tile = tn - 1 - part;
  for (bool first = true; tile >= t0; tile -= parts, first = false) {
    const int rr = tile * used;
    __syncthreads();                                     // the tile before is no longer read
    if (first) {
      sq.last(a.q_row, a.q_head, rr, rows, a.d, a.group, lds0);
      sg.last(a.do_row, a.do_head, rr, rows, a.d, a.group, lds0 + TB);
    } else {
      sq.send_tile((long)tile * toks * a.q_row, lds0);
      sg.send_tile((long)tile * toks * a.do_row, lds0 + TB);
    }
    stats(rr);
    arrived();
    if (threadIdx.x < BR) st[0][threadIdx.x] = stat == NEG_INF ? 0.f : -stat * LOG2E;
    else if (threadIdx.x < 2 * BR) st[1][threadIdx.x - BR] = stat;
    __syncthreads();
    const int j = rh * 32, rj = rr + j;
    const char* tq = smem + j * L::ROWB;
    const char* tg = tq + TB;
    f32x16 s = zero16(), dp = zero16();
#pragma unroll
    for (int i = 0; i < L::NS; ++i) {
      s = mma16(view.rows(tq, i), view.rows(tk, i), s);
      dp = mma16(view.rows(tg, i), view.rows(tv, i), dp);
    }
    const int end = min(rr + used, rows);
    const bool edge = rj + 32 > end || a.group.div(rj) < wave_last;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const f32x4 le = *(const f32x4*)&st[0][j + 8 * y + 4 * h];
#pragma unroll
      for (int x = 0; x < 4; ++x) s[4 * y + x] = __builtin_amdgcn_exp2f(fmaf(s[4 * y + x], c2, le[x]));
    }
    if (edge) {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int at = rj + 8 * (x >> 2) + 4 * h + (x & 3);
        s[x] = at >= end || a.group.div(at) < first_mine ? 0.f : s[x];
      }
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const f32x4 dl = *(const f32x4*)&st[1][j + 8 * y + 4 * h];
#pragma unroll
      for (int x = 0; x < 4; ++x) dp[4 * y + x] = s[4 * y + x] * (dp[4 * y + x] - dl[x]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Frag<T> p = from_acc<T>(s, i), ds = from_acc<T>(dp, i);
#pragma unroll
      for (int dt = 0; dt < L::NDT; ++dt) {
        dv[dt] = mma16(view.cols(tg + 16 * i * L::ROWB, dt), p, dv[dt]);
        dk[dt] = mma16(view.cols(tq + 16 * i * L::ROWB, dt), ds, dk[dt]);
      }
    }
  }
  // the second half's sums, then the first half adds them
  __syncthreads();
  float* half = (float*)smem + kh * 2 * 16 * L::NDT * 64 + lane;
  if (rh == 1) {
#pragma unroll
    for (int i = 0; i < L::NDT; ++i)
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        half[(i * 16 + x) * 64] = dk[i][x];
        half[((L::NDT + i) * 16 + x) * 64] = dv[i][x];
      }
  }
  __syncthreads();
  if (rh == 1) return;
#pragma unroll
  for (int i = 0; i < L::NDT; ++i)
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      dk[i][x] += half[(i * 16 + x) * 64];
      dv[i][x] += half[((L::NDT + i) * 16 + x) * 64];
    }
  if (!real) return;
  const long at = (krow * a.heads.d + kvh) * a.d;
  if (part_dk == nullptr) {
    store_row<T, DP>((T*)a.dv + at, a.d, h, dv, 1.f);
    store_row<T, DP>((T*)a.dk + at, a.d, h, dk, a.scale);
  } else {
    const long all = a.total_k * a.heads.d * a.d;
    store_row<float, DP>(part_dk + (2 * part) * all + at, a.d, h, dk, a.scale);
    store_row<float, DP>(part_dk + (2 * part + 1) * all + at, a.d, h, dv, 1.f);
  }
}

// dk and dv from `parts` partial sums, in their order: 8 values a thread
template <typename T>
__global__ void __launch_bounds__(NT) k_attn_packed_sum(const Args a, int parts, const float* __restrict__ part) {
  const long all = a.total_k * a.heads.d * a.d;
  for (long i = ((long)blockIdx.x * NT + threadIdx.x) * 8; i < 2 * all; i += (long)gridDim.x * NT * 8) {
    Frag<float> s, x;
    load8(s, part + i);
    for (int z = 1; z < parts; ++z) {
      load8(x, part + 2 * z * all + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) s.v[e] += x.v[e];
    }
    T* to = i < all ? (T*)a.dk + i : (T*)a.dv + (i - all);
    store4(to, s.v[0], s.v[1], s.v[2], s.v[3]);
    store4(to + 4, s.v[4], s.v[5], s.v[6], s.v[7]);
  }
}

// ------------------------------------------------------------------------------------------------ host
bool aligned(const void* p, long row, long head, int es) {
  return p != nullptr && ((uintptr_t)p & 15) == 0 && (row * es) % 16 == 0 && (head * es) % 16 == 0 && row >= 0 && head >= 0;
}

int check_shape(const hv_attn_packed_args* a) {
  if (a == nullptr || (a->dtype != HV_F32 && a->dtype != HV_BF16)) return HV_EINVAL;
  if (a->hq <= 0 || a->hkv <= 0 || a->hq % a->hkv || a->nseq < 0 || a->total_q < 0 || a->total_k < 0) return HV_EINVAL;
  if (!(a->scale > 0.f) || a->scale > 3.0e38f) return HV_EINVAL;
  if (a->d <= 0 || a->d % 8 || a->d > 128 || a->hq > 1024 || a->hq / a->hkv > 64) return HV_EUNSUPPORTED;
  if (a->total_q >= (1L << 30) || a->total_q * (a->hq / a->hkv) >= (1L << 30) || a->total_k >= (1L << 30)) return HV_EUNSUPPORTED;
  return HV_OK;
}

int check_args(const hv_attn_packed_args* a) {
  const int rc = check_shape(a);
  if (rc != HV_OK) return rc;
  if (a->cu_q == nullptr || a->cu_k == nullptr) return HV_EINVAL;
  const int es = a->dtype == HV_BF16 ? 2 : 4;
  if (a->total_q && (!aligned(a->q, a->q_row, a->q_head, es))) return HV_EINVAL;
  if (a->total_k && (!aligned(a->k, a->k_row, a->k_head, es) || !aligned(a->v, a->v_row, a->v_head, es))) return HV_EINVAL;
  return HV_OK;
}

constexpr long MAX_BLOCKS = 1L << 24;                    // a grid stays below 2^32 threads

// blocks that cover `total` rows in nseq sequences and the two ranges outside of them, BM packed rows each
long tile_bound(long total, int nseq, int G, int BM) { return total * G / BM + nseq + 2; }

// rows of the parts' workspace
size_t part_rows(const hv_attn_packed_args& a, long n) { return (size_t)((a.total_k + n - 1) / n) * a.total_q * a.hq; }

// Keys of a part in the few-rows form, 0: the tile form.  The few-rows form reads a sequence's keys once per 32 of its rows
// and needs a second launch; the tile form gives one block all the keys of 64 or 128 rows, 128 keys a step.  Averages per
// sequence decide: few rows where there are 512 keys for it and for each 32 rows (at most 8 times).  Measured, tile / few
// rows, us: 1 x 4 rows, 4096 keys of 128: 69 / 14; 8 x 4, 1024: 22 / 15; 64 x 4, 1024: 47 / 45; 8 x 64, 1024: 21 / 26; 1 x 64,
// 4096: 59 / 22; 64 columns: 64 x 1, 512: 12 / 18; 8 x 64, 1024: 13 / 19; 1 x 128, 4096: 35 / 25.
// Parts are sized for about two blocks per CU (12 queries against 85 056 keys, 8 heads: 78 us, four 85 us), 128 keys (one
// slab per wave) at least.  The join has a wave per (token, head): the tile form also where those pass a grid's 2^32 threads.
int part_keys(const hv_attn_packed_args& a) {
  if (a.nseq == 0 || a.total_q == 0 || a.total_k == 0 || a.total_q * a.hq > (1L << 26) - 4) return 0;
  const long tiles = (a.total_q * (a.hq / a.hkv) + 32L * a.nseq - 1) / (32L * a.nseq);      // of 32 rows a sequence
  if (tiles > 8 || a.total_k < 512 * (tiles + 1) * a.nseq) return 0;
  const long n0 = min((a.total_k * a.hkv + 511) / 512, a.total_k);      // <= 2^30, also with more than 512 heads
  long n = (n0 + 127) / 128 * 128;
  // longer parts where the workspace (the number of parts that one sequence with all the keys would have, for every row)
  // would pass 256 MiB: many sequences, which are short against all keys together
  while (n < a.total_k && part_rows(a, n) * (a.d + 4) * sizeof(float) > (256u << 20)) n *= 2;
  return tile_bound(a.total_k, a.nseq, 1, (int)n) * a.hkv < MAX_BLOCKS ? (int)n : 0;
}

template <typename T, int DP> void launch_keys(const Args& a, int n, hipStream_t s) {
  const size_t rows = part_rows(a, n);
  float* po = (float*)a.work;
  float4* pml = (float4*)(po + rows * a.d);
  const unsigned blocks = (unsigned)(tile_bound(a.total_k, a.nseq, 1, n) * a.hkv);
  k_attn_packed_keys<T, DP><<<blocks, NT, 0, s>>>(a, n, po, pml);
  k_attn_packed_join<T><<<hv_cdiv(a.total_q * a.hq, 4), NT, 0, s>>>(a, n, po, pml);
}

// Waves that share 32 rows of the forward's tile form: two where blocks of 128 rows would not give every CU two.  (4269 image
// tokens, 8 heads of 32, 272 such blocks: KS 1 / 2 / 4 take 24.9 / 16.7 / 22.4 us; 8569 tokens, 16 heads of 64 on 4, 1076
// blocks: 88.7 / 97.1 us.)
int key_split(const hv_attn_packed_args& a) {
  return (a.total_q * (a.hq / a.hkv) + 127) / 128 * a.hkv < 512 ? 2 : 1;
}

template <typename T, int DP, int KS> void launch_forward_ks(const Args& a, hipStream_t s) {
  const unsigned blocks = (unsigned)(tile_bound(a.total_q, a.nseq, a.group.d, 128 / KS) * a.hkv);
  if (a.lse != nullptr || a.out_low != nullptr) k_attn_packed<T, DP, true, KS><<<blocks, NT, 0, s>>>(a);
  else k_attn_packed<T, DP, false, KS><<<blocks, NT, 0, s>>>(a);
}
template <typename T, int DP> void launch_forward(const Args& a, hipStream_t s) {
  if (key_split(a) == 1) launch_forward_ks<T, DP, 1>(a, s);
  else launch_forward_ks<T, DP, 2>(a, s);
}

// Blocks that share the rows of a key tile (see k_attn_packed_dkv): up to four blocks per CU, eight row tiles each at least
int row_parts(const hv_attn_packed_args& a) {
  const int used = 64 / (a.hq / a.hkv) * (a.hq / a.hkv);
  const long blocks = (a.total_k + KEYS - 1) / KEYS * a.hkv, tiles = a.total_q * (a.hq / a.hkv) / used / (a.nseq > 0 ? a.nseq : 1);
  const long n = blocks > 0 ? min(1024 / blocks, tiles / 8) : 1;
  return (int)(n < 1 ? 1 : n > 8 ? 8 : n);
}
size_t delta_bytes(const hv_attn_packed_args& a) { return ((size_t)a.total_q * a.hq * sizeof(float) + 63) / 64 * 64; }

template <typename T, int DP>
void launch_backward(const Args& a, unsigned bk, hipStream_t s) {
  float* delta = (float*)a.work;
  float* part = (float*)((char*)a.work + delta_bytes(a));
  const int parts = row_parts(a);
  if (a.total_q) {
    k_attn_packed_delta<T><<<(unsigned)min((a.total_q * a.hq + 15) / 16, 1L << 20), NT, 0, s>>>(a, delta);
    if (a.dq && key_split(a) == 1)
      k_attn_packed_dq<T, DP, 1><<<(unsigned)(tile_bound(a.total_q, a.nseq, a.group.d, 128) * a.hkv), NT, 0, s>>>(a, delta);
    else if (a.dq)
      k_attn_packed_dq<T, DP, 2><<<(unsigned)(tile_bound(a.total_q, a.nseq, a.group.d, 64) * a.hkv), NT, 0, s>>>(a, delta);
  }
  if (a.total_k && a.dk) {
    k_attn_packed_dkv<T, DP><<<bk * parts, NT, 0, s>>>(a, delta, parts > 1 ? part : nullptr, parts);
    if (parts > 1)
      k_attn_packed_sum<T><<<(unsigned)min((2 * a.total_k * a.hkv * a.d / 8 + NT - 1) / NT, 4096L), NT, 0, s>>>(a, parts, part);
  }
}

// the tile width for a head dimension: the next of 32 / 64 / 128
#define HV_HEAD_DIM(d, CALL, ...)                  \
  do {                                             \
    if ((d) <= 32) CALL<T, 32>(__VA_ARGS__);       \
    else if ((d) <= 64) CALL<T, 64>(__VA_ARGS__);  \
    else CALL<T, 128>(__VA_ARGS__);                \
  } while (0)

}  // namespace

extern "C" size_t hv_attn_packed_args_bytes(void) { return sizeof(hv_attn_packed_args); }

extern "C" size_t hv_attn_packed_work_bytes(const hv_attn_packed_args* a) {
  if (check_shape(a) != HV_OK) return 0;
  const int n = part_keys(*a);
  return n ? part_rows(*a, n) * (a->d + 4) * sizeof(float) : 0;
}

extern "C" int hv_attn_packed(const hv_attn_packed_args* a, hv_stream_t stream) {
  const int rc = check_args(a);
  if (rc != HV_OK) return rc;
  if (a->total_q == 0) return HV_OK;
  if (a->out == nullptr || ((uintptr_t)a->out & 15) || ((uintptr_t)a->out_low & 15)) return HV_EINVAL;
  if (tile_bound(a->total_q, a->nseq, a->hq / a->hkv, 64) * a->hkv >= MAX_BLOCKS) return HV_EUNSUPPORTED;
  hipStream_t s = (hipStream_t)stream;
  const int n = part_keys(*a);
  if (n) {
    if (a->work == nullptr || ((uintptr_t)a->work & 15)) return HV_EINVAL;
    HV_DISPATCH(a->dtype, HV_HEAD_DIM(a->d, launch_keys, Args(*a), n, s));
  } else
    HV_DISPATCH(a->dtype, HV_HEAD_DIM(a->d, launch_forward, Args(*a), s));
  HV_CHECK_LAUNCH();
  hv_diag_count(HV_KF_ATTN_PACKED);
  return HV_OK;
}

extern "C" size_t hv_attn_packed_backward_work_bytes(const hv_attn_packed_args* a) {
  if (check_shape(a) != HV_OK) return 0;
  const int n = row_parts(*a);
  return delta_bytes(*a) + (n > 1 ? (size_t)n * 2 * a->total_k * a->hkv * a->d * sizeof(float) : 0);
}

extern "C" int hv_attn_packed_backward(const hv_attn_packed_args* a, hv_stream_t stream) {
  const int rc = check_args(a);
  if (rc != HV_OK) return rc;
  const int es = a->dtype == HV_BF16 ? 2 : 4;
  if (a->total_q && (!aligned(a->dout, a->do_row, a->do_head, es) || !aligned(a->out, 0, 0, es) ||
                     ((uintptr_t)a->out_low & 15) || a->lse == nullptr ||
                     ((uintptr_t)a->dq & 15) || a->work == nullptr))
    return HV_EINVAL;
  if ((a->dk == nullptr) != (a->dv == nullptr) || ((uintptr_t)a->dk & 15) || ((uintptr_t)a->dv & 15)) return HV_EINVAL;
  // a tile of 64 packed rows is addressed with 32-bit offsets
  const long reach = max(a->q_row, a->do_row) * 64 + max(a->q_head, a->do_head) * 64;
  if (reach >= (1L << 29)) return HV_EUNSUPPORTED;
  const long bq = tile_bound(a->total_q, a->nseq, a->hq / a->hkv, 64) * a->hkv;
  const long bk = tile_bound(a->total_k, a->nseq, 1, KEYS) * a->hkv;
  if (bq >= MAX_BLOCKS || bk >= MAX_BLOCKS / 8) return HV_EUNSUPPORTED;
  hipStream_t s = (hipStream_t)stream;
  HV_DISPATCH(a->dtype, HV_HEAD_DIM(a->d, launch_backward, Args(*a), (unsigned)bk, s));
  HV_CHECK_LAUNCH();
  hv_diag_count(HV_KF_ATTN_PACKED);
  return HV_OK;
}
