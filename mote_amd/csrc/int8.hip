// Products in 8-bit integers: y = x W^T with one fp32 scale per token of x and per output channel of W
// (mote_quantize_rows / mote_int8_linear; the rounding points stand in mote_relation.h).
//
// acc = sum_k xq wq runs on v_mfma_i32_16x16x64_i8, exact in 32 bits; y = (acc sx) sw in fp32, rounded once.
// One fragment convention for both operands: lane l holds 16 consecutive k of row l % 16, k group l / 16.
// Rows of xq and wq are Kp = K rounded up to 128 bytes, xq's zero past K, so no product looks at K.
#include "tiles.hpp"
#include "params.hpp"

namespace mote {

typedef __attribute__((ext_vector_type(4))) int i32x4;

constexpr float kSmall8 = 0x1p-120f;  // a row whose maximum is below stores zeros (127 / max would overflow)
constexpr int kMaxK8 = 131072;        // sums stay below 2^31: K 127^2
inline __host__ __device__ int64_t padded_k8(int64_t K) { return (K + 127) / 128 * 128; }

__device__ __forceinline__ i32x4 mma8(const Chunk& a, const Chunk& b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// bits of |x|: unsigned order is the order of magnitudes, infinities and NaNs on top
__device__ __forceinline__ uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
struct Scale8 {
  float scale, inv;
};
__device__ __forceinline__ Scale8 scale8(uint32_t top) {
  Scale8 s;
  const float a = __uint_as_float(top);
  const bool finite = top < 0x7f800000u, live = finite && a >= kSmall8;
  s.inv = live ? 127.0f / a : 0.f;
  s.scale = live ? a / 127.0f : finite ? 0.f : __builtin_nanf("");
  return s;
}
// the code of x, as a byte (inv 0: a row without a scale, whose infinities and NaNs must not come through)
__device__ __forceinline__ uint32_t code8(float x, float inv) {
  return inv == 0.f ? 0u : uint32_t(int(rintf(x * inv))) & 0xffu;
}

// x[k .. k + 8) of a row of K elements, zeros past its end; `wide`: the row is 16-byte aligned
template <typename T>
__device__ __forceinline__ void row_octet(const T* row, int k, int K, bool wide, float (&x)[8]) {
  using E = Elem<T>;
  if (wide && k + 8 <= K) {
    if constexpr (sizeof(T) == 2) {
      const Chunk c = load_chunk(row + k);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = __uint_as_float(c.w[j] << 16);
        x[2 * j + 1] = __uint_as_float(c.w[j] & 0xffff0000u);
      }
    } else {
      const float4 a = reinterpret_cast<const float4*>(row + k)[0], b = reinterpret_cast<const float4*>(row + k)[1];
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = k + j < K ? E::to_f(row[k + j]) : 0.f;
  }
}

__device__ __forceinline__ uint32_t wave_umax(uint32_t m) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = max(m, uint32_t(__shfl_xor(int(m), o, 64)));
  return m;
}

// ------------------------------------------------------------------------------------------------
// Rows in 8 bits: a wave per row, the row in registers up to 64 * 8 * NC values (beyond, read twice)
// ------------------------------------------------------------------------------------------------
constexpr int kQuantWaves = 4;

template <typename T>
__global__ void __launch_bounds__(64 * kQuantWaves)
quantize_rows_kernel(const T* x, int64_t x_sr, int M, int K, int Kp, bool wide, int8_t* q, float* scale) {
  constexpr int NC = 4;
  const int lane = threadIdx.x & 63;
  const int m = blockIdx.x * kQuantWaves + (threadIdx.x >> 6);
  if (m >= M) return;
  const T* row = x + int64_t(m) * x_sr;
  float v[NC][8];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int k = (i * 64 + lane) * 8;
    if (k < Kp) row_octet<T>(row, k, K, wide, v[i]);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, mag_bits(v[i][j]));
  }
  for (int k = (NC * 64 + lane) * 8; k < Kp; k += 512) {
    float w[8];
    row_octet<T>(row, k, K, wide, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, mag_bits(w[j]));
  }
  const Scale8 s = scale8(wave_umax(top));
  int8_t* out = q + int64_t(m) * Kp;
  auto put = [&](int k, const float (&w)[8]) {
    uint2 c = make_uint2(0u, 0u);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c.x |= code8(w[j], s.inv) << (8 * j);
      c.y |= code8(w[4 + j], s.inv) << (8 * j);
    }
    *reinterpret_cast<uint2*>(out + k) = c;
  };
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int k = (i * 64 + lane) * 8;
    if (k < Kp) put(k, v[i]);
  }
  for (int k = (NC * 64 + lane) * 8; k < Kp; k += 512) {
    float w[8];
    row_octet<T>(row, k, K, wide, w);
    put(k, w);
  }
  if (lane == 0) scale[m] = s.scale;
}

// ------------------------------------------------------------------------------------------------
// Few tokens (M <= 16): x is quantised where it is multiplied. One workgroup (4 waves) per 16 channels,
// the 64-wide k steps dealt to the waves in runs; a wave issues every load of its W rows, then reads its
// part of x, agrees on the rows' maxima with the other waves through LDS, and multiplies. The four
// partial sums are integers: their order does not matter.
// ------------------------------------------------------------------------------------------------
constexpr int kFewWaves = 4;
constexpr int kFewMaxK = 4096;

struct Few8Params {
  const void* x; int64_t x_sr;
  const int8_t* w;
  const float* sw;
  void* y; int64_t y_sr;
  const unsigned char* run;
  const float* g; float* xm;
  int M, N, K, Kp, heads;
  int wide;
};

template <typename T, int KS>
__global__ void __launch_bounds__(64 * kFewWaves) int8_few_kernel(const Few8Params p) {
  using E = Elem<T>;
  __shared__ uint32_t tops[kFewWaves][16];
  __shared__ __align__(16) int part[kFewWaves][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int nks = p.Kp / 64;                                 // k steps, an even number
  const int per = (nks + kFewWaves - 1) / kFewWaves;         // <= KS
  const int s0 = min(wave * per, nks), s1 = min(s0 + per, nks);
  const int8_t* wrow = p.w + int64_t(min(n0 + r, p.N - 1)) * p.Kp + 16 * q;
  const T* xrow = reinterpret_cast<const T*>(p.x) + int64_t(min(r, p.M - 1)) * p.x_sr;
  Chunk a[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s)
    if (s0 + s < s1) a[s] = load_chunk(wrow + 64 * (s0 + s));
  float x[KS][16];
  uint32_t top = 0;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    if (s0 + s < s1) {
      float lo[8], hi[8];
      row_octet<T>(xrow, 64 * (s0 + s) + 16 * q, p.K, p.wide, lo);
      row_octet<T>(xrow, 64 * (s0 + s) + 16 * q + 8, p.K, p.wide, hi);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[s][j] = lo[j];
        x[s][8 + j] = hi[j];
        top = max(top, max(mag_bits(lo[j]), mag_bits(hi[j])));
      }
    }
  }
  // the decode step's exchange mass on the side: workgroup 0, wave 1, lane b < M
  const int xb = int(threadIdx.x) - 64;
  const bool xm_lane = p.xm != nullptr && blockIdx.x == 0 && xb >= 0 && xb < p.M;
  float gsum = 0.f;
  if (xm_lane) {
    const float* gb = p.g + int64_t(xb) * p.heads;
    for (int h0 = 0; h0 < p.heads; h0 += 8) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = gb[min(h0 + j, p.heads - 1)];
#pragma unroll
      for (int j = 0; j < 8; ++j) gsum = h0 + j < p.heads ? gsum + v[j] : gsum;
    }
  }
  if (p.run && p.run[0] == 0) return;  // uniform: the whole workgroup leaves before its barrier
  if (xm_lane) p.xm[xb] = gsum / float(p.heads);
  top = max(top, uint32_t(__shfl_xor(int(top), 16, 64)));
  top = max(top, uint32_t(__shfl_xor(int(top), 32, 64)));
  if (q == 0) tops[wave][r] = top;
  __syncthreads();
  top = tops[0][r];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) top = max(top, tops[w][r]);
  const Scale8 sc = scale8(top);
  i32x4 acc = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    if (s0 + s < s1) {
      Chunk b;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        b.w[j] = code8(x[s][4 * j], sc.inv) | code8(x[s][4 * j + 1], sc.inv) << 8 |
                 code8(x[s][4 * j + 2], sc.inv) << 16 | code8(x[s][4 * j + 3], sc.inv) << 24;
      acc = mma8(a[s], b, acc);
    }
  }
  // acc: channels 4 q + i of token r
#pragma unroll
  for (int i = 0; i < 4; ++i) part[wave][4 * q + i][r] = acc[i];
  __syncthreads();
  if (wave == 0 && r < p.M) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int f = 4 * q + i;
      int v = part[0][f][r];
#pragma unroll
      for (int w = 1; w < kFewWaves; ++w) v += part[w][f][r];
      if (n0 + f < p.N)
        reinterpret_cast<T*>(p.y)[int64_t(r) * p.y_sr + n0 + f] = E::from_f(float(v) * sc.scale * p.sw[n0 + f]);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Many tokens: a tile of 128 tokens x 128 channels per workgroup (4 waves, 64 x 64 each), stages of 128 k
// brought to LDS with global_load_lds, 16-byte chunks swizzled by the row's low bits.
// ------------------------------------------------------------------------------------------------
constexpr int kTile8 = 128;
constexpr int kStage8 = 2 * kTile8 * 128;  // bytes

struct Many8Params {
  const int8_t* x;   // [M, Kp]
  const float* sx;
  const int8_t* w;   // [N, Kp]
  const float* sw;
  void* y; int64_t y_sr;
  int M, N, Kp, ntok, nch;
};

template <typename T>
__global__ void __launch_bounds__(256) int8_many_kernel(const Many8Params p) {
  using E = Elem<T>;
  __shared__ __align__(16) int8_t smem[2 * kStage8];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nwg = p.ntok * p.nch, per = (nwg + 7) / 8;
  const int seq = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (seq >= nwg) return;
  const int m0 = seq / p.nch * kTile8, n0 = seq % p.nch * kTile8;
  // a stage is 256 rows (128 of W, 128 of x) of 8 chunks: 32 wave transfers of 8 rows, 8 per wave
  const int lrow = lane >> 3, lch = (lane & 7) ^ lrow;  // rows 8 g + lrow: the swizzle is row & 7 = lrow
  const int8_t* src[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = (wave * 8 + i) * 8 + lrow;
    src[i] = (row < kTile8 ? p.w + int64_t(min(n0 + row, p.N - 1)) * p.Kp
                           : p.x + int64_t(min(m0 + row - kTile8, p.M - 1)) * p.Kp) + 16 * lch;
  }
  auto issue = [&](int kb, int slot) {
#pragma unroll
    for (int i = 0; i < 8; ++i) lds_dma16(src[i] + 128 * kb, smem + slot * kStage8 + (wave * 8 + i) * 1024);
  };
  const int wn = wave & 1, wm = wave >> 1;
  i32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  const int nk = p.Kp / 128;
  issue(0, 0);
  for (int kb = 0; kb < nk; ++kb) {
    __builtin_amdgcn_s_waitcnt(0);
    lds_barrier();  // stage kb is in LDS, and every wave is done with the slot the next one goes to
    if (kb + 1 < nk) issue(kb + 1, (kb + 1) & 1);
    const int8_t* st = smem + (kb & 1) * kStage8;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int ch = 4 * kk + (lane >> 4), r = lane & 15;
      Chunk a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = load_chunk(st + (wn * 64 + 16 * i + r) * 128 + ((ch ^ (r & 7)) * 16));
        b[i] = load_chunk(st + (kTile8 + wm * 64 + 16 * i + r) * 128 + ((ch ^ (r & 7)) * 16));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mma8(a[i], b[j], acc[i][j]);
    }
  }
  // acc[i][j]: channels n0 + 64 wn + 16 i + 4 (lane / 16) + e of token m0 + 64 wm + 16 j + lane % 16
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = m0 + 64 * wm + 16 * j + (lane & 15);
    if (m >= p.M) continue;
    const float sx = p.sx[m];
    T* yr = reinterpret_cast<T*>(p.y) + int64_t(m) * p.y_sr;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + 64 * wn + 16 * i + 4 * (lane >> 4);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) yr[n + e] = E::from_f(float(acc[i][j][e]) * sx * p.sw[n + e]);
    }
  }
}

// ------------------------------------------------------------------------------------------------
template <typename T>
static void quantize(const void* x, int64_t x_sr, int M, int K, int8_t* q, float* scale, hipStream_t stream) {
  const bool wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (x_sr * int64_t(sizeof(T))) % 16 == 0;
  const dim3 grid(unsigned((int64_t(M) + kQuantWaves - 1) / kQuantWaves)), block(64 * kQuantWaves);
  hipLaunchKernelGGL(quantize_rows_kernel<T>, grid, block, 0, stream, reinterpret_cast<const T*>(x), x_sr, M, K,
                     int(padded_k8(K)), wide, q, scale);
}

int launch_quantize_rows(const mote_quantize_rows_args* a, hipStream_t stream) {
  const char* what = "quantize_rows";
  if (!a) return set_error(MOTE_ERR_ARGUMENT, "%s: null args", what);
  if (a->dtype != MOTE_F32 && a->dtype != MOTE_BF16) return set_error(MOTE_ERR_ARGUMENT, "%s: bad dtype %d", what, a->dtype);
  if (a->M < 0 || a->K <= 0 || a->K > kMaxK8) return set_error(MOTE_ERR_SHAPE, "%s: M = %d, K = %d (1 to %d)", what, a->M, a->K, kMaxK8);
  if (a->M == 0) return MOTE_OK;
  if (!a->x || !a->q || !a->scale) return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  if (a->M > 1 && a->x_sr < 0) return set_error(MOTE_ERR_ARGUMENT, "%s: negative row stride", what);
  if (reinterpret_cast<uintptr_t>(a->q) % 16) return set_error(MOTE_ERR_ARGUMENT, "%s: q must start on a 16-byte boundary", what);
  if (a->dtype == MOTE_BF16) quantize<bf16_t>(a->x, a->x_sr, a->M, a->K, a->q, a->scale, stream);
  else quantize<float>(a->x, a->x_sr, a->M, a->K, a->q, a->scale, stream);
  return check_launch(what);
}

static bool few8(const mote_int8_linear_args* a) { return a->M <= 16 && a->K <= kFewMaxK; }

size_t int8_linear_workspace_bytes(const mote_int8_linear_args* a) {
  if (a->M <= 0 || a->K <= 0 || few8(a)) return 0;
  return size_t(a->M) * padded_k8(a->K) + size_t(a->M) * sizeof(float);
}

template <typename T>
static void launch_few8(const mote_int8_linear_args* a, hipStream_t stream) {
  Few8Params p;
  p.x = a->x; p.x_sr = a->x_sr; p.w = a->wq; p.sw = a->w_scale; p.y = a->y; p.y_sr = a->y_sr;
  p.run = a->run; p.g = a->xm ? a->g : nullptr; p.xm = a->xm; p.heads = a->xm ? a->heads : 0;
  p.M = a->M; p.N = a->N; p.K = a->K; p.Kp = int(padded_k8(a->K));
  p.wide = reinterpret_cast<uintptr_t>(a->x) % 16 == 0 && (a->x_sr * int64_t(sizeof(T))) % 16 == 0;
  const int per = (p.Kp / 64 + kFewWaves - 1) / kFewWaves;
  const dim3 grid(unsigned((a->N + 15) / 16)), block(64 * kFewWaves);
  if (per <= 4) hipLaunchKernelGGL((int8_few_kernel<T, 4>), grid, block, 0, stream, p);
  else if (per <= 8) hipLaunchKernelGGL((int8_few_kernel<T, 8>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((int8_few_kernel<T, 16>), grid, block, 0, stream, p);
}

template <typename T>
static void launch_many8(const mote_int8_linear_args* a, hipStream_t stream) {
  const int Kp = int(padded_k8(a->K));
  int8_t* xq = reinterpret_cast<int8_t*>(a->workspace);
  float* sx = reinterpret_cast<float*>(xq + size_t(a->M) * Kp);
  quantize<T>(a->x, a->x_sr, a->M, a->K, xq, sx, stream);
  Many8Params p;
  p.x = xq; p.sx = sx; p.w = a->wq; p.sw = a->w_scale; p.y = a->y; p.y_sr = a->y_sr;
  p.M = a->M; p.N = a->N; p.Kp = Kp;
  p.ntok = (a->M + kTile8 - 1) / kTile8; p.nch = (a->N + kTile8 - 1) / kTile8;
  const unsigned per = unsigned((int64_t(p.ntok) * p.nch + 7) / 8);
  hipLaunchKernelGGL(int8_many_kernel<T>, dim3(8 * per), dim3(256), 0, stream, p);
}

int launch_int8_linear(const mote_int8_linear_args* a, hipStream_t stream) {
  const char* what = "int8_linear";
  if (!a) return set_error(MOTE_ERR_ARGUMENT, "%s: null args", what);
  if (a->dtype != MOTE_F32 && a->dtype != MOTE_BF16) return set_error(MOTE_ERR_ARGUMENT, "%s: bad dtype %d", what, a->dtype);
  if (a->M < 0 || a->N <= 0 || a->K <= 0 || a->K > kMaxK8)
    return set_error(MOTE_ERR_SHAPE, "%s: M = %d, N = %d, K = %d (K at most %d)", what, a->M, a->N, a->K, kMaxK8);
  if (int64_t((a->M + kTile8 - 1) / kTile8) * ((a->N + kTile8 - 1) / kTile8) >= (int64_t(1) << 30))
    return set_error(MOTE_ERR_SHAPE, "%s: too many tiles for one launch", what);
  if (a->M == 0) return MOTE_OK;
  if (!a->x || !a->wq || !a->w_scale || !a->y) return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  if (a->M > 1 && (a->x_sr < 0 || a->y_sr < a->N)) return set_error(MOTE_ERR_ARGUMENT, "%s: row strides shorter than the rows", what);
  if (reinterpret_cast<uintptr_t>(a->wq) % 16) return set_error(MOTE_ERR_ARGUMENT, "%s: wq must start on a 16-byte boundary", what);
  if (a->xm && (!a->g || a->heads <= 0)) return set_error(MOTE_ERR_ARGUMENT, "%s: xm needs g and heads > 0", what);
  if (few8(a)) {
    if (a->dtype == MOTE_BF16) launch_few8<bf16_t>(a, stream);
    else launch_few8<float>(a, stream);
    return check_launch(what);
  }
  if (a->run || a->xm) return set_error(MOTE_ERR_SHAPE, "%s: run and xm need at most 16 rows of K <= %d", what, kFewMaxK);
  const size_t need = int8_linear_workspace_bytes(a);
  if (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16)
    return set_error(MOTE_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes, %zu needed", what, a->workspace_bytes, need);
  if (a->dtype == MOTE_BF16) launch_many8<bf16_t>(a, stream);
  else launch_many8<float>(a, stream);
  return check_launch(what);
}

}  // namespace mote
