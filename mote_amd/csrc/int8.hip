// Products in 8-bit integers: y = x W^T with one fp32 scale per token of x and per output channel of W
// (mote_quantize_rows / mote_int8_linear; the rounding points stand in mote_relation.h).
//
// acc = sum_k xq wq runs on v_mfma_i32_16x16x64_i8, exact in 32 bits; y = (acc sx) sw in fp32, rounded once.
// One fragment convention for both operands: lane l holds 16 consecutive k of row l % 16, k group l / 16.
// Rows of xq and wq are Kp = K rounded up to 128 bytes, xq's zero past K, so no product looks at K.
#include <algorithm>

#include "tiles.hpp"
#include "params.hpp"
#include "device.hpp"
#include "stream.hpp"

namespace mote {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;

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
// Four codes in a word. rint(fl(x inv)) through the 1.5 * 2^23 that leaves no fraction bits in a float: after the
// addition (ties to even, as rint) the integer's two's complement is in the low bits, and v_perm takes its byte:
// under three instructions a value. A row without a scale (inv 0) may hold infinities and NaNs, whose codes
// are noise: its scale is NaN then, so every product with it is too, and quantize_rows stores zeros instead.
__device__ __forceinline__ uint32_t codes8(float a, float b, float c, float d, float inv) {
#pragma clang fp contract(off)
  constexpr float kMagic = 12582912.0f;
  const uint32_t ua = __float_as_uint(a * inv + kMagic), ub = __float_as_uint(b * inv + kMagic);
  const uint32_t uc = __float_as_uint(c * inv + kMagic), ud = __float_as_uint(d * inv + kMagic);
  const uint32_t lo = __builtin_amdgcn_perm(ub, ua, 0x0c0c0400u), hi = __builtin_amdgcn_perm(ud, uc, 0x0c0c0400u);
  return lo | hi << 16;
}

// N elements of a row of K from k on, as they lie in memory (zeros past its end), and as numbers
template <typename T, int N>
struct RowPart {
  static constexpr int EPC = 16 / int(sizeof(T)), NC = N / EPC;
  Chunk c[NC];
  __device__ __forceinline__ void load(const T* row, int k, int K) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int k0 = k + EPC * i;
      if (k0 + EPC <= K) {
        c[i] = load_any(row + k0);
      } else {
        T* e = reinterpret_cast<T*>(&c[i]);
#pragma unroll
        for (int j = 0; j < EPC; ++j) e[j] = k0 + j < K ? row[k0 + j] : T(0);
      }
    }
  }
  __device__ __forceinline__ void load_whole(const T* row, int k) {
#pragma unroll
    for (int i = 0; i < NC; ++i) c[i] = load_any(row + k + EPC * i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < NC; ++i) c[i] = zero_chunk();
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(c[j / 4].w[j % 4]);
    const uint32_t w = c[j / 8].w[j % 8 / 2];
    return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
  }
  // the bits of the largest magnitude
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 2) {
      u16x2 m = u16x2{0, 0};
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, c[i].w[j] & 0x7fff7fffu));
      return uint32_t(max(m.x, m.y)) << 16;
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) m = max(m, mag_bits(get(j)));
    return m;
  }
  // codes of elements 4 i .. 4 i + 3
  __device__ __forceinline__ uint32_t codes(int i, float inv) const {
    return codes8(get(4 * i), get(4 * i + 1), get(4 * i + 2), get(4 * i + 3), inv);
  }
};

// the maximum over the lanes li, li + 16, li + 32, li + 48 (row swaps, no LDS)
__device__ __forceinline__ uint32_t lanegroup_umax(uint32_t m) {
  u32x2 a = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  m = max(a[0], a[1]);
  a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  return max(a[0], a[1]);
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t m) {
  return max(m, uint32_t(__builtin_amdgcn_mov_dpp(int(m), CTRL, 0xF, 0xF, false)));
}
// the maximum over the G lanes of a row
template <int G>
__device__ __forceinline__ uint32_t group_umax(uint32_t m) {
  if constexpr (G == 64) {
    m = lanegroup_umax(m);
  } else if constexpr (G == 32) {
    const u32x2 a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = max(a[0], a[1]);
  }
  m = dpp_umax<kDppNext4>(dpp_umax<kDppRor8>(m));
  return dpp_umax<kDppXor1>(dpp_umax<kDppXor2>(m));
}

// ------------------------------------------------------------------------------------------------
// Rows in 8 bits: G lanes per row, the row in registers up to 8 G NC values (beyond, read twice)
// ------------------------------------------------------------------------------------------------
constexpr int kQuantWaves = 4;

template <typename T, int G, int NC>
__global__ void __launch_bounds__(64 * kQuantWaves)
quantize_rows_kernel(const T* x, int64_t x_sr, int M, int K, int Kp, int8_t* q, float* scale) {
  const int lane = threadIdx.x % G;
  const uint32_t m = blockIdx.x * (64 / G * kQuantWaves) + threadIdx.x / G;
  if (m >= uint32_t(M)) return;  // whole groups
  const T* row = x + int64_t(m) * x_sr;
  RowPart<T, 8> v[NC];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int k = (i * G + lane) * 8;
    if ((i + 1) * G * 8 <= K) v[i].load_whole(row, k);  // every lane's
    else if (k < Kp) v[i].load(row, k, K);
    else v[i].zero();
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) top = max(top, v[i].top());
  if constexpr (G == 64)
    for (int k = (NC * 64 + lane) * 8; k < Kp; k += 512) {
      RowPart<T, 8> w;
      w.load(row, k, K);
      top = max(top, w.top());
    }
  const Scale8 s = scale8(group_umax<G>(top));
  const uint32_t keep = s.inv == 0.f ? 0u : ~0u;  // a row without a scale stores zeros
  int8_t* out = q + int64_t(m) * Kp;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int k = (i * G + lane) * 8;
    if (k < Kp) *reinterpret_cast<uint2*>(out + k) = make_uint2(v[i].codes(0, s.inv) & keep, v[i].codes(1, s.inv) & keep);
  }
  if constexpr (G == 64)
    for (int k = (NC * 64 + lane) * 8; k < Kp; k += 512) {
      RowPart<T, 8> w;
      w.load(row, k, K);
      *reinterpret_cast<uint2*>(out + k) = make_uint2(w.codes(0, s.inv) & keep, w.codes(1, s.inv) & keep);
    }
  if (lane == 0) scale[m] = s.scale;
}

// ------------------------------------------------------------------------------------------------
// Few tokens: x is quantised where it is multiplied. One workgroup of NW waves per 16 channels and 16 tokens,
// the 64-wide k steps dealt to the waves in runs; a wave issues every load of its W rows and of its part of
// x, agrees on the rows' maxima with the other waves through LDS, and multiplies. The partial sums are
// integers: their order does not matter. Every workgroup of a token tile quantises it again (24 KB at 768
// from the L2), which costs less than a launch of its own. A launch of this size is bound by its latencies:
// 3.5 us at 1 x 768 -> 768, 3.6 us at 1 x 768 -> 2304, whose W of 1.8 MB takes 0.4.
// ------------------------------------------------------------------------------------------------
constexpr int kFewRows = 64;
constexpr int kFewMaxK = 4096;

struct Few8Params {
  const void* x; int64_t x_sr;
  const int8_t* w;
  const float* sw;
  void* y; int64_t y_sr;
  const unsigned char* run;
  const float* g; float* xm;
  int M, N, K, Kp, heads;
};

template <typename T, int NW, int KS>
__global__ void __launch_bounds__(64 * NW) int8_few_kernel(const Few8Params p) {
  using E = Elem<T>;
  __shared__ uint32_t tops[NW][16];
  __shared__ __align__(16) int part[NW][16][17];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // the steps' conditions are the wave's
  const int r = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
  const int nks = p.Kp / 64;                                 // k steps, an even number
  const int per = (nks + NW - 1) / NW;                       // <= KS
  const int s0 = min(wave * per, nks), s1 = min(s0 + per, nks);
  const int8_t* wrow = p.w + int64_t(min(n0 + r, p.N - 1)) * p.Kp + 16 * q;
  const T* xrow = reinterpret_cast<const T*>(p.x) + int64_t(min(m0 + r, p.M - 1)) * p.x_sr;
  Chunk a[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s)
    if (s0 + s < s1) a[s] = load_chunk(wrow + 64 * (s0 + s));
  RowPart<T, 16> x[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    if (64 * (s0 + s) + 64 <= min(p.K, 64 * s1)) x[s].load_whole(xrow, 64 * (s0 + s) + 16 * q);
    else if (s0 + s < s1) x[s].load(xrow, 64 * (s0 + s) + 16 * q, p.K);
  }
  float sw[4];  // of the channels that this lane stores (wave 0)
#pragma unroll
  for (int i = 0; i < 4; ++i) sw[i] = p.sw[min(n0 + 4 * q + i, p.N - 1)];
  // the decode step's exchange mass on the side: workgroup 0, wave 1, lane b < M
  const int xb = int(threadIdx.x) - 64;
  const bool xm_lane = p.xm != nullptr && blockIdx.x == 0 && m0 == 0 && xb >= 0 && xb < p.M;
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
  uint32_t top = 0;
#pragma unroll
  for (int s = 0; s < KS; ++s)
    if (s0 + s < s1) top = max(top, x[s].top());
  top = lanegroup_umax(top);
  if (q == 0) tops[wave][r] = top;
  __syncthreads();
  top = tops[0][r];
#pragma unroll
  for (int w = 1; w < NW; ++w) top = max(top, tops[w][r]);
  const Scale8 sc = scale8(top);
  i32x4 acc = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    if (s0 + s < s1) {
      Chunk b;
#pragma unroll
      for (int j = 0; j < 4; ++j) b.w[j] = x[s].codes(j, sc.inv);
      acc = mma8(a[s], b, acc);
    }
  }
  // acc: channels 4 q + i of token r
#pragma unroll
  for (int i = 0; i < 4; ++i) part[wave][4 * q + i][r] = acc[i];
  __syncthreads();
  if (wave == 0 && m0 + r < p.M) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int f = 4 * q + i;
      int v = part[0][f][r];
#pragma unroll
      for (int w = 1; w < NW; ++w) v += part[w][f][r];
      if (n0 + f < p.N)
        reinterpret_cast<T*>(p.y)[int64_t(m0 + r) * p.y_sr + n0 + f] = E::from_f(float(v) * sc.scale * sw[i]);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Many tokens: a tile of 16 FA WN channels x 16 FB WM tokens per workgroup of WN x WM waves.
//
// k goes in stages of 128 (a whole cache line of every row: half lines double the L2's requests, which
// bound 64-wide stages: 65536 x 1024 -> 4096 405 us and 384 us) through a ring of LDS stages filled by
// global_load_lds, the eight 16-byte chunks of row r swizzled by r % 8, so the rows that a quarter of a wave
// reads at once cover every bank. While a wave multiplies one half of a stage from registers it reads the
// fragments of the next half into a second set, so no product waits for the LDS, and one barrier a stage
// hands the slots over.
// What bounds the 256 x 256 tile (8192 x 4096 -> 4096: 112 us, 2.45 POP/s): matrix cores 56 % busy at the
// 1.9 GHz that the card runs them at; without its products it takes 90 us, without its loads and reads 90.
// Short k (1024: 8 stages) adds the stores, which all CUs make at once: a third of a tile's time.
// ------------------------------------------------------------------------------------------------
struct Many8Params {
  const int8_t* x;   // [M, Kp]
  const float* sx;
  const int8_t* w;   // [N, Kp]
  const float* sw;
  void* y; int64_t y_sr;
  int M, N, Kp, ntok, nch;
  int gch;           // channel tiles of a group: the tiles of a group are a run, token tile by token tile
  int stream;        // whether y passes the caches by
};

template <int FA, int FB, int WN, int WM, int RING_>
struct Tile8 {
  static constexpr int CH = 16 * FA * WN, TOK = 16 * FB * WM, NW = WN * WM;
  static constexpr int ROWS = CH + TOK;             // rows of a stage: channels, then tokens
  static constexpr int STAGE = 128 * ROWS;          // bytes
  static constexpr int PER = ROWS / 8 / NW;         // transfers of a wave per stage (8 rows each)
  static constexpr int RING = RING_;                // stages, a power of two
  static constexpr int OUTW = 16 * FA + 8;          // a row of a wave's output tile in LDS (padded, in elements)
  static_assert(ROWS % (8 * NW) == 0, "every wave issues as many transfers");
};

// the wave's LDS reads are done, at most N of its transfers are outstanding, and every wave is here (the
// waits as builtins: the compiler then knows that the fragments have arrived)
template <int N>
__device__ __forceinline__ void arrive() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(kVmWaitStage<N>() & ~(0xF << 8));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename T, int FA, int FB, int WN, int WM, int RING>
__global__ void __launch_bounds__(64 * WN * WM) __attribute__((amdgpu_waves_per_eu(2)))
int8_many_kernel(const Many8Params p) {
  using E = Elem<T>;
  using S = Tile8<FA, FB, WN, WM, RING>;
  constexpr int kOut = S::NW * 16 * S::OUTW * int(sizeof(T));  // 16 tokens of every wave's tile at a time
  __shared__ __align__(16) int8_t smem[S::RING * S::STAGE > kOut ? S::RING * S::STAGE : kOut];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // workgroups go round-robin over the 8 XCDs: XCD j takes the j-th run of (token tile, channel tile)
  const int nwg = p.ntok * p.nch, per = (nwg + 7) / 8;
  const int seq = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (seq >= nwg) return;
  const int g = seq / (p.ntok * p.gch), in_g = seq - g * p.ntok * p.gch;
  const int gw = min(p.gch, p.nch - g * p.gch);  // channel tiles of this group (fewer in the last)
  const int m0 = in_g / gw * S::TOK, n0 = (g * p.gch + in_g % gw) * S::CH;

  const int8_t* wb = p.w + int64_t(n0) * p.Kp;
  const int8_t* xb = p.x + int64_t(m0) * p.Kp;
  uint32_t voff[S::PER];
#pragma unroll
  for (int i = 0; i < S::PER; ++i) {
    const int row = (wave * S::PER + i) * 8 + (lane >> 3);
    const int r = row < S::CH ? min(row, p.N - 1 - n0) : min(row - S::CH, p.M - 1 - m0);
    voff[i] = uint32_t(r) * uint32_t(p.Kp) + 16u * ((lane & 7) ^ (row & 7));
  }
  const uint32_t ring = lds_addr(smem);
  auto issue = [&](int kb, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < S::PER; ++i) {
      const int g = wave * S::PER + i;
      lds_dma16_sa((g < S::CH / 8 ? wb : xb) + 128 * kb, voff[i],
                   ring + uint32_t(slot * S::STAGE + g * 1024));
    }
  };

  const int wn = wave % WN, wm = wave / WN;
  const int r = lane & 15, q = lane >> 4;
  const int foff[2] = {r * 128 + 16 * (q ^ (r & 7)), r * 128 + 16 * ((q + 4) ^ (r & 7))};
  const int8_t* fa = smem + wn * FA * 2048;
  const int8_t* fb = smem + (S::CH / 16 + wm * FB) * 2048;
  struct Frags {
    Chunk a[FA], b[FB];
  };
  i32x4 acc[FA][FB];
#pragma unroll
  for (int i = 0; i < FA; ++i)
#pragma unroll
    for (int j = 0; j < FB; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  const int nk = p.Kp / 128;
  constexpr int RPG = (2 * FA + FB - 1) / FA;  // reads between FB products: FA + FB in FA groups
  Frags f0, f1;
  // the products of one half stage, the reads of the next half between them
  auto half = [&](const Frags& cur, Frags& next, int slot, int hf) __attribute__((always_inline)) {
    const int st = slot * S::STAGE + foff[hf];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < FA; ++i) {
#pragma unroll
      for (int k = RPG * i; k < RPG * i + RPG; ++k) {
        if (k < FB) next.b[k] = load_chunk(fb + st + k * 2048);
        else if (k < FA + FB) next.a[k - FB] = load_chunk(fa + st + (k - FB) * 2048);
      }
#pragma unroll
      for (int j = 0; j < FB; ++j) acc[i][j] = mma8(cur.a[i], cur.b[j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int s = 0; s < S::RING; ++s)
    if (s < nk) issue(s, s);
  if (nk >= S::RING) arrive<(S::RING - 1) * S::PER>();
  else arrive<0>();
#pragma unroll
  for (int i = 0; i < FB; ++i) f0.b[i] = load_chunk(fb + foff[0] + i * 2048);
#pragma unroll
  for (int i = 0; i < FA; ++i) f0.a[i] = load_chunk(fa + foff[0] + i * 2048);
  // Stage kb in slot kb % RING: its second half is read while the first is multiplied; then stage kb + 1 has
  // arrived (at most RING - 2 younger ones are outstanding) and every wave holds the whole of stage kb in
  // registers, so its slot takes stage kb + RING, and the first half of kb + 1 is read while the second of
  // kb is multiplied. The last stages issue nothing; the very last reads a slot for nothing (no condition in
  // the loop: at a join the compiler would wait for the reads before the products that do not need them).
  int kb = 0;
  for (; kb + S::RING < nk; ++kb) {
    half(f0, f1, kb & (S::RING - 1), 1);
    arrive<(S::RING - 2) * S::PER>();
    issue(kb + S::RING, kb & (S::RING - 1));
    half(f1, f0, (kb + 1) & (S::RING - 1), 0);
  }
  for (; kb < nk; ++kb) {
    half(f0, f1, kb & (S::RING - 1), 1);
    arrive<0>();
    half(f1, f0, (kb + 1) & (S::RING - 1), 0);
  }

  // acc[i][j]: channels n0 + 16 (wn FA + i) + 4 q + e of token m0 + 16 (wm FB + j) + r. Sixteen tokens at a
  // time go through LDS (each wave its own part), so that a store instruction writes whole rows; y passes
  // the caches by (65536 x 1024 -> 4096 381 -> 317 us, 4096 x 4096 -> 1024 34.7 -> 33.4 us, small y as before).
  lds_barrier();  // the ring is no longer read
  T* tile = reinterpret_cast<T*>(smem) + wave * 16 * S::OUTW;
  const int nw0 = n0 + wn * 16 * FA;
  float sw[FA][4];
#pragma unroll
  for (int i = 0; i < FA; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) sw[i][e] = p.sw[min(nw0 + 16 * i + 4 * q + e, p.N - 1)];
  constexpr int EPC = 16 / int(sizeof(T));      // elements of a 16-byte store
  constexpr int CPR = 16 * FA / EPC;            // stores of a row
#pragma unroll
  for (int j = 0; j < FB; ++j) {
    const int mt = m0 + 16 * (wm * FB + j);
    const float sx = p.sx[min(mt + r, p.M - 1)];
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = float(acc[i][j][e]) * sx * sw[i][e];
      T* d = tile + r * S::OUTW + 16 * i + 4 * q;
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint2*>(d) = make_uint2(uint32_t(f2bf(v[0])) | uint32_t(f2bf(v[1])) << 16,
                                                  uint32_t(f2bf(v[2])) | uint32_t(f2bf(v[3])) << 16);
      } else {
        *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    // the wave's own writes, read back by the wave: LDS operations of a wave complete in order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int c = lane; c < 16 * CPR; c += 64) {
      const int row = c / CPR, col = c % CPR * EPC;
      const int m = mt + row, n = nw0 + col;
      if (m >= p.M || n >= p.N) continue;
      T* yr = reinterpret_cast<T*>(p.y) + int64_t(m) * p.y_sr + n;
      const T* src = tile + row * S::OUTW + col;
      if (n + EPC <= p.N) {
        if (p.stream) {
          // between two of these, so that the compiler does not make one store of the two, without the hint
          asm volatile("" ::: "memory");
          store_stream_any(yr, load_chunk(src));
          asm volatile("" ::: "memory");
        } else {
          store_any(yr, load_chunk(src));
        }
      } else {
        for (int e = 0; e < EPC && n + e < p.N; ++e) yr[e] = src[e];
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// ------------------------------------------------------------------------------------------------
constexpr int kQuantMost = 1 << 25;  // rows of a launch: up to 64 threads each, and a grid holds fewer than 2^32

template <typename T>
static int quantize(const void* x, int64_t x_sr, int M, int K, int8_t* q, float* scale, hipStream_t stream, const char* what) {
  const int Kp = int(padded_k8(K));
  auto go = [&](auto kernel, int lanes) {
    const int rows = 64 / lanes * kQuantWaves;
    for (int64_t m0 = 0; m0 < M; m0 += kQuantMost) {
      const int part = int(std::min<int64_t>(M - m0, kQuantMost));
      hipLaunchKernelGGL(kernel, dim3(unsigned((part + rows - 1) / rows)), dim3(64 * kQuantWaves), 0, stream,
                         reinterpret_cast<const T*>(x) + m0 * x_sr, x_sr, part, K, Kp, q + m0 * Kp, scale + m0);
    }
    return check_launch(what);
  };
  // A row's share of a wave is as wide as the row needs, so that no lane idles and a row stays in registers:
  // 35304 x 64 11.2 -> 4.7 us and 16384 x 768 9.7 -> 8.1 us against a wave per row; 19417 x 3776 48 -> 37.6 us
  // against half of the row read twice. 65536 x 1024 takes 32.3 us either way.
  if (Kp <= 128) return go(quantize_rows_kernel<T, 16, 1>, 16);
  if (Kp <= 256) return go(quantize_rows_kernel<T, 16, 2>, 16);
  if (Kp <= 384) return go(quantize_rows_kernel<T, 16, 3>, 16);
  if (Kp <= 512) return go(quantize_rows_kernel<T, 32, 2>, 32);
  if (Kp <= 768) return go(quantize_rows_kernel<T, 32, 3>, 32);
  if (Kp <= 1024) return go(quantize_rows_kernel<T, 32, 4>, 32);
  if (Kp <= 2048) return go(quantize_rows_kernel<T, 64, 4>, 64);
  return go(quantize_rows_kernel<T, 64, 8>, 64);
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
  return a->dtype == MOTE_BF16 ? quantize<bf16_t>(a->x, a->x_sr, a->M, a->K, a->q, a->scale, stream, what)
                               : quantize<float>(a->x, a->x_sr, a->M, a->K, a->q, a->scale, stream, what);
}

// The one-launch form: for up to 16 tokens (16 x 768 -> 768 4.8 us, 6.4 with quantize_rows and tiles; 16 x
// 4096 -> 4096 10.4 and 11.4), and up to 64 while the workgroups that quantise a token again are few: two a CU
// of K up to 1024 (64 x 1024 -> 1536, 384 of them, 6.4 and 6.8 us; 64 x 768 -> 2304, 576, 6.5 and 6.5), one up to
// 2048 (32 x 2048 -> 2048, 256, 7.0 and 7.7; 48 x 1536 -> 1536, 288, 8.1 and 7.2), none beyond (32 x 4096 -> 1024
// 9.4 and 9.2, fp32 12.6 and 9.2); the predicate and the exchange mass exist in it alone, so calls with them take it at
// every size (64 x 4096 -> 4096 26.0 us, 10.0 with tiles).
static bool few8(const mote_int8_linear_args* a) {
  if (a->M > kFewRows || a->K > kFewMaxK) return false;
  const int64_t groups = (int64_t(a->M) + 15) / 16 * ((int64_t(a->N) + 15) / 16);
  return a->M <= 16 || a->run || a->xm || groups <= int64_t(a->K <= 1024 ? 2 : a->K <= 2048 ? 1 : 0) * device_cu_count();
}

size_t int8_linear_workspace_bytes(const mote_int8_linear_args* a) {
  if (a->M <= 0 || a->K <= 0 || few8(a)) return 0;
  return size_t(a->M) * padded_k8(a->K) + size_t(a->M) * sizeof(float);
}

template <typename T>
static int launch_few8(const mote_int8_linear_args* a, hipStream_t stream, const char* what) {
  Few8Params p;
  p.x = a->x; p.x_sr = a->x_sr; p.w = a->wq; p.sw = a->w_scale; p.y = a->y; p.y_sr = a->y_sr;
  p.run = a->run; p.g = a->xm ? a->g : nullptr; p.xm = a->xm; p.heads = a->xm ? a->heads : 0;
  p.M = a->M; p.N = a->N; p.K = a->K; p.Kp = int(padded_k8(a->K));
  auto go = [&](auto kernel, int waves) {
    const dim3 grid(unsigned((a->N + 15) / 16), unsigned((a->M + 15) / 16));
    if (!grid_fits(grid.x, 64 * waves)) return set_error(MOTE_ERR_SHAPE, "%s: N = %d is too many channels for one launch", what, a->N);
    hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, stream, p);
    return check_launch(what);
  };
  // Beyond K = 1024 eight waves (16 x 4096 -> 4096 11.4 -> 10.4 us, 1 x 2048 -> 2048 5.5 -> 5.2), four up to there
  // (16 x 768 -> 2304 4.7 us, 4.9 with eight).
  if (p.Kp <= 1024) return go(int8_few_kernel<T, 4, 4>, 4);
  if (p.Kp <= 2048) return go(int8_few_kernel<T, 8, 4>, 8);
  return go(int8_few_kernel<T, 8, 8>, 8);
}

template <typename T>
static int launch_many8(const mote_int8_linear_args* a, hipStream_t stream, const char* what) {
  const int Kp = int(padded_k8(a->K));
  int8_t* xq = reinterpret_cast<int8_t*>(a->workspace);
  float* sx = reinterpret_cast<float*>(xq + size_t(a->M) * Kp);
  Many8Params p;
  p.x = xq; p.sx = sx; p.w = a->wq; p.sw = a->w_scale; p.y = a->y; p.y_sr = a->y_sr;
  p.M = a->M; p.N = a->N; p.Kp = Kp;
  // y passes the caches by, except where it is larger than the L2s and its rows share cache lines: those
  // would go out in parts (30000 x 768 -> 1032 63 us, 57 through the L2s; 1056 channels 54 and 56 us)
  const bool whole = reinterpret_cast<uintptr_t>(a->y) % 64 == 0 && (a->y_sr * int64_t(sizeof(T))) % 64 == 0;
  p.stream = whole || double(a->M) * a->N * sizeof(T) < double(32 << 20);
  auto go = [&](auto kernel, int ch, int tok, int waves) {
    p.ntok = (a->M + tok - 1) / tok; p.nch = (a->N + ch - 1) / ch;
    // A weight that an XCD's 4 MB L2 holds stays there whatever the order; a larger one goes in groups of
    // up to eight channel tiles, each over all tokens (W of 4 MB: 65536 x 1024 -> 4096 392 -> 379 us, 8192
    // rows 53 -> 51 us; of 1.8 MB: 4964 x 768 -> 2304 24 us in one group, 26 us in three).
    const int groups = int64_t(a->N) * Kp <= (5 << 19) ? 1 : (p.nch + 7) / 8;
    p.gch = (p.nch + groups - 1) / groups;
    const int64_t grid = (int64_t(p.ntok) * p.nch + 7) / 8 * 8;
    if (!grid_fits(grid, 64 * waves)) return set_error(MOTE_ERR_SHAPE, "%s: M = %d, N = %d are too many tiles for one launch", what, a->M, a->N);
    if (const int rc = quantize<T>(a->x, a->x_sr, a->M, a->K, xq, sx, stream, what)) return rc;
    hipLaunchKernelGGL(kernel, dim3(unsigned(grid)), dim3(64 * waves), 0, stream, p);
    return check_launch(what);
  };
  // Tiles of channels x tokens. One round of workgroups of a small tile while that holds everything. Transfers into
  // LDS reach some 47 bytes a nanosecond per CU, so few tiles go to as many CUs as there are: 32 x 16 (258 x 3413
  // -> 523 10.6 us, 11.9 with 64 x 32; 128 x 768 -> 768 6.4 and 6.8; past two a CU 1000 x 520 -> 271 7.5 and 7.2).
  // Then 64 x 32, up to three a CU (512 x 768 -> 2304 8.5 us, 11.1 with 128 x 128), or two where k is long and one
  // of 128 x 64 a CU does, with fewer bytes a product and a ring of four (600 x 2048 -> 2048 12.2, 12.8 with 64 x
  // 32; 700 x 1024 -> 1600 9.4 and 9.2); that one (512 x 4096 -> 4096 19.5 us, 25.2 with a ring of two, 24.5 with
  // 64 x 32; 2048 x 1024 -> 1024 10.1, 11.2 and 11.6); one of 128 x 128 a CU with a ring of four where k is long
  // (4096 x 4096 -> 1024 31.0, 33.3 with the next; 2000 x 300 -> 2048 9.7 and 9.4); then 128 x 64 with a ring of
  // two, three a CU (2048 x 768 -> 2304 12.8, 13.0 with 128 x 128, 16.3 with 64 x 32).
  const int64_t cus = device_cu_count();
  auto tiles = [&](int ch, int tok) { return ((int64_t(a->M) + tok - 1) / tok) * ((a->N + ch - 1) / ch); };
  if (tiles(32, 16) <= 2 * cus) return go(int8_many_kernel<T, 1, 1, 2, 1, 4>, 32, 16, 2);
  const bool one_each = tiles(128, 64) <= cus;
  if (tiles(64, 32) <= (one_each && Kp > 1024 ? 2 : 3) * cus) return go(int8_many_kernel<T, 2, 1, 2, 2, 4>, 64, 32, 4);
  if (one_each) return go(int8_many_kernel<T, 2, 2, 4, 2, 4>, 128, 64, 8);
  if (tiles(128, 128) <= cus && Kp >= 1024) return go(int8_many_kernel<T, 4, 2, 2, 4, 4>, 128, 128, 8);
  if (tiles(128, 64) <= 3 * cus) return go(int8_many_kernel<T, 4, 2, 2, 2, 2>, 128, 64, 4);
  // Beyond, the tile whose rounds take least: a round of n stages of k takes fixed + n * stage us (fitted to
  // k = 768, 1024 and 4096 at 4964 to 65536 rows), with one workgroup per CU of the large tiles and two of
  // 128 x 128. 4964 x 768 -> 2304: 234 tiles of 256 x 192 in one round 20.9 us, 23.2 with 256 x 256 or 128 x
  // 128; 16384 rows: 768 tiles of 192 x 256 in three 52.8 us, 57.7 and 57.1; 65536 x 1024 -> 4096: 256 x 256
  // 328 us, 353 with 256 x 192, 366 with 128 x 128. The costs are those of bf16 results; fp32 ones store twice the
  // bytes and take the same rule (23.8, 60.2 and 391 us at these sizes, x quantised included; bf16 18.6, 46.6, 325),
  // their other tiles not measured.
  auto rounds_us = [&](int64_t t, int64_t slots, double fixed, double stage) {
    return double((t + slots - 1) / slots) * (fixed + Kp / 128 * stage);
  };
  const double big = rounds_us(tiles(256, 256), cus, 7.3, 1.5), wide = rounds_us(tiles(256, 192), cus, 5.6, 1.15),
               tall = rounds_us(tiles(192, 256), cus, 5.6, 1.15), mid = rounds_us(tiles(128, 128), 2 * cus, 3.5, 0.94);
  const double best = std::min(std::min(big, wide), std::min(tall, mid));
  if (big == best) return go(int8_many_kernel<T, 8, 4, 2, 4, 2>, 256, 256, 8);
  if (wide == best) return go(int8_many_kernel<T, 8, 3, 2, 4, 2>, 256, 192, 8);
  if (tall == best) return go(int8_many_kernel<T, 6, 4, 2, 4, 2>, 192, 256, 8);
  return go(int8_many_kernel<T, 4, 4, 2, 2, 2>, 128, 128, 4);
}

int launch_int8_linear(const mote_int8_linear_args* a, hipStream_t stream) {
  const char* what = "int8_linear";
  if (!a) return set_error(MOTE_ERR_ARGUMENT, "%s: null args", what);
  if (a->dtype != MOTE_F32 && a->dtype != MOTE_BF16) return set_error(MOTE_ERR_ARGUMENT, "%s: bad dtype %d", what, a->dtype);
  if (a->M < 0 || a->M > (1 << 30) || a->N <= 0 || a->N > (1 << 30) || a->K <= 0 || a->K > kMaxK8)
    return set_error(MOTE_ERR_SHAPE, "%s: M = %d, N = %d (at most 2^30), K = %d (at most %d)", what, a->M, a->N, a->K, kMaxK8);
  if (((int64_t(a->M) + 127) / 128) * ((int64_t(a->N) + 127) / 128) >= (int64_t(1) << 30))
    return set_error(MOTE_ERR_SHAPE, "%s: too many tiles for one launch", what);
  if (a->M == 0) return MOTE_OK;
  if (!a->x || !a->wq || !a->w_scale || !a->y) return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  if (a->M > 1 && (a->x_sr < 0 || a->y_sr < a->N)) return set_error(MOTE_ERR_ARGUMENT, "%s: row strides shorter than the rows", what);
  if (reinterpret_cast<uintptr_t>(a->wq) % 16) return set_error(MOTE_ERR_ARGUMENT, "%s: wq must start on a 16-byte boundary", what);
  if (a->xm && (!a->g || a->heads <= 0)) return set_error(MOTE_ERR_ARGUMENT, "%s: xm needs g and heads > 0", what);
  if (few8(a)) return a->dtype == MOTE_BF16 ? launch_few8<bf16_t>(a, stream, what) : launch_few8<float>(a, stream, what);
  if (a->run || a->xm) return set_error(MOTE_ERR_SHAPE, "%s: run and xm need at most %d rows of K <= %d", what, kFewRows, kFewMaxK);
  const size_t need = int8_linear_workspace_bytes(a);
  if (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16)
    return set_error(MOTE_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes, %zu needed", what, a->workspace_bytes, need);
  return a->dtype == MOTE_BF16 ? launch_many8<bf16_t>(a, stream, what) : launch_many8<float>(a, stream, what);
}

}  // namespace mote
