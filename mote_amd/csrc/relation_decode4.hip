// One decode step of one Relation layer over the cache in 4 bits, one launch: the step of
// relation_decode.hip (RoPE / Givens / append / softmax read, split-S sweep with an in-kernel merge)
// with past rows decoded in registers as they arrive.
//
// Per past row j: U_j = sum_groups s_jg <q_g, c_jg> / sqrt(D), e_j = SiLU(U_j), running max m and sum l,
// z += exp(e_j - m) s_jg c_jg. A row is 18 G bytes of P2 and of I~ against 64 G in bf16, so a sweep is bound
// by memory as there, at 3.6 times fewer bytes, with the conversions close behind: a lane holds one group of
// a row (16 bytes of codes, one load), one to four lanes a row, so a group's scale is applied once per group
// and not per value: to the finished partial product on the P2 side, to the weight on the I~ side. For bf16
// queries the codes become bf16 pairs (exact) for v_dot2_f32_bf16; the weighted sums stay in fp32.
// Three groups (head dim 96) take three lanes, 21 rows a wave step and one idle lane; with a fourth lane that
// repeated the last group the step took 9.5 us at batch 1 and 20.7 at batch 16, now 8.5 and 17.2.
//
// Measured (the step alone in a graph): 453 MB of rows 90 us (5.0 TB/s; a copy reaches 5.2), 49 MB 16.1 us,
// 3.5 MB (batch 1, S 4096) 8.5 us, an almost empty cache 5.5 us: launch, one round of loads, the new rows,
// and, where a head has several splits, three trips to the device-coherent level for the merge. fp32 rows cost the
// same (16 x 4096 rows of 8 x 96: 16.0 us, bf16 15.5; 16 x 32768 of 8 x 128, 604 MB: 103 us, 5.8 TB/s, in both).
//
// Grid, rings, splits, predicate and the publish / count / merge protocol are those of relation_decode.hip;
// its comments give the reasons.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "params.hpp"
#include "device.hpp"
#include "fp4.hpp"

namespace mote {

struct Dec4Params {
  const float* lam;
  const float* inv_freq;  // never null: without RoPE / Givens the launcher points both at lam
  const float* theta;
  int rope, givens;
  int64_t* S;
  const void* p1;
  const void* p2;
  const void* info;
  int64_t in_sb;
  uint8_t* kc;
  uint8_t* vc;
  bf16_t* ks;
  bf16_t* vs;
  int64_t c_sb, c_sh, s_sb, s_sh;
  void* y;
  int64_t y_sb;
  float* g;
  float* xm;
  const unsigned char* run;
  float* part;  // [BH][nsplit][D + 2]  (max, l, z)
  int* cnt;
  int* cnt_seq;
  int B, H, D, cap, parity, flags, nsplit;
  float scale, tau_inv;
};

constexpr int kD4MaxSplits = 64;
constexpr int kD4Waves = 4;
constexpr int kD4Threads = 64 * kD4Waves;
constexpr int kD4CntStride = 64;  // ints between two completion counters: 256 bytes

__device__ __forceinline__ void put_coherent(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get_coherent(const float* p) {
  return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// <q, codes> over a group of 32, and z += w codes
template <typename T>
struct Query4;
template <>
struct Query4<bf16_t> {
  bf16x2 v[16];
  __device__ __forceinline__ void set(const float* q) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = bf16x2{(__bf16)q[2 * j], (__bf16)q[2 * j + 1]};
  }
  __device__ __forceinline__ float dot(const Chunk& c) const {
    float a = 0.f, b = 0.f;  // two independent chains
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a = __builtin_amdgcn_fdot2_f32_bf16(codes_bf16<0>(c.w[k]), v[4 * k], a, false);
      b = __builtin_amdgcn_fdot2_f32_bf16(codes_bf16<1>(c.w[k]), v[4 * k + 1], b, false);
      a = __builtin_amdgcn_fdot2_f32_bf16(codes_bf16<2>(c.w[k]), v[4 * k + 2], a, false);
      b = __builtin_amdgcn_fdot2_f32_bf16(codes_bf16<3>(c.w[k]), v[4 * k + 3], b, false);
    }
    return a + b;
  }
};
template <>
struct Query4<float> {
  float v[32];
  __device__ __forceinline__ void set(const float* q) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = q[j];
  }
  __device__ __forceinline__ float dot(const Chunk& c) const {
    float a = 0.f, b = 0.f;
    auto two = [&](f32x2 x, int j) {
      a = fmaf(x.x, v[j], a);
      b = fmaf(x.y, v[j + 1], b);
    };
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      two(codes_f32<0>(c.w[k]), 8 * k);
      two(codes_f32<1>(c.w[k]), 8 * k + 2);
      two(codes_f32<2>(c.w[k]), 8 * k + 4);
      two(codes_f32<3>(c.w[k]), 8 * k + 6);
    }
    return a + b;
  }
};
__device__ __forceinline__ void add4(float (&z)[32], const Chunk& c, float w) {
  auto two = [&](f32x2 x, int j) {
    z[j] = fmaf(w, x.x, z[j]);
    z[j + 1] = fmaf(w, x.y, z[j + 1]);
  };
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    two(codes_f32<0>(c.w[k]), 8 * k);
    two(codes_f32<1>(c.w[k]), 8 * k + 2);
    two(codes_f32<2>(c.w[k]), 8 * k + 4);
    two(codes_f32<3>(c.w[k]), 8 * k + 6);
  }
}

// the sum of a row's LPR neighbouring lanes, in each of them (c: the lane's place among them); three lanes
// lie across the rows of 16 that DPP works in, so they take its whole-wave shifts
template <int LPR>
__device__ __forceinline__ float row_sum(float x, int c) {
  if constexpr (LPR == 2 || LPR == 4) x += dpp<kDppXor1>(x);
  if constexpr (LPR == 4) x += dpp<kDppXor2>(x);
  if constexpr (LPR == 3) {
    constexpr int kNext = 0x130, kPrev = 0x138;  // wave_shl:1 reads lane + 1, wave_shr:1 lane - 1
    const float x1 = dpp<kNext>(x), x2 = dpp<kNext>(x1);
    const float s = (x + x1) + x2;  // the row's, in its first lane
    const float s1 = dpp<kPrev>(s), s2 = dpp<kPrev>(s1);
    x = c == 0 ? s : c == 1 ? s1 : s2;
  }
  return x;
}

template <typename T, int G, bool STREAM>
__global__ void __launch_bounds__(kD4Threads) relation_decode4_kernel(const Dec4Params p) {
  using E = Elem<T>;
  constexpr int LPR = G;                          // lanes of a row, one per group
  constexpr int RPW = 64 / LPR;                   // rows of a wave's step (three groups: lane 63 has none)
  constexpr int ROWS = RPW * kD4Waves;            // rows of a step
  constexpr int DP = 32 * G, ZS = DP + 4;         // a row group's z in LDS (16-byte aligned)
  constexpr int CL = 32 * LPR, PARTS = kD4Threads / CL;  // column sums: PARTS threads a column
  static_assert(ROWS * ZS >= kD4MaxSplits * (DP + 2), "the partials of a head fit the table of row groups");
  __shared__ __align__(16) float zred[ROWS * ZS];
  __shared__ __align__(16) float sq[DP], knew[128], inew[128];
  __shared__ float csum[PARTS][CL];
  __shared__ float sm[kD4Waves], sl[kD4Waves];
  __shared__ float wsp[kD4MaxSplits];
  __shared__ float sML[3];
  __shared__ int s_last;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int BH = p.B * p.H;
  const int bh = blockIdx.x % BH;
  const int split = blockIdx.x / BH;
  const int b = bh / p.H, h = bh % p.H;
  const int D = p.D, half = D / 2;
  const int nsp = p.nsplit;
  const int c = lane % LPR;                   // this lane's group
  const bool act = lane < RPW * LPR;
  const int rr = min(lane / LPR, RPW - 1);
  const int roff = wave * RPW + rr;           // its row within a step
  const uint8_t* kbase = p.kc + b * p.c_sb + h * p.c_sh + 16 * c;
  const uint8_t* vbase = p.vc + b * p.c_sb + h * p.c_sh + 16 * c;
  const bf16_t* ksb = p.ks + b * p.s_sb + h * p.s_sh + c;
  const bf16_t* vsb = p.vs + b * p.s_sb + h * p.s_sh + c;

  // the small loads first: they complete in order, ahead of the cache rows issued after them
  int vzero;
  asm volatile("v_mov_b32 %0, 0" : "=v"(vzero));
  const float lam = p.lam[vzero];
  const int64_t S64 = p.S[b + vzero];
  const int run_v = (p.run ? p.run : reinterpret_cast<const unsigned char*>(p.lam))[vzero];
  const int odd = h & 1, par = p.parity;
  const bool first = (odd ^ par) == 0;
  int nb = h + 2 * odd - 1;  // odd layers pair h with h + 1 for odd h, h - 1 for even h, modulo H
  nb += int(nb < 0) * p.H - int(nb >= p.H) * p.H;
  const int other = (h ^ 1) + par * (nb - (h ^ 1));
  const int pair = (h >> 1) + (par & (odd ^ 1)) * ((other >> 1) - (h >> 1));
  const float th = p.theta[(p.givens ? pair : 0) + vzero];
  const int qi = min(tid, half - 1);
  const int di = min(tid & 127, D - 1);
  const T* in_b = reinterpret_cast<const T*>(p.p1) + b * p.in_sb + h * D;
  const float q0 = E::to_f(in_b[qi]), q1 = E::to_f(in_b[qi + half]);
  const T* kn_b = reinterpret_cast<const T*>(p.p2) + b * p.in_sb + h * D;
  const float k0 = E::to_f(kn_b[qi]), k1 = E::to_f(kn_b[qi + half]);
  const T* i_raw = reinterpret_cast<const T*>(p.info) + b * p.in_sb;
  const float iself = E::to_f(i_raw[h * D + di]), ioth = E::to_f(i_raw[other * D + di]);
  const float invf = p.inv_freq[p.rope ? qi : 0];

  // a ring of four register sets; rows are clamped to rlim (the cache's last row until S is known)
  Chunk kr[4], vr[4];
  bf16_t ksr[4], vsr[4];
  int rlim = p.cap - 1;
  auto fetch = [&](int j, auto u) {
    constexpr int U = decltype(u)::value;
    const int64_t rc = min((split + j * nsp) * ROWS + roff, rlim);
    kr[U] = load_chunk_as<STREAM>(kbase + rc * (16 * G));
    ksr[U] = ksb[rc * G];
    vr[U] = load_chunk_as<STREAM>(vbase + rc * (16 * G));
    vsr[U] = vsb[rc * G];
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  fetch(0, I0{});
  fetch(1, I1{});
  fetch(2, I2{});
  asm volatile("" ::: "memory");  // keeps the predicate's test (an early exit) after the cache loads

  if (p.run && run_v == 0) return;  // the predicate: every workgroup leaves before any write or count
  const bool bad = S64 < 0 || S64 >= p.cap;
  const int S = bad ? 0 : int(S64);

  float cs, sn;
  sincosf((float)S * invf, &sn, &cs);
  const bool rope32 = (p.flags & MOTE_DECODE_ROPE_F32) != 0;
  const float cs32 = p.rope ? cs : 1.f, sn32 = p.rope ? sn : 0.f;
  cs = p.rope ? round_elem<T>(cs) : 1.f;
  sn = p.rope ? round_elem<T>(sn) : 0.f;
  const float rq0 = rope32 ? round_elem<T>(rot_round<float>(q0, cs32, q1, -sn32)) : rot_round<T>(q0, cs, q1, -sn);
  const float rq1 = rope32 ? round_elem<T>(rot_round<float>(q1, cs32, q0, sn32)) : rot_round<T>(q1, cs, q0, sn);
  const float rk0 = rope32 ? round_elem<T>(rot_round<float>(k0, cs32, k1, -sn32)) : rot_round<T>(k0, cs, k1, -sn);
  const float rk1 = rope32 ? round_elem<T>(rot_round<float>(k1, cs32, k0, sn32)) : rot_round<T>(k1, cs, k0, sn);
  float gc, gs;
  sincosf(th, &gs, &gc);
  gc = p.givens ? round_elem<T>(gc) : 1.f;
  gs = p.givens ? round_elem<T>(gs) : 0.f;
  const float rin = p.givens ? rot_round<T>(iself, gc, ioth, first ? -gs : gs) : iself;
  if (tid < half) {
    sq[tid] = rq0;
    sq[tid + half] = rq1;
    knew[tid] = rk0;
    knew[tid + half] = rk1;
  } else if (tid >= 128 && tid < 128 + D) {
    inew[tid - 128] = rin;
  }
  for (int d = D + tid; d < 128; d += kD4Threads) {  // a group past the head dim holds zeros
    if (d < DP) sq[d] = 0.f;
    knew[d] = 0.f;
    inew[d] = 0.f;
  }
  __syncthreads();

  // this split's steps: s + j nsplit for j < ns, rows below S
  const int nst = (S + ROWS - 1) / ROWS;
  const int ns = nst > split ? (nst - split + nsp - 1) / nsp : 0;
  rlim = ns > 0 ? min((split + (ns - 1) * nsp) * ROWS + ROWS, S) - 1 : 0;

  Query4<T> q;
  {
    float qf[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) qf[j] = sq[32 * c + j];
    q.set(qf);
  }
  float m = kNegInf, l = 0.f;
  float z[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) z[j] = 0.f;

  const float c2 = p.scale * kLog2e;
  auto consume = [&](int jstep, auto u) {
    constexpr int U = decltype(u)::value;
    if (jstep >= ns) return;
    const float dot = row_sum<LPR>(q.dot(kr[U]) * bf2f(ksr[U]), c);
    const int row = (split + jstep * nsp) * ROWS + roff;
    if (act && row < S) {
      const float u2 = dot * c2;
      const float ev = u2 * frcp(1.0f + fexp2(-u2));
      if (ev > m + kRescale) {
        const float alpha = fexp2(m - ev);  // 0 on the first row
        l *= alpha;
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] *= alpha;
        m = ev;
      }
      const float pr = fexp2(ev - m);
      l += pr;
      add4(z, vr[U], pr * bf2f(vsr[U]));
    }
  };
  for (int j = 0; j < ns; j += 4) {
    fetch(j + 3, I3{});
    consume(j, I0{});
    fetch(j + 4, I0{});
    consume(j + 1, I1{});
    fetch(j + 5, I1{});
    consume(j + 2, I2{});
    fetch(j + 6, I2{});
    consume(j + 3, I3{});
  }

  // ---- merge of the workgroup's row groups (the lanes of a row hold the same m and l) ----
  const float mw = wave_max(m);
  if (lane == 0) sm[wave] = mw;
  __syncthreads();
  float M = sm[0];
#pragma unroll
  for (int w = 1; w < kD4Waves; ++w) M = fmaxf(M, sm[w]);
  const float a = fexp2(m - (M == kNegInf ? 0.f : M));  // 0 for a row group without rows
  const float lw = wave_sum_lane0(act && c == 0 ? l * a : 0.f);
  if (lane == 0) sl[wave] = lw;
  float* zg = zred + roff * ZS + 32 * c;
  if (act) {
#pragma unroll
    for (int j = 0; j < 32; j += 4)
      *reinterpret_cast<float4*>(zg + j) = make_float4(z[j] * a, z[j + 1] * a, z[j + 2] * a, z[j + 3] * a);
  }
  __syncthreads();
  {
    const int d = tid % CL, part = tid / CL;
    if (part < PARTS) {
      constexpr int N = ROWS / PARTS;
      const float* col = zred + part * N * ZS + d;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int g2 = 0; g2 < N; g2 += 2) {
        s0 += col[g2 * ZS];
        s1 += col[(g2 + 1) * ZS];
      }
      csum[part][d] = s0 + s1;
    }
  }
  __syncthreads();
  float zs = 0.f, L4 = 0.f;
  if (tid < D) {
#pragma unroll
    for (int k = 0; k < PARTS; ++k) zs += csum[k][tid];
  }
#pragma unroll
  for (int w = 0; w < kD4Waves; ++w) L4 += sl[w];
  if (nsp == 1) {
    // one split: its sums are the head's, and no other workgroup counts (start of a conversation at
    // batch 1, head dim 48: 6.7 us a step with the publication, see the figures above)
    if (tid < D) zred[2 + tid] = zs;
    if (tid == 0) {
      zred[0] = M;
      zred[1] = L4;
    }
  } else {
    float* part = p.part + (int64_t(bh) * nsp + split) * (D + 2);
    if (tid < D) put_coherent(part + 2 + tid, zs);
    if (tid == 0) {
      put_coherent(part, M);
      put_coherent(part + 1, L4);
    }
    // publish, then count: agent-scope stores are acknowledged at the device-coherent level before the
    // barrier, the count's add is issued after it, and the workgroup that sees the last count reads the
    // partials with agent-scope loads
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      const int before = __hip_atomic_fetch_add(p.cnt + bh * kD4CntStride, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_last = before == nsp - 1;
    }
    __syncthreads();
    if (!s_last) return;

    // ---- the last workgroup of the head ----
    const int np = nsp * (D + 2);
    const float* pb = p.part + int64_t(bh) * np;
    constexpr int KP = (kD4MaxSplits * (DP + 2) + kD4Threads - 1) / kD4Threads;
    float pv[KP];
#pragma unroll
    for (int k = 0; k < KP; ++k) pv[k] = get_coherent(pb + min(tid + k * kD4Threads, np - 1));
#pragma unroll
    for (int k = 0; k < KP; ++k)
      if (tid + k * kD4Threads < np) zred[tid + k * kD4Threads] = pv[k];
  }
  __syncthreads();
  const int stride = D + 2;
  if (wave == 0) {
    const float ms = lane < nsp ? zred[lane * stride] : kNegInf;
    const float mx = wave_max(ms);
    const float Mh = mx == kNegInf ? 0.f : mx;
    const float w = fexp2(ms - Mh);
    if (lane < nsp) wsp[lane] = w;
    const float ls = wave_sum_lane0(lane < nsp ? zred[lane * stride + 1] * w : 0.f);
    if (lane == 0) {
      sML[0] = Mh;
      sML[1] = ls;
    }
  } else if (wave == 1) {
    float u = 0.f;
    for (int d = lane; d < D; d += 64) u = fmaf(sq[d], knew[d], u);
    u = wave_sum_lane0(u);
    if (lane == 0) sML[2] = u;
  } else if (wave == 2 && lane < 32 && !bad) {
    // the new rows in 4 bits: 16 octets of P2, then 16 of I~ (those past the padded head dim hold zeros)
    const int o = lane & 15;
    const float* src = (lane < 16 ? knew : inew) + 8 * o;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = src[j];
    bf16_t s;
    const uint32_t w = encode4(x, s);
    if (o < 4 * G) {
      uint8_t* cb = (lane < 16 ? p.kc : p.vc) + b * p.c_sb + h * p.c_sh + int64_t(S) * (16 * G);
      *reinterpret_cast<uint32_t*>(cb + 4 * o) = w;
      bf16_t* sb = (lane < 16 ? p.ks : p.vs) + b * p.s_sb + h * p.s_sh + int64_t(S) * G;
      if ((o & 3) == 0) sb[o >> 2] = s;
    }
  }
  __syncthreads();
  const float Mh = sML[0], L = sML[1];
  const float sself = sigmoid_acc(sML[2] * p.scale * p.tau_inv);
  const bool has = L != 0.f;  // NaN rows keep their NaN
  const float lse = has ? (Mh + __log2f(L)) * kLn2 : kNegInf;
  const float gate = has ? sigmoid_acc(lse - lam * logf((float)S + 1.0f) - sself) : 0.f;
  const float invL = has ? 1.0f / L : 0.f;
  T* y = reinterpret_cast<T*>(p.y) + b * p.y_sb + h * D;
  for (int d = tid; d < D; d += kD4Threads) {
    float zsum = 0.f;
#pragma unroll 8
    for (int s2 = 0; s2 < nsp; ++s2) zsum = fmaf(zred[s2 * stride + 2 + d], wsp[s2], zsum);
    const float yv = (1.0f - gate) * inew[d] + gate * zsum * invL;
    y[d] = E::from_f(bad ? __builtin_nanf("") : yv);
  }
  if (tid == 0) {
    if (nsp > 1) __hip_atomic_store(p.cnt + bh * kD4CntStride, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    p.g[bh] = bad ? __builtin_nanf("") : gate;
    if ((p.flags & MOTE_DECODE_ADVANCE) || p.xm) {
      // the last head of the sequence: every workgroup of it has read S[b] by now
      int before;
      if (p.xm)
        before = __hip_atomic_fetch_add(p.cnt_seq + b * kD4CntStride, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
      else
        before = __hip_atomic_fetch_add(p.cnt_seq + b * kD4CntStride, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (before == p.H - 1) {
        __hip_atomic_store(p.cnt_seq + b * kD4CntStride, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (p.flags & MOTE_DECODE_ADVANCE) p.S[b] = S64 + 1;
        if (p.xm) {
          float sum = 0.f;  // fixed head order
          for (int hh = 0; hh < p.H; ++hh) sum += p.g[b * p.H + hh];
          p.xm[b] = sum / float(p.H);
        }
      }
    }
  }
}

static int groups4(int D) { return (D + kGroup4 - 1) / kGroup4; }
static int rows4(int G) { return 64 / G * kD4Waves; }

// Splits per head. One for a cache of up to four steps, which needs no merge over workgroups (batch 1, head
// dim 48, 256 rows: 5.5 us a step, 7.0 as two splits). Else a workgroup per CU over the whole batch, each of
// at least two steps; two per CU where each still has a dozen steps (more loads in flight: batch 16, 4700
// rows, 17.2 -> 16.1 us; 32768 rows 106 -> 104 us; below, the merge costs more: batch 4, 10.3 and 10.9 us).
// At most one split per lane of the merging wave.
static int splits4(const mote_relation_decode4_args* a) {
  const int64_t BH = int64_t(a->B) * a->H, rows = rows4(groups4(a->D));
  const int64_t steps = (int64_t(a->capacity) + rows - 1) / rows;
  if (steps <= 4) return 1;
  int64_t n = device_cu_count() / BH;
  if (n < 1) n = 1;
  if (steps >= 12 * 2 * n) n *= 2;
  if (n > (steps + 1) / 2) n = (steps + 1) / 2;
  return int(n < kD4MaxSplits ? n : kD4MaxSplits);
}

struct Dec4Ws {
  size_t cnt, total;
  int nsplit;
};
// Counters in the first half of a workspace, partials in the second, whatever the sizes: a call of other sizes on
// the same bytes finds its counters at zero, never where an earlier one left partials. (With the partials right
// behind the counters, B = 1, H = 4, D = 40 with 5120 rows and B = H = 4, D = 48 with 768 shared their 14720 bytes,
// and the second call counted on the first one's floats: no workgroup was the last, nothing was written.)
static Dec4Ws ws4(const mote_relation_decode4_args* a) {
  const size_t BH = size_t(a->B) * a->H, line = kD4CntStride * sizeof(int);
  Dec4Ws w;
  w.cnt = size_t(a->B) * line;
  w.nsplit = splits4(a);
  const size_t counters = w.cnt + BH * line, partials = BH * size_t(w.nsplit) * size_t(a->D + 2) * sizeof(float);
  w.total = 2 * ((std::max(counters, partials) + 15) / 16 * 16);
  return w;
}

size_t decode4_workspace_bytes(const mote_relation_decode4_args* a) {
  if (a->B <= 0 || a->H <= 0 || a->D <= 0 || a->D > 128 || a->capacity <= 0) return 0;
  return ws4(a).total;
}

int launch_decode4(const mote_relation_decode4_args* a, hipStream_t stream) {
  const char* what = "relation_decode4";
  if (!a) return set_error(MOTE_ERR_ARGUMENT, "%s: null args", what);
  if (a->dtype != MOTE_F32 && a->dtype != MOTE_BF16) return set_error(MOTE_ERR_ARGUMENT, "%s: bad dtype %d", what, a->dtype);
  if (a->D <= 0 || a->D > 128 || a->D % 8)
    return set_error(MOTE_ERR_SHAPE, "%s: head dim %d unsupported (need 8 <= D <= 128, D %% 8 == 0)", what, a->D);
  if (a->B <= 0 || a->H <= 0 || a->H % 2 || a->capacity <= 0 || a->capacity > (1 << 30) ||
      int64_t(a->B) * a->H > (1 << 24))
    return set_error(MOTE_ERR_SHAPE, "%s: bad sizes", what);
  if (!a->lam || !a->S || !a->p1 || !a->p2 || !a->info || !a->y || !a->g)
    return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  if (const char* bad = bad_cache4(a->cache)) return set_error(MOTE_ERR_ARGUMENT, "%s: %s", what, bad);
  const Dec4Ws w = ws4(a);
  if (!a->workspace || a->workspace_bytes < w.total || reinterpret_cast<uintptr_t>(a->workspace) % 16)
    return set_error(MOTE_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes, %zu needed", what, a->workspace_bytes,
                     w.total);
  if (const char* bad = shared_cache4(a->cache, a->B, a->H, a->capacity, groups4(a->D)))
    return set_error(MOTE_ERR_ARGUMENT, "%s: %s", what, bad);
  if (!grid_fits(int64_t(a->B) * a->H * w.nsplit, kD4Threads))
    return set_error(MOTE_ERR_SHAPE, "%s: %d sequences of %d heads are too many for one launch", what, a->B, a->H);
  Dec4Params p;
  p.lam = a->lam; p.S = a->S;
  p.rope = a->inv_freq != nullptr;
  p.givens = a->theta != nullptr;
  p.inv_freq = p.rope ? a->inv_freq : a->lam;
  p.theta = p.givens ? a->theta : a->lam;
  p.p1 = a->p1; p.p2 = a->p2; p.info = a->info; p.in_sb = a->in_sb;
  p.kc = reinterpret_cast<uint8_t*>(a->cache.p2); p.vc = reinterpret_cast<uint8_t*>(a->cache.info);
  p.ks = reinterpret_cast<bf16_t*>(a->cache.p2_scale); p.vs = reinterpret_cast<bf16_t*>(a->cache.info_scale);
  p.c_sb = a->cache.codes_sb; p.c_sh = a->cache.codes_sh; p.s_sb = a->cache.scale_sb; p.s_sh = a->cache.scale_sh;
  p.y = a->y; p.y_sb = a->y_sb; p.g = a->g; p.xm = a->xm; p.run = a->run;
  char* ws = reinterpret_cast<char*>(a->workspace);
  p.part = reinterpret_cast<float*>(ws + a->workspace_bytes / 32 * 16);
  p.cnt = reinterpret_cast<int*>(ws + w.cnt);
  p.cnt_seq = reinterpret_cast<int*>(ws);
  p.B = a->B; p.H = a->H; p.D = a->D; p.cap = a->capacity; p.parity = a->layer_parity & 1; p.flags = a->flags;
  p.nsplit = w.nsplit;
  p.scale = 1.0f / sqrtf((float)a->D);
  p.tau_inv = 1.0f / a->tau_s;
  const dim3 grid(unsigned(a->B * a->H * p.nsplit)), block(kD4Threads);
  // a cache beyond the Infinity Cache (256 MB) is read past it: 453 MB of rows in 604 MB 105 -> 91 us a step; one
  // of 45 MB that it keeps between steps 16.2 us, 16.4 so
  const bool stream_rows = double(a->B) * a->H * a->capacity * 36 * groups4(a->D) > 268e6;
#define MOTE_DEC4_G(T_, G_)                                                                                    \
  if (stream_rows) hipLaunchKernelGGL((relation_decode4_kernel<T_, G_, true>), grid, block, 0, stream, p);     \
  else hipLaunchKernelGGL((relation_decode4_kernel<T_, G_, false>), grid, block, 0, stream, p);
#define MOTE_DEC4(T_)                                                                                          \
  switch (groups4(a->D)) {                                                                                     \
    case 1: MOTE_DEC4_G(T_, 1) break;                                                                          \
    case 2: MOTE_DEC4_G(T_, 2) break;                                                                          \
    case 3: MOTE_DEC4_G(T_, 3) break;                                                                          \
    default: MOTE_DEC4_G(T_, 4) break;                                                                         \
  }
  if (a->dtype == MOTE_BF16) MOTE_DEC4(bf16_t) else MOTE_DEC4(float)
#undef MOTE_DEC4
#undef MOTE_DEC4_G
  return check_launch(what);
}

}  // namespace mote
