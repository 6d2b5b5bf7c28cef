// One decode step of one Relation layer over the paged cache in 8 bits, one launch: the step of relation_decode.hip
// (RoPE / Givens / append / softmax read, split-S sweep with an in-kernel merge) with whole blocks decoded from
// their pages in registers, and the newest rows from the tail in the model's type.
//
// Per past row j: U_j = s_page <q, c_j> / sqrt(D), e_j = SiLU(U_j), running max m and sum l,
// z += exp(e_j - m) s'_page c'_j. A row is D bytes of P2 and of I~ and a page's two scales, half of bf16's bytes, so a
// sweep is bound by memory; a wave has a page at a time. P2: lane r holds row r, whose score is a sum of its own
// (codes as bf16 pairs, exact, for v_dot2_f32_bf16; fp32 queries in fp32). The
// weights go round in LDS (64 floats of the wave's own), and for I~ a lane holds 16 rows of one dim of each
// 16-dim chunk, so a sweep keeps D / 16 sums a lane and its end is two steps within a quad. The running maximum is
// the wave's: a rescale multiplies D / 16 sums and is taken when the maximum has grown by 2^8. Page numbers and
// scales are loaded a lane each, 64 pages a time, ahead of the pages.
//
// Grid, splits, predicate and the publish / count / merge protocol are those of relation_decode.hip; its comments
// give the reasons. The last workgroup of a head appends: it counts itself after every other one has read. 8 heads of 96,
// bf16: 1 x 4130 rows 8.4 us (the chain of it), 16 sequences of up to 4700 19.9 (87 MB, 4.4 TB/s); of 128, 16 of up to
// 32768 132 us (805 MB, 6.1 TB/s).
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "device.hpp"
#include "fp8.hpp"

namespace mote {

struct Dec8Params {
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
  float* ks;
  float* vs;
  void* kt;
  void* vt;
  const int32_t* table;
  int64_t codes_sp, scale_sp, tail_sb, table_sb;
  void* y;
  int64_t y_sb;
  float* g;
  float* xm;
  const unsigned char* run;
  float* part;  // [BH][nsplit][D + 2]  (max, l, z)
  int* cnt;
  int* cnt_seq;
  int B, H, D, pages, blocks, parity, flags, nsplit;
  float scale, tau_inv;
};

constexpr int kD8MaxSplits = 64;
constexpr int kD8Waves = 4;
constexpr int kD8Threads = 64 * kD8Waves;
constexpr int kD8CntStride = 64;  // ints between two completion counters: 256 bytes

__device__ __forceinline__ void put_coherent8(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get_coherent8(const float* p) {
  return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float lane_f32(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// <q, codes> over the 16 dims of chunk c; the query in LDS, read by all lanes at once (bf16 pairs in scalar registers
// spilled from head dim 96 on: batch 1, 4130 rows 10.6 us, 9.6 so)
template <typename T>
__device__ __forceinline__ void dot8(const T* q, int c, const Chunk& k, float& a, float& b) {
  if constexpr (sizeof(T) == 2) {
    const Chunk q0 = load_chunk(q + 16 * c), q1 = load_chunk(q + 16 * c + 8);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const Chunk& h = w < 2 ? q0 : q1;
      a = __builtin_amdgcn_fdot2_f32_bf16(codes8_bf16<false>(k.w[w]), __builtin_bit_cast(bf16x2, h.w[2 * w % 4]), a, false);
      b = __builtin_amdgcn_fdot2_f32_bf16(codes8_bf16<true>(k.w[w]), __builtin_bit_cast(bf16x2, h.w[2 * w % 4 + 1]), b, false);
    }
  } else {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float4 f = *reinterpret_cast<const float4*>(q + 16 * c + 4 * w);
      const f32x2 x = codes8_f32<false>(k.w[w]), y = codes8_f32<true>(k.w[w]);
      a = fmaf(x.x, f.x, a);
      b = fmaf(x.y, f.y, b);
      a = fmaf(y.x, f.z, a);
      b = fmaf(y.y, f.w, b);
    }
  }
}

template <typename T, int C, bool STREAM>
__global__ void __launch_bounds__(kD8Threads) relation_decode8_kernel(const Dec8Params p) {
  using E = Elem<T>;
  constexpr int DP = 16 * C;                  // padded head dim
  constexpr int PAGE = kPage8 * DP;           // bytes of a head's page
  constexpr int PER = 16 / int(sizeof(T));    // values of a 16-byte piece of a tail row
  constexpr int PIECES = DP / PER;            // pieces of a padded tail row
  __shared__ __align__(16) float zred[kD8MaxSplits * (DP + 2)];
  __shared__ __align__(16) float sq[DP], knew[DP], inew[DP];
  __shared__ __align__(16) T sqt[DP];  // the query as it is
  __shared__ __align__(16) float sp[kD8Waves][kPage8];
  __shared__ float sm[kD8Waves], sl[kD8Waves];
  __shared__ float wsp[kD8MaxSplits];
  __shared__ float sML[3];
  __shared__ int s_last;
  static_assert(kD8MaxSplits * (DP + 2) * 4 >= DP * kPitchT + 16, "a block being stored fits the table of partials");

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int BH = p.B * p.H;
  const int bh = blockIdx.x % BH;
  const int split = blockIdx.x / BH;
  const int b = bh / p.H, h = bh % p.H;
  const int D = p.D, half = D / 2;
  const int nsp = p.nsplit;

  // the small loads first: S and the page numbers arrive together, and the pages' loads need both
  int vzero;
  asm volatile("v_mov_b32 %0, 0" : "=v"(vzero));
  const int64_t S64 = p.S[b + vzero];
  const int run_v = (p.run ? p.run : reinterpret_cast<const unsigned char*>(p.lam))[vzero];
  const int32_t* tab = p.table + b * p.table_sb;
  const int psp = nsp > 1 ? nsp - 1 : 1;  // splits of the pages; the tail has the last one to itself
  const int t0 = split + psp * wave, step = psp * kD8Waves;  // this wave's pages: t0 + j step
  int32_t pid = tab[min(t0 + int64_t(lane) * step, int64_t(p.blocks) - 1)];
  const float lam = p.lam[vzero];
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

  if (p.run && run_v == 0) return;  // the predicate: every workgroup leaves before any write or count
  const bool bad = S64 < 0 || S64 >= int64_t(p.blocks) * kPage8;
  const int64_t S = bad ? 0 : S64;
  const int nfull = __builtin_amdgcn_readfirstlane(int(S / kPage8)), rest = __builtin_amdgcn_readfirstlane(int(S % kPage8));
  const int np = split < psp && nfull > t0 ? (nfull - t0 + step - 1) / step : 0;  // this wave's pages

  // two register sets for pages, the next one's loads ahead of this one's sums
  bool gone = false;  // a block without a page
  float ksl = 0.f, vsl = 0.f;
  auto resolve = [&](int j0) {  // numbers and scales of pages j0 + lane
    const bool live = j0 + lane < np;
    gone = gone || (live && (pid < 0 || pid >= p.pages));
    pid = min(max(pid, 0), p.pages - 1);
    if (live) {
      ksl = p.ks[pid * p.scale_sp + h];
      vsl = p.vs[pid * p.scale_sp + h];
    }
  };
  Chunk kr[2][C], vr[2][C];
  auto fetch = [&](int j, auto u) {
    constexpr int U = decltype(u)::value;
    const int64_t at = int64_t(__builtin_amdgcn_readlane(pid, j & 63)) * p.codes_sp + int64_t(h) * PAGE + 16 * lane;
#pragma unroll
    for (int c = 0; c < C; ++c) kr[U][c] = load_chunk_as<STREAM>(p.kc + at + c * (16 * kPage8));
#pragma unroll
    for (int c = 0; c < C; ++c) vr[U][c] = load_chunk_as<STREAM>(p.vc + at + c * (16 * kPage8));
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  if (np > 0) {
    resolve(0);
    fetch(0, I0{});
  }
  // the tail, by the last split: 16 rows a wave, a quad of lanes a row of P2, and for I~ a lane the dims that it has of a
  // page
  const int r0 = 16 * wave, quad = lane >> 2, part4 = lane & 3;
  const bool tailed = split == nsp - 1 && rest > r0;
  Chunk tk[(PIECES + 3) / 4];
  T tv[4][C];
  if (tailed) {
    const int64_t off = b * p.tail_sb + int64_t(h) * (kPage8 * D);
    const T* kt = reinterpret_cast<const T*>(p.kt) + off + (r0 + quad) * D;
    const T* vt = reinterpret_cast<const T*>(p.vt) + off + (r0 + part4) * D;
#pragma unroll
    for (int i = 0; i < (PIECES + 3) / 4; ++i) tk[i] = load_chunk(kt + min((part4 + 4 * i) * PER, D - PER));
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < C; ++c) tv[i][c] = vt[4 * i * D + min(16 * c + quad, D - 1)];
  }

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
    sqt[tid] = E::from_f(rq0);
    sqt[tid + half] = E::from_f(rq1);
    knew[tid] = rk0;
    knew[tid + half] = rk1;
  } else if (tid >= 128 && tid < 128 + D) {
    inew[tid - 128] = rin;
  }
  if (tid < DP - D) {  // padded dims hold zeros
    sq[D + tid] = 0.f;
    sqt[D + tid] = E::from_f(0.f);
    knew[D + tid] = 0.f;
    inew[D + tid] = 0.f;
  }
  __syncthreads();

  float m = kNegInf, l = 0.f;
  float z[C];
#pragma unroll
  for (int c = 0; c < C; ++c) z[c] = 0.f;
  float* spw = sp[wave];
  const float c2 = p.scale * kLog2e;

  // a row's weight from its score in log2 units; the maximum over the wave moves m
  auto silu2 = [&](float u2) { return u2 * frcp(1.0f + fexp2(-u2)); };
  auto raise = [&](float ev) {
    const float mx = wave_max(ev);
    if (mx > m + kRescale) {
      const float alpha = fexp2(m - mx);  // 0 on the first rows
      l *= alpha;
#pragma unroll
      for (int c = 0; c < C; ++c) z[c] *= alpha;
      m = mx;
    }
  };

  if (tailed) {
    const int row = r0 + quad;
    float u = 0.f;
#pragma unroll
    for (int i = 0; i < (PIECES + 3) / 4; ++i) {
      const int d = (part4 + 4 * i) * PER;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        float x;
        if constexpr (sizeof(T) == 2) x = __uint_as_float(k % 2 ? tk[i].w[k / 2] & 0xffff0000u : tk[i].w[k / 2] << 16);
        else x = __uint_as_float(tk[i].w[k]);
        if (d < D) u = fmaf(x, sq[d + k], u);
      }
    }
    u += dpp<kDppXor1>(u);
    u += dpp<kDppXor2>(u);
    const float ev = row < rest ? silu2(u * c2) : kNegInf;
    raise(ev);
    const float pr = row < rest ? fexp2(ev - m) : 0.f;
    if (part4 == 0) {
      l += pr;
      spw[quad] = pr;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = spw[part4 + 4 * i];
      const bool in = r0 + part4 + 4 * i < rest;  // rows behind may hold anything
#pragma unroll
      for (int c = 0; c < C; ++c) z[c] = in ? fmaf(w, E::to_f(tv[i][c]), z[c]) : z[c];
    }
    __builtin_amdgcn_wave_barrier();
  }

  auto consume = [&](int j, auto u) {
    constexpr int U = decltype(u)::value;
    float d0 = 0.f, d1 = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) dot8(sqt, c, kr[U][c], d0, d1);
    const float ev = silu2((d0 + d1) * (lane_f32(ksl, j & 63) * c2));
    raise(ev);
    const float pr = fexp2(ev - m);
    l += pr;
    spw[lane] = pr * lane_f32(vsl, j & 63);
    __builtin_amdgcn_wave_barrier();
    float w[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 f = *reinterpret_cast<const float4*>(spw + 16 * part4 + 4 * k);
      w[4 * k] = f.x; w[4 * k + 1] = f.y; w[4 * k + 2] = f.z; w[4 * k + 3] = f.w;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const f32x2 x = codes8_f32<false>(vr[U][c].w[k]), y = codes8_f32<true>(vr[U][c].w[k]);
        z[c] = fmaf(w[4 * k], x.x, z[c]);
        z[c] = fmaf(w[4 * k + 1], x.y, z[c]);
        z[c] = fmaf(w[4 * k + 2], y.x, z[c]);
        z[c] = fmaf(w[4 * k + 3], y.y, z[c]);
      }
    __builtin_amdgcn_wave_barrier();
  };
  for (int j0 = 0; j0 < np; j0 += 64) {
    if (j0 > 0) {  // the next 64 page numbers (the loads of their first page wait for them)
      pid = tab[min(t0 + (j0 + int64_t(lane)) * step, int64_t(p.blocks) - 1)];
      resolve(j0);
      fetch(j0, I0{});
    }
    const int n = min(64, np - j0);
    for (int j = 0; j < n; j += 2) {
      if (j + 1 < n) fetch(j0 + j + 1, I1{});
      consume(j0 + j, I0{});
      if (j + 1 < n) {
        if (j + 2 < n) fetch(j0 + j + 2, I0{});
        consume(j0 + j + 1, I1{});
      }
    }
  }
  if (__ballot(gone)) l = __builtin_nanf("");

  // ---- merge of the waves (m is the wave's, l a lane's rows, z a quad's dims over its lanes' rows) ----
  if (lane == 0) sm[wave] = m;
  __syncthreads();
  float M = sm[0];
#pragma unroll
  for (int w = 1; w < kD8Waves; ++w) M = fmaxf(M, sm[w]);
  const float a = fexp2(m - (M == kNegInf ? 0.f : M));  // 0 for a wave without rows
  const float lw = wave_sum_lane0(l * a);
  if (lane == 0) sl[wave] = lw;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float s = z[c];
    s += dpp<kDppXor1>(s);
    s += dpp<kDppXor2>(s);
    if (part4 == 0) zred[wave * DP + 16 * c + quad] = s * a;
  }
  __syncthreads();
  float zs = 0.f, L4 = 0.f;
#pragma unroll
  for (int w = 0; w < kD8Waves; ++w) L4 += sl[w];
  if (tid < D)
#pragma unroll
    for (int w = 0; w < kD8Waves; ++w) zs += zred[w * DP + tid];
  __syncthreads();
  if (nsp == 1) {  // one split: its sums are the head's
    if (tid < D) zred[2 + tid] = zs;
    if (tid == 0) {
      zred[0] = M;
      zred[1] = L4;
    }
  } else {
    float* part = p.part + (int64_t(bh) * nsp + split) * (D + 2);
    if (tid < D) put_coherent8(part + 2 + tid, zs);
    if (tid == 0) {
      put_coherent8(part, M);
      put_coherent8(part + 1, L4);
    }
    // publish, then count: agent-scope stores are acknowledged at the device-coherent level before the
    // barrier, the count's add is issued after it, and the workgroup that sees the last count reads the
    // partials with agent-scope loads
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      const int before = __hip_atomic_fetch_add(p.cnt + bh * kD8CntStride, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_last = before == nsp - 1;
    }
    __syncthreads();
    if (!s_last) return;

    // ---- the last workgroup of the head ----
    const int n = nsp * (D + 2);
    const float* pb = p.part + int64_t(bh) * n;
    constexpr int KP = (kD8MaxSplits * (DP + 2) + kD8Threads - 1) / kD8Threads;
    float pv[KP];
#pragma unroll
    for (int k = 0; k < KP; ++k) pv[k] = get_coherent8(pb + min(tid + k * kD8Threads, n - 1));
#pragma unroll
    for (int k = 0; k < KP; ++k)
      if (tid + k * kD8Threads < n) zred[tid + k * kD8Threads] = pv[k];
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
  }
  __syncthreads();
  const float Mh = sML[0], L = sML[1];
  const float sself = sigmoid_acc(sML[2] * p.scale * p.tau_inv);
  const bool has = L != 0.f;  // NaN rows keep their NaN
  const float lse = has ? (Mh + __log2f(L)) * kLn2 : kNegInf;
  const float gate = has ? sigmoid_acc(lse - lam * logf((float)S + 1.0f) - sself) : 0.f;
  const float invL = has ? 1.0f / L : 0.f;
  T* y = reinterpret_cast<T*>(p.y) + b * p.y_sb + h * D;
  for (int d = tid; d < D; d += kD8Threads) {
    float zsum = 0.f;
#pragma unroll 8
    for (int s2 = 0; s2 < nsp; ++s2) zsum = fmaf(zred[s2 * stride + 2 + d], wsp[s2], zsum);
    const float yv = (1.0f - gate) * inew[d] + gate * zsum * invL;
    y[d] = E::from_f(bad ? __builtin_nanf("") : yv);
  }
  if (!bad) {
    // the append: every workgroup of the head has read the tail by now
    const int64_t off = b * p.tail_sb + int64_t(h) * (kPage8 * D);
    T* kt = reinterpret_cast<T*>(p.kt) + off;
    T* vt = reinterpret_cast<T*>(p.vt) + off;
    for (int d = tid; d < 2 * D; d += kD8Threads) {
      if (d < D) kt[rest * D + d] = E::from_f(knew[d]);
      else vt[rest * D + d - D] = E::from_f(inew[d - D]);
    }
    if (rest == kPage8 - 1) {  // the block is whole: into its page
      const int32_t page = tab[nfull];
      if (page >= 0 && page < p.pages) {
        __syncthreads();  // y's sums are done with the table of partials
        uint32_t* top = reinterpret_cast<uint32_t*>(zred);
        uint8_t* bytes = reinterpret_cast<uint8_t*>(zred + 4);
        auto from = [&](const T* t, const float* fresh) {
          return [=](int row, int ch, float* x) {
            const float* f = fresh + ch * 16;
            const T* s = t + row * D + ch * 16;
            if (row == kPage8 - 1) {
#pragma unroll
              for (int k = 0; k < 16; ++k) x[k] = f[k];
            } else {
              load_values<8>(s, x);
              if (ch * 16 + 8 < D) load_values<8>(s + 8, x + 8);
            }
          };
        };
        const int64_t at = page * p.codes_sp + int64_t(h) * PAGE, sat = page * p.scale_sp + h;
        store_block8<C, false>(from(kt, knew), p.kc + at, p.ks + sat, top, bytes);
        __syncthreads();
        store_block8<C, true>(from(vt, inew), p.vc + at, p.vs + sat, top, bytes);
      }
    }
  }
  if (tid == 0) {
    if (nsp > 1) __hip_atomic_store(p.cnt + bh * kD8CntStride, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    p.g[bh] = bad ? __builtin_nanf("") : gate;
    if ((p.flags & MOTE_DECODE_ADVANCE) || p.xm) {
      // the last head of the sequence: every workgroup of it has read S[b] by now
      int before;
      if (p.xm)
        before = __hip_atomic_fetch_add(p.cnt_seq + b * kD8CntStride, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
      else
        before = __hip_atomic_fetch_add(p.cnt_seq + b * kD8CntStride, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (before == p.H - 1) {
        __hip_atomic_store(p.cnt_seq + b * kD8CntStride, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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

// Splits per head: a workgroup per CU over the whole batch, each with a page for every wave; two per CU where every wave
// still has two pages (more loads in flight, and sequences of unlike lengths even out: 16 x 4700 rows of 4 x 48, fp32
// 11.1 -> 10.1 us, 2 x 32768 of 8 x 128 27.3 -> 26.7; below, the merge costs more: 1 x 1000 rows 9.4 and 9.7). Where there
// are several, one more for the tail alone, which is as long a chain as a page (1 x 4130 rows of 8 x 96 9.5 -> 8.4 us,
// 4 x 4130 10.8 -> 9.3, 16 x 4700 19.4 -> 18.8). At most one split per lane of the merging wave.
static int splits8(const mote_relation_decode8_args* a) {
  const int64_t BH = int64_t(a->B) * a->H, blocks = a->cache.blocks;
  int64_t n = device_cu_count() / BH;
  if (n < 1) n = 1;
  if (blocks >= 2 * kD8Waves * 2 * n) n *= 2;
  n = std::min(n, (blocks + kD8Waves - 1) / kD8Waves);
  if (n > 1) ++n;
  return int(n < kD8MaxSplits ? n : kD8MaxSplits);
}

// counters in the first half of a workspace, partials in the second, whatever the sizes: a call of other sizes on
// the same bytes finds its counters at zero, never where an earlier one left partials
struct Dec8Ws {
  size_t cnt, total;
  int nsplit;
};
static Dec8Ws ws8(const mote_relation_decode8_args* a) {
  const size_t BH = size_t(a->B) * a->H, line = kD8CntStride * sizeof(int);
  Dec8Ws w;
  w.cnt = size_t(a->B) * line;
  w.nsplit = splits8(a);
  const size_t counters = w.cnt + BH * line, partials = BH * size_t(w.nsplit) * size_t(a->D + 2) * sizeof(float);
  w.total = 2 * ((std::max(counters, partials) + 15) / 16 * 16);
  return w;
}

size_t decode8_workspace_bytes(const mote_relation_decode8_args* a) {
  if (a->B <= 0 || a->H <= 0 || a->D <= 0 || a->D > 128 || a->cache.blocks <= 0) return 0;
  return ws8(a).total;
}

int launch_decode8(const mote_relation_decode8_args* a, hipStream_t stream) {
  const char* what = "relation_decode8";
  if (!a) return set_error(MOTE_ERR_ARGUMENT, "%s: null args", what);
  if (a->dtype != MOTE_F32 && a->dtype != MOTE_BF16) return set_error(MOTE_ERR_ARGUMENT, "%s: bad dtype %d", what, a->dtype);
  if (a->D <= 0 || a->D > 128 || a->D % 8)
    return set_error(MOTE_ERR_SHAPE, "%s: head dim %d unsupported (need 8 <= D <= 128, D %% 8 == 0)", what, a->D);
  if (a->B <= 0 || a->H <= 0 || a->H % 2 || int64_t(a->B) * a->H > (1 << 24))
    return set_error(MOTE_ERR_SHAPE, "%s: bad sizes", what);
  if (!a->lam || !a->S || !a->p1 || !a->p2 || !a->info || !a->y || !a->g)
    return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  if (const char* bad = bad_cache8(a->cache, a->B, a->H, a->D, a->dtype == MOTE_F32 ? 4 : 2))
    return set_error(MOTE_ERR_ARGUMENT, "%s: %s", what, bad);
  const Dec8Ws w = ws8(a);
  if (!a->workspace || a->workspace_bytes < w.total || reinterpret_cast<uintptr_t>(a->workspace) % 16)
    return set_error(MOTE_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes, %zu needed", what, a->workspace_bytes,
                     w.total);
  if (!grid_fits(int64_t(a->B) * a->H * w.nsplit, kD8Threads))
    return set_error(MOTE_ERR_SHAPE, "%s: %d sequences of %d heads are too many for one launch", what, a->B, a->H);
  Dec8Params p;
  p.lam = a->lam; p.S = a->S;
  p.rope = a->inv_freq != nullptr;
  p.givens = a->theta != nullptr;
  p.inv_freq = p.rope ? a->inv_freq : a->lam;
  p.theta = p.givens ? a->theta : a->lam;
  p.p1 = a->p1; p.p2 = a->p2; p.info = a->info; p.in_sb = a->in_sb;
  const mote_cache8& c = a->cache;
  p.kc = reinterpret_cast<uint8_t*>(c.p2); p.vc = reinterpret_cast<uint8_t*>(c.info);
  p.ks = c.p2_scale; p.vs = c.info_scale; p.kt = c.p2_tail; p.vt = c.info_tail; p.table = c.table;
  p.codes_sp = c.codes_sp; p.scale_sp = c.scale_sp; p.tail_sb = c.tail_sb; p.table_sb = c.table_sb;
  p.pages = c.pages; p.blocks = c.blocks;
  p.y = a->y; p.y_sb = a->y_sb; p.g = a->g; p.xm = a->xm; p.run = a->run;
  char* ws = reinterpret_cast<char*>(a->workspace);
  p.part = reinterpret_cast<float*>(ws + a->workspace_bytes / 32 * 16);
  p.cnt = reinterpret_cast<int*>(ws + w.cnt);
  p.cnt_seq = reinterpret_cast<int*>(ws);
  p.B = a->B; p.H = a->H; p.D = a->D; p.parity = a->layer_parity & 1; p.flags = a->flags;
  p.nsplit = w.nsplit;
  p.scale = 1.0f / sqrtf((float)a->D);
  p.tau_inv = 1.0f / a->tau_s;
  const dim3 grid(unsigned(a->B * a->H * p.nsplit)), block(kD8Threads);
  // pages are read past the caches once a layer's pool outgrows the L2s, though the Infinity Cache may hold it: 87 MB of
  // rows in 117 MB 22.0 -> 19.8 us, 805 MB in 1.07 GB 159 -> 140; 53 MB in 53 MB 10.8 either way
  const bool stream_rows = 2.0 * c.pages * a->H * kPage8 * 16 * chunks8(a->D) > 64e6;
#define MOTE_D8(C_)                                                                                                    \
  if (stream_rows) hipLaunchKernelGGL((relation_decode8_kernel<T, C_, true>), grid, block, 0, stream, p);              \
  else hipLaunchKernelGGL((relation_decode8_kernel<T, C_, false>), grid, block, 0, stream, p);
#define MOTE_D8_ALL                  \
  switch (chunks8(a->D)) {           \
    case 1: MOTE_D8(1) break;        \
    case 2: MOTE_D8(2) break;        \
    case 3: MOTE_D8(3) break;        \
    case 4: MOTE_D8(4) break;        \
    case 5: MOTE_D8(5) break;        \
    case 6: MOTE_D8(6) break;        \
    case 7: MOTE_D8(7) break;        \
    default: MOTE_D8(8) break;       \
  }
  if (a->dtype == MOTE_BF16) {
    using T = bf16_t;
    MOTE_D8_ALL
  } else {
    using T = float;
    MOTE_D8_ALL
  }
#undef MOTE_D8_ALL
#undef MOTE_D8
  return check_launch(what);
}

}  // namespace mote
