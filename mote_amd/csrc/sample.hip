// The next token of every row of logits from one random number (mote_sample; mote_relation.h has the definition).
//
// Every step of it is one search: tokens in the order of their logits (ties to the lowest index), find the first
// at which a running sum passes a target. Top-k asks for the weight of the first k (the sum counts), top-p for the
// weight up to the token at which p of that is reached, the draw for the token at which u of the weight kept is
// passed; min-p is a sum over the row. Nothing is sorted. Weights are fixed-point numbers of 2^-43 of the largest,
// rounded from an fp64 exponential, in 64 bits: sums of up to 2^20 of them are exact, so their order does not matter
// and atomics may make them, and a border differs from the real one by V 2^-44 of the largest weight at most.
//
// A row: its maximum; a histogram over intervals of the logit (an interval's count and weight); its prefix sums, in
// which a search finds an interval; then that interval's tokens, which are gathered in LDS unless they are too many
// (many equal logits): up to 64 each count the ones before them, more are told apart by the digits of their keys, and
// equal ones by those of their indices.
//
// Up to 8192 logits a workgroup has a row, in registers. Longer rows go in pieces over three launches: the maximum; the
// histogram; then in every piece (a last one's, handed to the others, took two more trips) the prefix sums and the intervals
// that a search can end in, of which it gathers its tokens, and the searches by the row's last piece.
//
// A short row is a chain of a launch, its loads and some barriers: 1 x 271 5.0 us, 256 x 271 7.0. 64 x 131072 in fp32 (34 MB,
// 6.6 us at a copy's rate) with top-k 2000, top-p and min-p: 6.3 + 16.9 + 20.9 us.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "device.hpp"
#include "params.hpp"
#include "stream.hpp"
#include "wave_uint.hpp"

namespace mote {

typedef unsigned long long u64;

struct SampleParams {
  const void* logits;
  int64_t l_sr;
  const float* u;
  float temperature, top_p, min_p;
  int64_t top_k;
  const float* temperature_dev;
  const float* top_p_dev;
  const float* min_p_dev;
  const int64_t* top_k_dev;
  int64_t* tokens;
  const unsigned char* run;
  int V;
  // rows in pieces
  char* ws;
  int pieces, piece;  // logits of a piece: whole 16-byte chunks
};

// intervals of a long row (512, 1024, 2048: 64 x 131072 fp32 with top-k 1000, top-p and min-p 43.5, 41.2, 44.7 us, 1 x
// 131072 25.4, 22.5, 21.7; fewer cost less to add up, and more than 64 tokens in one cost a search in digits)
constexpr int kBins = 1024;
constexpr int kList = 1024;                      // tokens of an interval that are searched in LDS
constexpr double kOne = 8796093022208.0;         // 2^43: the largest weight
constexpr float kReach = 31.0f;                  // exp(-31) < 2^-44: no weight from there on
constexpr double kReach2 = 46.0;                 // nor at 2^-46
constexpr int kMaxPieces = 64;

// order of logits: a larger key comes first (the sum with +0 makes one zero of two)
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// The intervals that each stage can end in (the weight that the ones before it leave is only known to within an interval
// until they are searched), and how many tokens are in them.
struct Plan {
  int from[3], to[3];
  uint32_t total;
  __device__ __forceinline__ bool has(int bin) const {
    return (bin >= from[0] && bin <= to[0]) || (bin >= from[1] && bin <= to[1]) || (bin >= from[2] && bin <= to[2]);
  }
};
struct Digits {
  u64 mass[256];
  uint32_t cnt[256];
};
template <int BINS, int LIST>
struct Lds {
  u64 mass[BINS];  // prefix sums once scanned
  uint32_t cnt[BINS];
  u64 lw[LIST];  // the tokens of the intervals that a search can end in
  uint32_t lkey[LIST], lidx[LIST];
  int lbin[LIST];
  u64 order[64];
  uint16_t slot[64];
  Digits dig[3];
  u64 red64[16];
  uint32_t red32[16], low32[16];
  float redf[16], redm[16];
  u64 high, kept;
  uint32_t idx, n, first, token;
  int last, stage;
  Plan plan;
};

// wave prefix sums by DPP moves within and across rows of 16 lanes (a shuffle through LDS costs several times more)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_or0(uint32_t x) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(x), CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_or0(u64 x) {
  return (u64(dpp_or0<CTRL, ROWS>(uint32_t(x >> 32))) << 32) | dpp_or0<CTRL, ROWS>(uint32_t(x));
}
template <typename N>
__device__ __forceinline__ N wave_scan(N x) {  // inclusive
  x += dpp_or0<0x111, 0xF>(x);  // row_shr:1
  x += dpp_or0<0x112, 0xF>(x);
  x += dpp_or0<0x114, 0xF>(x);
  x += dpp_or0<0x118, 0xF>(x);
  x += dpp_or0<0x142, 0xA>(x);  // row_bcast:15 into rows 1 and 3
  x += dpp_or0<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
  return x;
}

// exclusive prefix over the workgroup's threads
template <int NT, typename S>
__device__ __forceinline__ void scan_block(u64& m, uint32_t& c, S& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 m1 = wave_scan(m);
  const uint32_t c1 = wave_scan(c);
  __syncthreads();
  if (lane == 63) {
    s.red64[wave] = m1;
    s.red32[wave] = c1;
  }
  __syncthreads();
  m = m1 - m;
  c = c1 - c;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) {
      m += s.red64[w];
      c += s.red32[w];
    }
  }
}

// R > 0: a thread holds elements tid + r NT of the row; R == 0: the row is read each time, 16 bytes a thread
template <typename T, int NT, int R>
struct Row {
  static constexpr int PER = 16 / int(sizeof(T));
  static constexpr int AHEAD = 4;  // loads in flight, the first ones from open() on: 64 x 131072 fp32 in 56 us with one, 53 so
  const T* p;
  int from, to;
  float x[R > 0 ? R : 1];
  Chunk head[R > 0 ? 1 : AHEAD];
  __device__ __forceinline__ void load(Chunk (&q)[AHEAD], int c0) const {
    const int whole = (to - from) / PER;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (c0 + u * NT < whole) q[u] = load_any(p + from + (c0 + u * NT) * PER);
  }
  __device__ __forceinline__ void open(const T* row, int f, int t) {
    p = row;
    from = f;
    to = t;
    if constexpr (R == 0) load(head, threadIdx.x);
    if constexpr (R > 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int i = from + int(threadIdx.x) + r * NT;
        x[r] = i < to ? Elem<T>::to_f(p[i]) : 0.f;
      }
    }
  }
  // many(v, i) for PER logits from i on, one(v, i) for single ones
  template <typename Many, typename One>
  __device__ __forceinline__ void each(Many many, One one) const {
    if constexpr (R > 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int i = from + int(threadIdx.x) + r * NT;
        if (i < to) one(x[r], i);
      }
    } else {
      const int whole = (to - from) / PER;
      Chunk q[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) q[u] = head[u];
      for (int c0 = threadIdx.x; c0 < whole; c0 += NT * AHEAD) {
        if (c0 != int(threadIdx.x)) load(q, c0);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int c = c0 + u * NT;
          if (c >= whole) break;
          float v[PER];
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            if constexpr (sizeof(T) == 2) v[k] = __uint_as_float(k % 2 ? q[u].w[k / 2] & 0xffff0000u : q[u].w[k / 2] << 16);
            else v[k] = __uint_as_float(q[u].w[k]);
          }
          many(v, from + c * PER);
        }
      }
      for (int i = from + whole * PER + int(threadIdx.x); i < to; i += NT) one(Elem<T>::to_f(p[i]), i);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    each([&](const float (&v)[PER], int i) {
#pragma unroll
      for (int k = 0; k < PER; ++k) f(v[k], i + k);
    }, f);
  }
};

// a row's settings
struct Setting {
  float temperature, top_p, min_p, u;
  int64_t top_k;
  __device__ __forceinline__ Setting(const SampleParams& p, int b)
      : temperature(p.temperature_dev ? p.temperature_dev[b] : p.temperature), top_p(p.top_p_dev ? p.top_p_dev[b] : p.top_p),
        min_p(p.min_p_dev ? p.min_p_dev[b] : p.min_p), u(p.u[b]), top_k(p.top_k_dev ? p.top_k_dev[b] : p.top_k) {}
  __device__ __forceinline__ bool nan() const {
    return u != u || temperature != temperature || top_p != top_p || min_p != min_p;
  }
  // the first of the order is all that is kept: no weight reaches a min-p above 1, not even those equal to the first's
  __device__ __forceinline__ bool greedy() const { return !(temperature > 0.f) || min_p > 1.f; }
};

// intervals and weights of a row
template <int BINS>
struct Scale {
  float top;     // the largest logit
  float per;     // intervals per unit of the logit
  double rate;   // log2(e) / temperature
  __device__ __forceinline__ Scale(const Setting& o, float top_, float low) : top(top_) {
    rate = fmax(1.44269504088896340736 / double(o.temperature), 1e-300);  // no 0 times infinity
    const float span = fminf(kReach * o.temperature, top - low);  // at most as far as weights reach
    per = span > 0.f ? (float(BINS) - 1.5f) / span : 0.f;  // the last interval is for masked logits (see reach())
    if (!(per < __builtin_inff())) per = 3e38f;  // a span below the normal numbers
  }
  // Never smaller for a smaller logit. Infinite differences end up in the last interval, and so does 0 times one; the
  // NaN between two infinite logits is a difference of 0.
  __device__ __forceinline__ int bin(float x) const { return int(fminf(fmaxf(top - x, 0.f) * per, float(BINS - 1))); }
  // The weight in units of 2^-43, from 2^n (1 + f q(f)) with |f| <= 1/2, q of degree 9 through (2^f - 1) / f at Chebyshev's
  // points (off by 2^-50), in fp64 without a branch.
  __device__ __forceinline__ u64 weight(float x) const {
    constexpr double magic = 6755399441055744.0;  // 1.5 x 2^52: a sum with it holds the nearest whole number in its low bits
    const double y = fmax(fmin((double(x) - double(top)) * rate, 0.0), -kReach2);  // NaN between two infinite logits: 0
    const double t = y + magic, f = y - (t - magic);
    double e = fma(0x1.e5e9f548e5725p-28, f, 0x1.b6571de2f2351p-24);
    e = fma(e, f, 0x1.62bfe46117445p-20);
    e = fma(e, f, 0x1.ffcb76789860fp-17);
    e = fma(e, f, 0x1.4309130378460p-13);
    e = fma(e, f, 0x1.5d87fe908f88ap-10);
    e = fma(e, f, 0x1.3b2ab6fba385fp-7);
    e = fma(e, f, 0x1.c6b08d7044119p-5);
    e = fma(e, f, 0x1.ebfbdff82c590p-3);
    e = fma(e, f, 0x1.62e42fefa39f7p-1);
    e = fma(e, f, 1.0);
    const uint32_t n = uint32_t(__double_as_longlong(t));
    const double scale = __longlong_as_double(static_cast<long long>(u64((n + 1023 + 43) << 20) << 32));  // 2^(n + 43)
    return u64(__double_as_longlong(fma(e, scale, 4503599627370496.0))) & ((u64(1) << 52) - 1);
  }
  // Bounds of the logits of intervals `from` to `to` and of some beside them: half an interval covers the roundings of
  // bin() and of `width` (1 / per), and the bounds' own are monotonic, so they pass no logit. A bound that is not finite is
  // none: where differences and 31 T overflow, `per` is 0 and the last interval holds logits that have weight.
  __device__ __forceinline__ void reach(int from, int to, float width, float& lo, float& hi) const {
    const float a = fmaf(-(float(from) - 0.5f), width, top), b = fmaf(-(float(to) + 1.5f), width, top), inf = __builtin_inff();
    hi = from > to ? -inf : from > 0 && a > -inf ? a : inf;
    lo = from > to ? inf : to < BINS - 1 && b == b ? b : -inf;
  }
};

// the smallest weight that min_p (at most 1) keeps: the exact product is a whole number or lies between two
__device__ __forceinline__ u64 floor_of(float min_p) { return u64(__builtin_ceil(double(fmaxf(min_p, 0.f)) * kOne)); }
// What a row's three searches are for: the last token that top-k keeps (of the running count), the last that top-p keeps,
// the draw.
struct Goals {
  u64 fp, fu;  // top_p and u in units of 2^-64
  int64_t last;
  bool by_k, by_p;
  __device__ __forceinline__ Goals(const Setting& o, int V)
      : fp(u64(fmaxf(o.top_p, 0.f) * 18446744073709551616.0)),
        fu(u64(double(fminf(fmaxf(o.u, 0.f), 0x1.fffffep-1f)) * 18446744073709551616.0)), last(o.top_k - 1),
        by_k(o.top_k > 0 && o.top_k < V), by_p(o.top_p < 1.f) {}
  __device__ __forceinline__ bool has(int stage) const { return stage == 0 ? by_k : stage == 1 ? by_p : true; }
  // passed by the token that the stage is for, when the weight `kept` is left before it
  __device__ __forceinline__ u64 target(int stage, u64 kept) const {
    if (stage == 0) return u64(last);
    const u64 f = stage == 1 ? fp : fu, up = __umul64hi(f, kept);
    if (stage == 2) return up;
    const u64 want = up + (f * kept != 0);  // top-p: the first token that reaches p kept
    return want > 0 ? want - 1 : 0;
  }
};

// A row's (or a piece's) histogram in LDS. Where every logit that a wave holds is in the first or the last interval (equal
// or masked ones) it adds them at once: 64 additions to one place take their turns.
template <int BINS, typename Rows, typename S>
__device__ __forceinline__ u64 histogram(const Rows& row, const Scale<BINS>& sc, float min_p, S& s) {
  constexpr int PER = Rows::PER;
  const bool cut = min_p > 0.f;
  const u64 least = floor_of(min_p);
  u64 high = 0;  // the weight that min_p keeps
  auto above = [&](u64 w) {
    if (cut) high += w >= least ? w : 0;
  };
  row.each(
      [&](const float (&v)[PER], int) {
        u64 w[PER];
        int bin[PER], any = 0, all = BINS - 1;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          w[k] = sc.weight(v[k]);
          bin[k] = sc.bin(v[k]);
          any |= bin[k];
          all &= bin[k];
          above(w[k]);
        }
        if (__ballot(any == 0) == ~u64(0) || __ballot(all == BINS - 1) == ~u64(0)) {
          u64 sum = w[0];
#pragma unroll
          for (int k = 1; k < PER; ++k) sum += w[k];
          sum = wave_scan(sum);
          if ((threadIdx.x & 63) == 63) {
            atomicAdd(&s.mass[bin[0]], sum);
            atomicAdd(&s.cnt[bin[0]], uint32_t(64 * PER));
          }
          return;
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          atomicAdd(&s.mass[bin[k]], w[k]);
          atomicAdd(&s.cnt[bin[k]], 1u);
        }
      },
      [&](float x, int) {
        const u64 w = sc.weight(x);
        const int bin = sc.bin(x);
        atomicAdd(&s.mass[bin], w);
        atomicAdd(&s.cnt[bin], 1u);
        above(w);
      });
  return high;
}
// An addition to a histogram of digits; a wave whose lanes all have one digit makes one.
__device__ __forceinline__ void add_to(Digits& d, int at, bool weighs, u64 w) {
  if (__ballot(at == __builtin_amdgcn_readfirstlane(at)) == ~u64(0)) {
    const u64 sum = weighs ? wave_scan(w) : 0;
    if ((threadIdx.x & 63) == 63) {
      atomicAdd(&d.mass[at], sum);
      atomicAdd(&d.cnt[at], 64u);
    }
    return;
  }
  atomicAdd(&d.mass[at], w);
  atomicAdd(&d.cnt[at], 1u);
}

// What a workgroup keeps between its searches: which of the buffers comes next (one is cleared while the last one may
// still be read, so a search costs one barrier a step).
struct Turn {
  int digits = 0;
};

struct Found {
  u64 before, w;  // the weight before the token, and its own
  uint32_t idx;
};
__device__ __forceinline__ uint32_t lane_u32(uint32_t x, int lane) { return uint32_t(__builtin_amdgcn_readlane(int(x), lane)); }
__device__ __forceinline__ u64 lane_u64(u64 x, int lane) {
  return (u64(lane_u32(uint32_t(x >> 32), lane)) << 32) | lane_u32(uint32_t(x), lane);
}

// The first of the tokens that each(f) gives f(key, index, weight) of, at which the running count (by_count) or weight,
// `cnt0` and `mass0` before the first, passes `target`: by digits of 8 bits of the key, the largest first, until one token is
// left, then of the index, the smallest first. There are `c` of them of the weight `m`; their least and largest keys are
// `klo` and `khi` and differ from bit LOW on, indices are below `V`. Every thread is here; every wave has the result.
template <int LOW, int NT, typename S, typename Each>
__device__ __forceinline__ Found select(bool by_count, bool index, const Each& each, u64 target, u64 mass0, u64 cnt0, u64 m, uint32_t c, uint32_t klo,
                                        uint32_t khi, int V, S& s, Turn& turn) {
  const int tid = threadIdx.x, lane = tid & 63;
  auto above = [](int bit) { return bit >= 32 ? 0u : ~0u << bit; };
  int kbits = klo == khi ? LOW : max(32 - __builtin_clz(klo ^ khi), LOW), ibits = V > 1 ? 32 - __builtin_clz(uint32_t(V - 1)) : 0;
  const uint32_t last = (1u << ibits) - 1;  // the inverse of index 0
  uint32_t kmask = above(kbits), kp = khi & kmask, ip = 0, imask = 0;
  auto mine = [&](uint32_t key, uint32_t inv) { return ((key ^ kp) & kmask) == 0 && ((inv ^ ip) & imask) == 0; };
  bool weighs = true;
  while (c > 1 && (kbits > LOW || (index && ibits > 0))) {
    const bool on_key = kbits > LOW;
    if (!on_key && weighs) {  // equal logits: the token by its place among them
      weighs = false;
      by_count = true;
      target = (target - mass0) / (m / c);
      cnt0 = 0;
    }
    const int shift = on_key ? max(kbits - 8, LOW) : max(ibits - 8, 0), width = (on_key ? kbits : ibits) - shift;
    const uint32_t digits = (1u << width) - 1;
    Digits& now = s.dig[turn.digits % 3];
    Digits& next = s.dig[(turn.digits + 1) % 3];
    ++turn.digits;
    for (int i = tid; i < 256; i += NT) {
      next.mass[i] = 0;
      next.cnt[i] = 0;
    }
    each([&](uint32_t key, uint32_t idx, auto weight) {
      const uint32_t inv = last - idx;
      if (!mine(key, inv)) return;
      add_to(now, int(((on_key ? key : inv) >> shift) & digits), weighs, weighs ? weight() : 0);
    });
    __syncthreads();
    // lane l has digits 255 - 4 l and the three below it
    u64 dm[4], tm = 0;
    uint32_t dc[4], tc = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      dm[k] = now.mass[255 - 4 * lane - k];
      dc[k] = now.cnt[255 - 4 * lane - k];
      tm += dm[k];
      tc += dc[k];
    }
    u64 bm = mass0 + wave_scan(tm) - tm, bc = cnt0 + wave_scan(tc) - tc, hm = 0, hbm = 0, hbc = 0;
    uint32_t hc = 0, digit = 0;
    bool hit = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const u64 lo = by_count ? bc : bm, hi = lo + (by_count ? u64(dc[k]) : dm[k]);
      if (lo <= target && target < hi) {
        hit = true;
        digit = uint32_t(255 - 4 * lane - k);
        hm = dm[k]; hc = dc[k]; hbm = bm; hbc = bc;
      }
      bm += dm[k];
      bc += dc[k];
    }
    const int src = __ffsll(static_cast<u64>(__ballot(hit))) - 1;
    digit = lane_u32(digit, src);
    m = lane_u64(hm, src);
    c = lane_u32(hc, src);
    mass0 = lane_u64(hbm, src);
    cnt0 = lane_u64(hbc, src);
    if (on_key) {
      kbits = shift;
      kp |= digit << shift;
      kmask = above(kbits);
    } else {
      ibits = shift;
      ip |= digit << shift;
      imask = above(ibits) & last;
    }
  }
  if (!index) {  // of equal logits each has the same weight
    const u64 w = c == 1 ? m : m / c, place = c == 1 ? 0 : by_count ? target - cnt0 : (target - mass0) / w;
    return {mass0 + place * w, w, 0};
  }
  each([&](uint32_t key, uint32_t idx, auto) {
    if (mine(key, last - idx)) s.idx = idx;
  });
  __syncthreads();
  return {mass0, m, s.idx};
}

// The same by one wave where there are at most 64 tokens, the lane's own being (key, idx, w) where `in`: each counts the
// ones before it. MANY: four instructions a token make its place in `order`, 64 words of LDS, and a scan the sums; else
// the sums with the count, fifteen instructions and no scan (2000 of 131072 in 64 rows 44.4 us so, 43.1 by places; 1 x 271
// 5.5, 5.7).
template <bool MANY>
__device__ __forceinline__ Found select_wave(bool by_count, bool in, uint32_t key, uint32_t idx, u64 w, u64 target, u64 mass0,
                                             u64 cnt0, u64* order) {
  const int lane = threadIdx.x & 63;
  const int n = __popcll(__ballot(in));  // lanes 0 to n - 1
  if constexpr (MANY) {
    const u64 mine = (u64(key) << 32) | ~idx;
    int place = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) place += lane_u64(mine, j) > mine ? 1 : 0;
    if (in) order[place] = w;
    __builtin_amdgcn_wave_barrier();
    const u64 here = lane < n ? order[lane] : 0, upto = mass0 + wave_scan(here), before = upto - here;
    __builtin_amdgcn_wave_barrier();
    const bool hit = by_count ? u64(lane) == target - cnt0 : before <= target && target < upto;
    const int at = __ffsll(static_cast<u64>(__ballot(hit))) - 1;
    const int src = __ffsll(static_cast<u64>(__ballot(in && place == at))) - 1;
    return {lane_u64(before, at), lane_u64(here, at), lane_u32(idx, src)};
  } else {
    u64 mass = mass0;
    uint32_t cnt = uint32_t(cnt0);
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const uint32_t kj = lane_u32(key, j), ij = lane_u32(idx, j);
      const u64 wj = lane_u64(w, j);
      const bool before = kj > key || (kj == key && ij < idx);
      mass += before ? wj : 0;
      cnt += before ? 1u : 0u;
    }
    const u64 lo = by_count ? u64(cnt) : mass;
    const int src = __ffsll(static_cast<u64>(__ballot(in && lo <= target && target < lo + (by_count ? 1 : w)))) - 1;
    return {lane_u64(mass, src), lane_u64(w, src), lane_u32(idx, src)};
  }
}

// Prefix sums of the intervals in LDS, every BINS / 64-th of them in a wave's registers.
struct Interval {
  int bin;
  u64 mass0, mass1;  // the weight before it and up to its end
  uint32_t cnt0, cnt1;
};
template <int BINS>
struct Prefix {
  static constexpr int STEP = BINS / 64;
  const u64* mass;
  const uint32_t* cnt;
  u64 m;
  uint32_t c;
  __device__ __forceinline__ Prefix(const u64* mass_, const uint32_t* cnt_) : mass(mass_), cnt(cnt_) {
    const int i = int(threadIdx.x & 63) * STEP + STEP - 1;
    m = mass[i];
    c = cnt[i];
  }
  __device__ __forceinline__ u64 all() const { return lane_u64(m, 63); }
  // The interval in which the running count or weight passes `target` (below their sum): the first whose prefix sum is
  // larger, by two steps of 64. Every wave for itself, in scalar registers but for the comparisons.
  __device__ __forceinline__ Interval find(int stage, u64 target) const {
    const bool by_count = stage == 0;
    const int lane = threadIdx.x & 63;
    const int a = __ffsll(static_cast<u64>(__ballot(target < (by_count ? u64(c) : m)))) - 1;
    const int k = a * STEP + min(lane, STEP - 1);
    const u64 fm = mass[k];
    const uint32_t fc = cnt[k];
    const int f = __ffsll(static_cast<u64>(__ballot(target < (by_count ? u64(fc) : fm)))) - 1;
    Interval r;
    r.bin = a * STEP + f;
    r.mass1 = lane_u64(fm, f);
    r.cnt1 = lane_u32(fc, f);
    const int before = f > 0 ? f - 1 : a > 0 ? a - 1 : 0;
    r.mass0 = f > 0 ? lane_u64(fm, before) : a > 0 ? lane_u64(m, before) : 0;
    r.cnt0 = f > 0 ? lane_u32(fc, before) : a > 0 ? lane_u32(c, before) : 0;
    return r;
  }
};

template <int BINS>
__device__ __forceinline__ Plan plan_row(const Goals& goals, u64 high, const Prefix<BINS>& prefix) {
  Plan r{{0, 0, 0}, {-1, -1, -1}, 0};
  u64 lo = prefix.all(), hi = lo;  // the weight kept lies in [lo, hi]
#pragma unroll
  for (int stage = 0; stage < 3; ++stage) {
    if (!goals.has(stage)) continue;
    if (stage == 2) {
      lo = min(lo, high);
      hi = min(hi, high);
    }
    const u64 t0 = goals.target(stage, lo), t1 = goals.target(stage, hi);
    const Interval a = prefix.find(stage, t0), b = t1 == t0 ? a : prefix.find(stage, t1);
    lo = a.mass0;
    hi = b.mass1;
    if (stage == 0 && lo == hi) continue;  // of tokens without weight any number may go (top-k over masked ones)
    r.total += b.cnt1 - a.cnt0;
    r.from[stage] = a.bin;
    r.to[stage] = b.bin;
  }
  return r;
}

// The searches of a row: prefix sums in s, the tokens of its plan's intervals in the list (n of them), or FROM_ROW when
// they do not fit, then each(f) gives f(key, index, interval, weight) of every token of the row. dig[0] is clear. The
// first wave goes by itself, the others asleep at the barrier (all of them beside it: 1 x 8000 16.9 us, 14.0 so), as long as
// the intervals have at most 64 tokens; where one has more all go on from there.
template <bool FROM_ROW, bool MANY, int LOW, int NT, int BINS, typename S, typename Each>
__device__ __forceinline__ uint32_t resolve(const Goals& goals, const Prefix<BINS>& prefix, const Scale<BINS>& sc, u64 high, int n, int V,
                                            S& s, const Each& each) {
  const int lane = threadIdx.x & 63;
  u64 kept = prefix.all();
  uint32_t token = 0;
  int stage = 0;
  if constexpr (!FROM_ROW) {
    if (threadIdx.x < 64) {
#pragma unroll
      for (; stage < 3; ++stage) {
        if (!goals.has(stage)) continue;
        const u64 all = stage == 2 ? min(kept, high) : kept, target = goals.target(stage, all);
        const Interval at = prefix.find(stage, target);
        const int c = int(at.cnt1 - at.cnt0);
        if (stage < 2 && (c == 1 || at.mass1 == at.mass0)) {  // the token is the interval, or has no weight
          kept = at.mass1;
          continue;
        }
        if (c > 64) break;
        int have = 0;
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += 64) {  // where in the list the interval's tokens are
          const bool in = i0 + lane < n && s.lbin[min(i0 + lane, n - 1)] == at.bin;
          const u64 mask = __ballot(in);
          if (in) s.slot[have + __popcll(mask & ((u64(1) << lane) - 1))] = uint16_t(i0 + lane);
          have += __popcll(mask);
        }
        __builtin_amdgcn_wave_barrier();
        const int mine = lane < c ? s.slot[lane] : 0;
        __builtin_amdgcn_wave_barrier();
        const Found f = select_wave<MANY>(stage == 0, lane < c, s.lkey[mine], s.lidx[mine], s.lw[mine], target, at.mass0, at.cnt0, s.order);
        kept = f.before + f.w;
        token = f.idx;
      }
      if (lane == 0) {
        s.kept = kept;
        s.token = token;
        s.stage = stage;
      }
    }
    __syncthreads();
    if (threadIdx.x >= 64) {
      stage = s.stage;
      kept = s.kept;
      token = s.token;
    }
  }
  Turn turn;
#pragma unroll 1
  for (; stage < 3; ++stage) {
    if (!goals.has(stage)) continue;
    if (stage == 2) kept = min(kept, high);
    const u64 target = goals.target(stage, kept);
    const Interval at = prefix.find(stage, target);
    const uint32_t c = at.cnt1 - at.cnt0;
    if (stage < 2 && (c == 1 || at.mass1 == at.mass0)) {
      kept = at.mass1;
      continue;
    }
    auto of_bin = [&](auto g) {
      each([&](uint32_t k, uint32_t i, int bin, auto weight) {
        if (bin == at.bin) g(k, i, weight);
      });
    };
    uint32_t klo = ~0u, khi = 0;  // the keys there are: one where logits are equal
    of_bin([&](uint32_t k, uint32_t, auto) {
      klo = min(klo, k);
      khi = max(khi, k);
    });
    klo = ~wave_umax(~klo);
    khi = wave_umax(khi);
    __syncthreads();
    if (lane == 0) {
      s.red32[threadIdx.x >> 6] = khi;
      s.low32[threadIdx.x >> 6] = klo;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
      khi = max(khi, s.red32[w]);
      klo = min(klo, s.low32[w]);
    }
    const Found f = select<LOW, NT>(stage == 0, stage == 2, of_bin, target, at.mass0, at.cnt0, at.mass1 - at.mass0, c, klo, khi, V, s, turn);
    kept = f.before + f.w;
    token = f.idx;
  }
  return token;
}
template <typename T, bool MANY, int NT, int BINS, typename S>
__device__ __forceinline__ uint32_t resolve_list(const Goals& goals, const Prefix<BINS>& prefix, const Scale<BINS>& sc, u64 high, int n, int V, S& s) {
  return resolve<false, MANY, sizeof(T) == 2 ? 16 : 0, NT>(goals, prefix, sc, high, n, V, s, [&](auto f) {
    for (int i = threadIdx.x; i < n; i += NT) f(s.lkey[i], s.lidx[i], s.lbin[i], [&] { return s.lw[i]; });
  });
}
// (from memory, AHEAD loads at a time)
template <typename T, int AHEAD, int NT, int BINS, typename S>
__device__ __forceinline__ uint32_t resolve_row(const Goals& goals, const Prefix<BINS>& prefix, const Scale<BINS>& sc, u64 high,
                                                const T* logits, int V, S& s) {
  return resolve<true, true, sizeof(T) == 2 ? 16 : 0, NT>(goals, prefix, sc, high, 0, V, s, [&](auto f) {
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < V; i0 += AHEAD * NT) {
      float x[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) x[k] = Elem<T>::to_f(logits[min(i0 + k * NT, V - 1)]);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int i = i0 + k * NT;
        if (i < V) f(key_of(x[k]), uint32_t(i), sc.bin(x[k]), [&] { return sc.weight(x[k]); });
      }
    }
  });
}

// counts and weights of the intervals to their prefix sums, in place; a barrier ends it
template <int NT, int BINS, typename S>
__device__ __forceinline__ void scan_bins(S& s) {
  constexpr int N = BINS / NT;
  const int tid = threadIdx.x;
  u64 m[N], tm = 0;
  uint32_t c[N], tc = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    tm += s.mass[tid * N + i];
    tc += s.cnt[tid * N + i];
    m[i] = tm;
    c[i] = tc;
  }
  scan_block<NT>(tm, tc, s);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s.mass[tid * N + i] = m[i] + tm;
    s.cnt[tid * N + i] = c[i] + tc;
  }
  __syncthreads();
}

// the largest logit, the smallest finite one and whether there is a NaN, over the workgroup
template <int NT, typename S, typename Rows>
__device__ __forceinline__ void extremes(const Rows& row, float& top, float& low, bool& nan, S& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  top = kNegInf;
  low = __builtin_inff();
  nan = false;
  row.each([&](float x, int) {
    nan = nan || x != x;
    top = fmaxf(top, x);
    low = x > kNegInf ? fminf(low, x) : low;
  });
  top = wave_max(top);
  low = -wave_max(-low);
  nan = __ballot(nan) != 0;
  if (lane == 0) {
    s.redf[wave] = top;
    s.redm[wave] = low;
    s.red32[wave] = nan;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    top = fmaxf(top, s.redf[w]);
    low = fminf(low, s.redm[w]);
    nan = nan || s.red32[w];
  }
}

// ---- a workgroup a row -------------------------------------------------------------------------------------
template <typename T, int NT, int R, int BINS>
__global__ void __launch_bounds__(NT, 4) sample_kernel(const SampleParams p) {
  constexpr int LIST = BINS < kList ? BINS : kList;
  __shared__ Lds<BINS, LIST> s;
  const int tid = threadIdx.x, b = blockIdx.x;
  const Setting o(p, b);
  Row<T, NT, R> row;
  row.open(reinterpret_cast<const T*>(p.logits) + b * p.l_sr, 0, p.V);
  if (p.run && *p.run == 0) return;
#pragma unroll
  for (int i = 0; i < BINS / NT; ++i) {
    s.mass[tid + i * NT] = 0;
    s.cnt[tid + i * NT] = 0;
  }
  if (tid == 0) {
    s.high = 0;
    s.first = p.V;
  }
  float top, low;
  bool nan;
  extremes<NT>(row, top, low, nan, s);
  if (nan || top == kNegInf || o.nan()) {
    if (tid == 0) p.tokens[b] = -1;
    return;
  }
  if (o.greedy()) {
    row.each([&](float x, int i) {
      if (x == top) atomicMin(&s.first, uint32_t(i));
    });
    __syncthreads();
    if (tid == 0) p.tokens[b] = s.first;
    return;
  }
  const Scale<BINS> sc(o, top, low);
  const bool cut = o.min_p > 0.f;
  u64 high = histogram<BINS>(row, sc, o.min_p, s);
  if (cut) {
    high = wave_scan(high);
    if ((tid & 63) == 63) atomicAdd(&s.high, high);
  }
  __syncthreads();
  if (tid == 0) s.n = 0;
  for (int i = tid; i < 256; i += NT) {
    s.dig[0].mass[i] = 0;
    s.dig[0].cnt[i] = 0;
  }
  scan_bins<NT, BINS>(s);
  high = cut ? s.high : ~u64(0);
  const Goals goals(o, p.V);
  const Prefix<BINS> prefix(s.mass, s.cnt);
  if (tid < 64) {
    const Plan plan = plan_row(goals, high, prefix);
    if (tid == 0) s.plan = plan;
  }
  __syncthreads();
  const Plan plan = s.plan;
  uint32_t token;
  if (plan.total <= LIST) {
    row.each([&](float x, int i) {
      const int bin = sc.bin(x);
      if (!plan.has(bin)) return;
      const int at = atomicAdd(&s.n, 1u);
      s.lkey[at] = key_of(x);
      s.lidx[at] = i;
      s.lw[at] = sc.weight(x);
      s.lbin[at] = bin;
    });
    __syncthreads();
    token = resolve_list<T, (R > 2), NT>(goals, prefix, sc, high, int(s.n), p.V, s);
  } else {
    token = resolve_row<T, 1, NT>(goals, prefix, sc, high, row.p, p.V, s);
  }
  if (tid == 0) p.tokens[b] = token;
}

// ---- a row in pieces ---------------------------------------------------------------------------------------
constexpr int kPieceThreads = 512;
constexpr int kRowList = 2048;  // tokens of the intervals that a row's searches can end in
struct RowWs {                  // in the workspace: what a launch leaves for the next, and pieces for their row's last
  u64 mass[kBins];
  u64 high;
  uint32_t cnt[kBins];
  float top[kMaxPieces], low[kMaxPieces];
  uint32_t nan[kMaxPieces], first[kMaxPieces];
  uint32_t done, n;
  uint32_t key[kRowList], idx[kRowList];
};
// publish, then count: agent-scope stores and additions are acknowledged at the device-coherent level before the
// barrier, the count's addition is issued after it, and the workgroup that sees the last count reads with agent-scope
// loads. Every thread is here; the same answer for all.
__device__ __forceinline__ bool last_piece(RowWs& w, int pieces, int& flag) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) flag = __hip_atomic_fetch_add(&w.done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == uint32_t(pieces - 1);
  __syncthreads();
  return flag != 0;
}
template <typename N>
__device__ __forceinline__ N agent_load(const N* p) {
  return __hip_atomic_load(const_cast<N*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <typename T>
__global__ void __launch_bounds__(kPieceThreads) sample_top_kernel(const SampleParams p) {
  constexpr int NT = kPieceThreads;
  __shared__ struct {
    float redf[16], redm[16];
    uint32_t red32[16], first;
  } s;
  const int tid = threadIdx.x, b = blockIdx.x / p.pieces, g = blockIdx.x % p.pieces;
  RowWs& w = reinterpret_cast<RowWs*>(p.ws)[b];
  Row<T, NT, 0> row;
  row.open(reinterpret_cast<const T*>(p.logits) + b * p.l_sr, g * p.piece, min(p.V, (g + 1) * p.piece));
  if (p.run && *p.run == 0) return;
  for (int i = g * NT + tid; i < kBins; i += p.pieces * NT) {
    w.mass[i] = 0;
    w.cnt[i] = 0;
  }
  if (tid == 0) s.first = p.V;
  float top, low;
  bool nan;
  extremes<NT>(row, top, low, nan, s);
  const Setting o(p, b);
  if (o.greedy()) {
    row.each([&](float x, int i) {
      if (x == top) atomicMin(&s.first, uint32_t(i));
    });
    __syncthreads();
  }
  if (tid == 0) {
    w.top[g] = top;
    w.low[g] = low;
    w.nan[g] = nan;
    w.first[g] = s.first;
    if (g == 0) {
      w.high = 0;
      w.done = 0;
      w.n = 0;
    }
  }
}

// a row's extremes from its pieces' (every lane of every wave), and the token where there is nothing to search
struct Whole {
  float top, low;
  bool over;
  int64_t token;
};
__device__ __forceinline__ Whole whole_row(const RowWs& w, const SampleParams& p, const Setting& o) {
  const int lane = threadIdx.x & 63;
  const bool in = lane < p.pieces;
  Whole r;
  const float mine = in ? w.top[lane] : kNegInf;
  r.top = wave_max(mine);
  r.low = -wave_max(in ? -w.low[lane] : kNegInf);
  const bool nan = __ballot(in && w.nan[lane]) != 0 || r.top == kNegInf || o.nan();
  r.over = nan || o.greedy();
  r.token = -1;
  if (!nan && o.greedy()) {
    const uint64_t has = __ballot(in && mine == r.top);
    r.token = w.first[__ffsll(static_cast<unsigned long long>(has)) - 1];
  }
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kPieceThreads, 4) sample_hist_kernel(const SampleParams p) {
  constexpr int NT = kPieceThreads;
  __shared__ struct {
    u64 mass[kBins];
    uint32_t cnt[kBins];
    u64 red64[16];
    uint32_t red32[16];
  } s;
  const int tid = threadIdx.x, b = blockIdx.x / p.pieces, g = blockIdx.x % p.pieces;
  Row<T, NT, 0> row;
  row.open(reinterpret_cast<const T*>(p.logits) + b * p.l_sr, g * p.piece, min(p.V, (g + 1) * p.piece));
  if (p.run && *p.run == 0) return;
  RowWs& w = reinterpret_cast<RowWs*>(p.ws)[b];
  const Setting o(p, b);
  const Whole all = whole_row(w, p, o);
  if (all.over) {
    if (g == 0 && tid == 0) p.tokens[b] = all.token;
    return;
  }
#pragma unroll
  for (int i = 0; i < kBins / NT; ++i) {
    s.mass[tid + i * NT] = 0;
    s.cnt[tid + i * NT] = 0;
  }
  __syncthreads();
  const Scale<kBins> sc(o, all.top, all.low);
  u64 high = histogram<kBins>(row, sc, o.min_p, s);
  if (o.min_p > 0.f) {
    high = wave_scan(high);
    if ((tid & 63) == 63 && high) __hip_atomic_fetch_add(&w.high, high, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBins / NT; ++i) {
    const int k = tid + i * NT;
    if (s.cnt[k]) __hip_atomic_fetch_add(&w.cnt[k], s.cnt[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (s.mass[k]) __hip_atomic_fetch_add(&w.mass[k], s.mass[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

template <typename T>
__global__ void __launch_bounds__(kPieceThreads, 4) sample_pick_kernel(const SampleParams p) {
  constexpr int NT = kPieceThreads;
  __shared__ Lds<kBins, kRowList> s;
  const int tid = threadIdx.x, b = blockIdx.x / p.pieces, g = blockIdx.x % p.pieces;
  const T* logits = reinterpret_cast<const T*>(p.logits) + b * p.l_sr;
  Row<T, NT, 0> row;
  row.open(logits, g * p.piece, min(p.V, (g + 1) * p.piece));
  RowWs& w = reinterpret_cast<RowWs*>(p.ws)[b];
  u64 m[kBins / NT];
  uint32_t c[kBins / NT];
#pragma unroll
  for (int i = 0; i < kBins / NT; ++i) {
    m[i] = w.mass[tid + i * NT];
    c[i] = w.cnt[tid + i * NT];
  }
  if (p.run && *p.run == 0) return;
  const Setting o(p, b);
  const Whole all = whole_row(w, p, o);
  if (all.over) return;
#pragma unroll
  for (int i = 0; i < kBins / NT; ++i) {
    s.mass[tid + i * NT] = m[i];
    s.cnt[tid + i * NT] = c[i];
  }
  for (int i = tid; i < 256; i += NT) {
    s.dig[0].mass[i] = 0;
    s.dig[0].cnt[i] = 0;
  }
  if (tid == 0) s.n = 0;
  const u64 high = o.min_p > 0.f ? w.high : ~u64(0);
  const Goals goals(o, p.V);
  __syncthreads();
  scan_bins<NT, kBins>(s);
  const Prefix<kBins> prefix(s.mass, s.cnt);
  if (tid < 64) {
    const Plan plan = plan_row(goals, high, prefix);
    if (tid == 0) s.plan = plan;
  }
  __syncthreads();
  const Plan plan = s.plan;
  const bool fits = plan.total <= kRowList;
  const Scale<kBins> sc(o, all.top, all.low);
  if (fits) {
    float l0, h0, l1, h1, l2, h2;
    const float width = 1.0f / sc.per;
    sc.reach(plan.from[0], plan.to[0], width, l0, h0);
    sc.reach(plan.from[1], plan.to[1], width, l1, h1);
    sc.reach(plan.from[2], plan.to[2], width, l2, h2);
    row.each([&](float x, int i) {
      // six comparisons for nearly all; the interval is for the few
      if (!(((x >= l0) & (x <= h0)) | ((x >= l1) & (x <= h1)) | ((x >= l2) & (x <= h2)))) return;
      if (!plan.has(sc.bin(x))) return;
      const int at = atomicAdd(&s.n, 1u);
      s.lkey[at] = key_of(x);
      s.lidx[at] = i;
    });
    __syncthreads();
    const uint32_t n = s.n;
    if (tid == 0 && n) s.first = __hip_atomic_fetch_add(&w.n, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    for (uint32_t i = tid; i < n; i += NT) {
      __hip_atomic_store(&w.key[s.first + i], s.lkey[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(&w.idx[s.first + i], s.lidx[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (!last_piece(w, p.pieces, s.last)) return;

  // ---- the row's last piece: the searches ----
  uint32_t token;
  if (fits) {
    const int n = int(agent_load(&w.n));
    for (int i = tid; i < n; i += NT) {
      const uint32_t k = agent_load(&w.key[i]), idx = agent_load(&w.idx[i]);
      const float x = of_key(k);
      s.lkey[i] = k;
      s.lidx[i] = idx;
      s.lw[i] = sc.weight(x);
      s.lbin[i] = sc.bin(x);
    }
    __syncthreads();
    token = resolve_list<T, true, NT>(goals, prefix, sc, high, n, p.V, s);
  } else {
    token = resolve_row<T, 8, NT>(goals, prefix, sc, high, logits, p.V, s);
  }
  if (tid == 0) p.tokens[b] = token;
}

constexpr int kWholeRow = 8192;  // longer rows go in pieces

// Pieces of a row: a workgroup a CU over the batch, two where a piece would be over 16384 logits, of at least 4096 (64 x
// 131072 in bf16 in 4, 8 pieces 46.4, 45.0 us; 1 x 131072 in fp32 in 32, 64 pieces 22.0, 24.6; 1 x 32000 in 3, 7, 15
// 23.1, 19.5, 18.9, 16 x 32000 in 3, 7, 15 24.6, 22.1, 23.4).
static int pieces_of(int B, int V) {
  if (V <= kWholeRow) return 1;
  int64_t n = std::max<int64_t>(device_cu_count() / B, 1);
  if (V / n > 16384) n *= 2;
  n = std::min<int64_t>(n, V / 4096);
  return int(std::max<int64_t>(2, std::min<int64_t>(n, kMaxPieces)));
}

size_t sample_workspace_bytes(const mote_sample_args* a) {
  return a->B > 0 && a->V > kWholeRow ? size_t(a->B) * sizeof(RowWs) : 0;
}

int launch_sample(const mote_sample_args* a, hipStream_t stream) {
  const char* what = "sample";
  if (!a) return set_error(MOTE_ERR_ARGUMENT, "%s: null args", what);
  if (a->dtype != MOTE_F32 && a->dtype != MOTE_BF16) return set_error(MOTE_ERR_ARGUMENT, "%s: bad dtype %d", what, a->dtype);
  if (a->B < 0 || a->V < 1 || a->V > (1 << 20))
    return set_error(MOTE_ERR_SHAPE, "%s: %d rows of %d logits (1 to 2^20 a row)", what, a->B, a->V);
  if (a->B == 0) return MOTE_OK;
  if (!a->logits || !a->u || !a->tokens) return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  SampleParams p{};
  p.logits = a->logits; p.l_sr = a->l_sr; p.u = a->u;
  p.temperature = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p; p.top_k = a->top_k;
  p.temperature_dev = a->temperature_dev; p.top_p_dev = a->top_p_dev; p.min_p_dev = a->min_p_dev; p.top_k_dev = a->top_k_dev;
  p.tokens = a->tokens; p.run = a->run; p.V = a->V;
  p.pieces = pieces_of(a->B, a->V);
  if (!grid_fits(int64_t(a->B) * p.pieces, 1024)) return set_error(MOTE_ERR_SHAPE, "%s: %d rows are too many for one launch", what, a->B);
  if (p.pieces > 1) {
    const size_t need = sample_workspace_bytes(a);
    if (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16)
      return set_error(MOTE_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes, %zu needed", what, a->workspace_bytes, need);
    p.ws = reinterpret_cast<char*>(a->workspace);
    p.piece = ((a->V + p.pieces - 1) / p.pieces + 7) / 8 * 8;
    p.pieces = (a->V + p.piece - 1) / p.piece;
    const dim3 grid(unsigned(a->B) * p.pieces), block(kPieceThreads);
    const bool draws = a->temperature_dev || a->temperature > 0.f;  // else the second launch has every token
    auto launch = [&](auto t) {
      using T = decltype(t);
      hipLaunchKernelGGL((sample_top_kernel<T>), grid, block, 0, stream, p);
      hipLaunchKernelGGL((sample_hist_kernel<T>), grid, block, 0, stream, p);
      if (draws) hipLaunchKernelGGL((sample_pick_kernel<T>), grid, block, 0, stream, p);
    };
    if (a->dtype == MOTE_BF16) launch(bf16_t{});
    else launch(0.f);
    return check_launch(what);
  }
#define MOTE_SAMPLE(NT_, R_, BINS_) hipLaunchKernelGGL((sample_kernel<T, NT_, R_, BINS_>), dim3(a->B), dim3(NT_), 0, stream, p)
  // few waves a row: their barriers and scans are its chain (16 x 2900 with 16 waves 12.0 us, 8 waves 10.8). Beyond 4096
  // logits 16 waves are as fast while every row has a CU, two rows of 8 a CU when it has not (1 x 8000 15.1 and 15.6 us,
  // 300 x 8000 28.7 and 20.6).
  const bool crowded = a->B > device_cu_count();
#define MOTE_SAMPLE_V                               \
  if (a->V <= 512) MOTE_SAMPLE(256, 2, 512);        \
  else if (a->V <= 1024) MOTE_SAMPLE(512, 2, 1024); \
  else if (a->V <= 4096) MOTE_SAMPLE(512, 8, 1024); \
  else if (crowded) MOTE_SAMPLE(512, 16, 1024);     \
  else MOTE_SAMPLE(1024, 8, 2048);
  if (a->dtype == MOTE_BF16) {
    using T = bf16_t;
    MOTE_SAMPLE_V
  } else {
    using T = float;
    MOTE_SAMPLE_V
  }
#undef MOTE_SAMPLE_V
#undef MOTE_SAMPLE
  return check_launch(what);
}

}  // namespace mote
