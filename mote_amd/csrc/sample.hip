// The next token of every row of logits from one random number (mote_sample; mote_relation.h has the definition).
//
// Every step of it is one search: tokens in the order of their logits (ties to the lowest index), find the first
// at which a running sum passes a target. Top-k asks for the weight of the first k (the sum counts), top-p for the
// weight up to the token at which p of that is reached, the draw for the token at which u of the weight kept is
// passed; min-p is a sum over the row. Nothing is sorted. Weights are fixed-point numbers of 2^-43 of the largest,
// rounded from an fp64 exponential, in 64 bits: sums of up to 2^20 of them are exact, so their order does not matter
// and atomics may make them, and a border differs from the real one by 2^-33 of the largest weight at most.
//
// A row: its maximum; a histogram over 2048 intervals of the logit (an interval's count and weight); its prefix
// sums, in which a search finds an interval; the interval's tokens gathered in LDS, where each counts the ones before
// it. An interval of more tokens than LDS holds (many equal logits) is searched by the digits of its keys instead.
#include <algorithm>

#include "common.hpp"
#include "device.hpp"
#include "params.hpp"
#include "stream.hpp"

namespace mote {

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
};

typedef unsigned long long u64;
constexpr int kBins = 2048;
constexpr int kList = 1024;                      // tokens of an interval that are searched in LDS
constexpr double kOne = 8796093022208.0;         // 2^43: the largest weight
constexpr float kReach = 31.0f;                  // exp(-31) < 2^-44: no weight from there on

// order of logits: a larger key comes first (the sum with +0 makes one zero of two)
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}

template <int NT>
struct Lds {
  u64 mass[kBins];  // prefix sums once scanned
  uint32_t cnt[kBins];
  u64 lw[kList];
  uint32_t lkey[kList], lidx[kList];
  u64 red64[16];
  uint32_t red32[16];
  float redf[16], redm[16];
  int redi[16];
  u64 out_before, out_w;
  uint32_t out_idx, n;
  int nan;
};

// exclusive prefix over the workgroup's threads
template <int NT>
__device__ __forceinline__ void scan_block(u64& m, uint32_t& c, Lds<NT>& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 m0 = m;
  const uint32_t c0 = c;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64 mm = __shfl_up(m, d);
    const uint32_t cc = __shfl_up(c, d);
    if (lane >= d) {
      m += mm;
      c += cc;
    }
  }
  __syncthreads();
  if (lane == 63) {
    s.red64[wave] = m;
    s.red32[wave] = c;
  }
  __syncthreads();
  m -= m0;
  c -= c0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) {
      m += s.red64[w];
      c += s.red32[w];
    }
  }
}

// R > 0: a thread holds elements tid + r NT of the row; R == 0: the row is read again each time
template <typename T, int NT, int R>
struct Row {
  const T* p;
  int V;
  float x[R > 0 ? R : 1];
  __device__ __forceinline__ void open(const T* row, int v) {
    p = row;
    V = v;
    if constexpr (R > 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int i = int(threadIdx.x) + r * NT;
        x[r] = i < V ? Elem<T>::to_f(p[i]) : 0.f;
      }
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if constexpr (R > 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int i = int(threadIdx.x) + r * NT;
        if (i < V) f(x[r], i);
      }
    } else {
      constexpr int PER = 16 / int(sizeof(T));
      const int whole = V / PER;
      for (int c = threadIdx.x; c < whole; c += NT) {
        const Chunk q = load_any(p + c * PER);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          float v;
          if constexpr (sizeof(T) == 2) v = __uint_as_float(k % 2 ? q.w[k / 2] & 0xffff0000u : q.w[k / 2] << 16);
          else v = __uint_as_float(q.w[k]);
          f(v, c * PER + k);
        }
      }
      for (int i = whole * PER + int(threadIdx.x); i < V; i += NT) f(Elem<T>::to_f(p[i]), i);
    }
  }
};

struct Scale {
  float top;       // the largest logit
  float per;       // intervals per unit of the logit
  double inv_t;
  __device__ __forceinline__ int bin(float x) const {
    if (x == top) return 0;
    const float t = (top - x) * per;  // inf where the logit or the largest one is infinite
    return t < float(kBins - 1) ? int(t) : kBins - 1;
  }
  __device__ __forceinline__ double weight(float x) const {
    const double d = double(x) - double(top);
    return x == top ? 1.0 : d > -__builtin_inf() ? exp(d * inv_t) : 0.0;
  }
  __device__ __forceinline__ u64 fixed(double w) const { return u64(w * kOne + 0.5); }
};

// The first token at which the running count (COUNT) or weight passes `target`: its index, its weight and the weight
// before it into s.out_*. The prefix sums stand in s; every thread is here, and a barrier ends it.
template <bool COUNT, typename T, int NT, int R>
__device__ void cross(const Row<T, NT, R>& row, const Scale& sc, u64 target, Lds<NT>& s) {
  const int tid = threadIdx.x;
  // the interval
  if (tid == 0) s.n = 0;
#pragma unroll
  for (int i = 0; i < kBins / NT; ++i) {
    const int b = tid + i * NT;
    const u64 hi = COUNT ? u64(s.cnt[b]) : s.mass[b];
    const u64 lo = b == 0 ? 0 : COUNT ? u64(s.cnt[b - 1]) : s.mass[b - 1];
    if (lo <= target && target < hi) s.out_idx = b;
  }
  __syncthreads();
  const int bin = int(s.out_idx);
  u64 mass0 = bin == 0 ? 0 : s.mass[bin - 1];
  u64 cnt0 = bin == 0 ? 0 : s.cnt[bin - 1];
  const int n = int(s.cnt[bin] - cnt0);
  if (n <= kList) {
    row.each([&](float x, int i) {
      if (sc.bin(x) != bin) return;
      const int at = atomicAdd(&s.n, 1u);
      s.lkey[at] = key_of(x);
      s.lidx[at] = i;
      s.lw[at] = sc.fixed(sc.weight(x));
    });
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const uint32_t k = s.lkey[i], id = s.lidx[i];
      u64 mass = mass0, cnt = cnt0;
      for (int j = 0; j < n; ++j) {
        const uint32_t kj = s.lkey[j];
        if (kj > k || (kj == k && s.lidx[j] < id)) {
          mass += s.lw[j];
          ++cnt;
        }
      }
      const u64 before = COUNT ? cnt : mass;
      if (before <= target && target < before + (COUNT ? 1 : s.lw[i])) {
        s.out_before = mass;
        s.out_w = s.lw[i];
        s.out_idx = id;
      }
    }
    __syncthreads();
    return;
  }
  // by digits of 8 bits of the key, the list's memory as their histogram (256 digits, the largest first)
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += NT) {
      s.lw[i] = 0;
      s.lidx[i] = 0;
    }
    __syncthreads();
    row.each([&](float x, int) {
      const uint32_t k = key_of(x);
      if (sc.bin(x) != bin || (shift < 24 && (k ^ prefix) >> (shift + 8))) return;
      const int d = int((k >> shift) & 255u);
      atomicAdd(&s.lw[d], sc.fixed(sc.weight(x)));
      atomicAdd(&s.lidx[d], 1u);
    });
    __syncthreads();
    if (tid == 0) {
      for (int d = 255; d >= 0; --d) {
        const u64 m = s.lw[d], c = s.lidx[d];
        if (target < (COUNT ? cnt0 + c : mass0 + m)) {
          s.out_before = mass0;
          s.out_w = cnt0;
          s.out_idx = uint32_t(d);
          break;
        }
        mass0 += m;
        cnt0 += c;
      }
    }
    __syncthreads();
    mass0 = s.out_before;
    cnt0 = s.out_w;
    prefix |= s.out_idx << shift;
    __syncthreads();
  }
  // tokens of one logit: the one that many places on, in the order of their indices
  const float x = __uint_as_float(prefix & 0x80000000u ? prefix ^ 0x80000000u : ~prefix);
  const u64 w = sc.fixed(sc.weight(x));
  const u64 place = COUNT ? target - cnt0 : (target - mass0) / w;
  const int per = (row.V + NT - 1) / NT, i0 = min(tid * per, row.V), i1 = min(i0 + per, row.V);
  uint32_t mine = 0;
  for (int i = i0; i < i1; ++i) mine += key_of(Elem<T>::to_f(row.p[i])) == prefix;
  u64 unused = 0;
  uint32_t before = mine;
  scan_block<NT>(unused, before, s);
  if (before <= place && place < before + mine) {
    uint32_t at = before;
    for (int i = i0; i < i1; ++i) {
      if (key_of(Elem<T>::to_f(row.p[i])) != prefix) continue;
      if (at++ == place) {
        s.out_before = mass0 + place * w;
        s.out_w = w;
        s.out_idx = uint32_t(i);
        break;
      }
    }
  }
  __syncthreads();
}

template <typename T, int NT, int R>
__global__ void __launch_bounds__(NT) sample_kernel(const SampleParams p) {
  __shared__ Lds<NT> s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
  if (p.run && *p.run == 0) return;
  Row<T, NT, R> row;
  row.open(reinterpret_cast<const T*>(p.logits) + b * p.l_sr, p.V);
  const float temperature = p.temperature_dev ? p.temperature_dev[b] : p.temperature;
  const float top_p = p.top_p_dev ? p.top_p_dev[b] : p.top_p;
  const float min_p = p.min_p_dev ? p.min_p_dev[b] : p.min_p;
  const int64_t top_k = p.top_k_dev ? p.top_k_dev[b] : p.top_k;
  const float u = p.u[b];

  // the largest logit, the first token that has it, the smallest finite one
  float top = kNegInf, low = __builtin_inff();
  int first = p.V;
  bool nan = false;
  row.each([&](float x, int i) {
    nan = nan || x != x;
    if (x > top || (x == top && i < first)) {
      top = x;
      first = i;
    }
    if (x > kNegInf) low = fminf(low, x);
  });
  auto best = [&](float t, int f) {
    if (t > top || (t == top && f < first)) {
      top = t;
      first = f;
    }
  };
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const float t = __shfl_xor(top, d);
    const int f = __shfl_xor(first, d);
    best(t, f);
    low = fminf(low, __shfl_xor(low, d));
  }
  if (tid == 0) s.nan = 0;
  __syncthreads();
  if (__ballot(nan) && lane == 0) s.nan = 1;
  if (lane == 0) {
    s.redf[wave] = top;
    s.redi[wave] = first;
    s.redm[wave] = low;
  }
#pragma unroll
  for (int i = 0; i < kBins / NT; ++i) {
    s.mass[tid + i * NT] = 0;
    s.cnt[tid + i * NT] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    best(s.redf[w], s.redi[w]);
    low = fminf(low, s.redm[w]);
  }
  const bool bad = s.nan || top == kNegInf || u != u || temperature != temperature || top_p != top_p || min_p != min_p;
  if (bad || !(temperature > 0.f)) {  // nothing to draw from, or the first of the order
    if (tid == 0) p.tokens[b] = bad ? -1 : first;
    return;
  }

  Scale sc;
  sc.top = top;
  sc.inv_t = 1.0 / double(temperature);
  const float span = fminf(kReach * temperature, top - low);  // at most as far as weights reach
  sc.per = span > 0.f ? float(kBins) / span : 0.f;
  if (!(sc.per < __builtin_inff())) sc.per = 3e38f;  // a span below the normal numbers
  const double floor_p = fminf(min_p, 1.f);
  u64 high = 0;
  row.each([&](float x, int) {
    const double w = sc.weight(x);
    const u64 f = sc.fixed(w);
    const int bin = sc.bin(x);
    if (f) atomicAdd(&s.mass[bin], f);
    atomicAdd(&s.cnt[bin], 1u);
    if (w >= floor_p) high += f;
  });
  __syncthreads();
  {  // prefix sums, in place
    constexpr int N = kBins / NT;
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
    u64 all = high;
    uint32_t unused = 0;
    scan_block<NT>(all, unused, s);
    if (tid == NT - 1) s.lw[0] = all + high;
    __syncthreads();
    high = s.lw[0];
    __syncthreads();
  }
  u64 kept = s.mass[kBins - 1];
  if (top_k > 0 && top_k < p.V) {
    cross<true>(row, sc, u64(top_k - 1), s);
    kept = s.out_before + s.out_w;
    __syncthreads();
  }
  if (top_p < 1.f) {
    // the first token at which the running weight reaches p kept, a whole number at or above it
    const u64 pf = u64(fmaxf(top_p, 0.f) * 18446744073709551616.0);  // exact: p in units of 2^-64
    const u64 want = __umul64hi(pf, kept) + (pf * kept != 0);
    cross<false>(row, sc, want > 0 ? want - 1 : 0, s);
    kept = s.out_before + s.out_w;
    __syncthreads();
  }
  kept = min(kept, high);
  const float uc = fminf(fmaxf(u, 0.f), 0x1.fffffep-1f);
  cross<false>(row, sc, __umul64hi(u64(double(uc) * 18446744073709551616.0), kept), s);
  if (tid == 0) p.tokens[b] = s.out_idx;
}

int launch_sample(const mote_sample_args* a, hipStream_t stream) {
  const char* what = "sample";
  if (!a) return set_error(MOTE_ERR_ARGUMENT, "%s: null args", what);
  if (a->dtype != MOTE_F32 && a->dtype != MOTE_BF16) return set_error(MOTE_ERR_ARGUMENT, "%s: bad dtype %d", what, a->dtype);
  if (a->B < 0 || a->V < 1 || a->V > (1 << 20))
    return set_error(MOTE_ERR_SHAPE, "%s: %d rows of %d logits (1 to 2^20 a row)", what, a->B, a->V);
  if (a->B == 0) return MOTE_OK;
  if (!a->logits || !a->u || !a->tokens) return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  if (!grid_fits(a->B, 1024)) return set_error(MOTE_ERR_SHAPE, "%s: %d rows are too many for one launch", what, a->B);
  SampleParams p;
  p.logits = a->logits; p.l_sr = a->l_sr; p.u = a->u;
  p.temperature = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p; p.top_k = a->top_k;
  p.temperature_dev = a->temperature_dev; p.top_p_dev = a->top_p_dev; p.min_p_dev = a->min_p_dev; p.top_k_dev = a->top_k_dev;
  p.tokens = a->tokens; p.run = a->run; p.V = a->V;
#define MOTE_SAMPLE(NT_, R_) hipLaunchKernelGGL((sample_kernel<T, NT_, R_>), dim3(a->B), dim3(NT_), 0, stream, p)
#define MOTE_SAMPLE_V                            \
  if (a->V <= 512) MOTE_SAMPLE(512, 1);          \
  else if (a->V <= 1024) MOTE_SAMPLE(1024, 1);   \
  else if (a->V <= 8192) MOTE_SAMPLE(1024, 8);   \
  else if (a->V <= 32768) MOTE_SAMPLE(1024, 32); \
  else MOTE_SAMPLE(1024, 0);
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
