// Rows of the {P2, I~} cache in 4 bits: written from a prompt's projections, read back for the prefix
// attention (mote_cache4_write / mote_cache4_read; the format stands in mote_relation.h).
//
// Both are one pass over memory, bound by it: 2 D e bytes a row and head on the wide side, D + 4 G on the
// narrow one. Wide accesses are 16 bytes a lane. A writing thread holds one octet (eight values) of P2 and of
// I~, and a group's maximum is two DPP steps over its quad; a reading one a 16-byte chunk of either. What a value
// costs in instructions counts beside the bytes: positions by 32-bit sums instead of divisions (8 x 4984 rows of
// 8 x 96, bf16, 156 MB: write 35.7 -> 33.8 us), scales without divisions and no clamps (-> 31.2 us, 5.0 TB/s).
// Values read back pass the caches by (4407 rows, 17 MB: 6.5 -> 5.5 us, 4.8 with the 32-bit positions; 8 x 4984
// rows 26.6 -> 24.8 us, 6.3 TB/s).
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "params.hpp"
#include "fp4.hpp"

namespace mote {

struct Rows4Params {
  char* x[2];      // p2, info (T elements)
  int64_t x_sb[2], x_sh[2], x_sr[2];
  uint8_t* code[2];
  bf16_t* scale[2];
  int64_t c_sb, c_sh, s_sb, s_sh;
  int64_t start;
  const int64_t* start_dev;
  const int64_t* lens;
  int T, D, G, cap;
  uint32_t over_mul, over_shift;  // n over_mul / 2^over_shift = n / (chunks of a row), n < 2^31 (reads)
};

constexpr int kRows4Threads = 256;
constexpr int kMaxGrid4 = 65535;  // of a grid's second and third dimensions: heads, sequences of a launch

// n / G for the 1 to 4 groups of a row and n < 2^30
__device__ __forceinline__ uint32_t over_groups4(uint32_t n, int G) {
  return G == 3 ? __umulhi(n, 0x55555556u) : n >> (G >> 1);
}

// the (sequence, head) of the workgroup and this thread's (row, octet) in it
struct Rows4At {
  int b, h, t, o;
  bool in;
};
__device__ __forceinline__ Rows4At rows4_at(const Rows4Params& p) {
  Rows4At a;
  a.b = blockIdx.z;
  a.h = blockIdx.y;
  const uint32_t i = blockIdx.x * kRows4Threads + threadIdx.x;
  a.t = int(over_groups4(i >> 2, p.G));
  a.o = int(i - uint32_t(a.t) * (4 * p.G));
  a.in = a.t < p.T;
  return a;
}

template <typename T, bool STREAM>
__global__ void __launch_bounds__(kRows4Threads) cache4_write_kernel(const Rows4Params p) {
  const Rows4At a = rows4_at(p);
  const int64_t len = p.lens ? p.lens[a.b] : p.T;
  const int64_t row = (p.start_dev ? p.start_dev[a.b] : p.start) + a.t;
  // quads are whole (4 G octets a row): a row is written by all of its lanes or by none
  if (!a.in || a.t >= len || row < 0 || row >= p.cap) return;
  // the octets past the head dim hold its last one, of the same group, and store zeros
  const bool pad = 8 * a.o >= p.D;
  float x[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    load_octet<STREAM>(reinterpret_cast<const T*>(p.x[k]) + a.b * p.x_sb[k] + a.h * p.x_sh[k] + a.t * p.x_sr[k] +
                       (pad ? p.D - 8 : 8 * a.o), x[k]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    bf16_t s;
    const uint32_t w = encode4(x[k], s);
    *reinterpret_cast<uint32_t*>(p.code[k] + a.b * p.c_sb + a.h * p.c_sh + row * (16 * p.G) + 4 * a.o) = pad ? 0u : w;
    if ((a.o & 3) == 0) p.scale[k][a.b * p.s_sb + a.h * p.s_sh + row * p.G + (a.o >> 2)] = s;
  }
}

// A thread per 16-byte chunk of the rows, in memory order, so that a store writes whole lines where rows follow
// each other. Past the caches, lines written in parts cost twice their time: with an octet of fp32 a thread, stored
// in halves, 9 x 1144 rows of head dim 128 (84 MB) took 31.6 us, now 15.9; with whole groups and idle threads past
// the head dim 4 x 3001 rows of 120 24.1, now 15.0. (Writing fp32 rows so as well, eight lanes a group: 118 MB
// 31.0 -> 29.8 us, but 3 MB 3.6 -> 3.9.)
template <typename T>
__global__ void __launch_bounds__(kRows4Threads) cache4_read_kernel(const Rows4Params p) {
  constexpr int EPC = 16 / int(sizeof(T));
  const uint32_t i = blockIdx.x * kRows4Threads + threadIdx.x;
  const int t = int(uint64_t(i) * p.over_mul >> p.over_shift);
  const int c = int(i) - t * (p.D / EPC);
  const int b = blockIdx.z, h = blockIdx.y;
  if (t >= p.T) return;
  const int64_t row = (p.start_dev ? p.start_dev[b] : p.start) + t;
  const bool held = row >= 0 && row < p.cap;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint32_t w = 0;
    float s = __builtin_nanf("");
    if (held) {
      using Codes = std::conditional_t<EPC == 8, uint32_t, uint16_t>;
      w = *reinterpret_cast<const Codes*>(p.code[k] + b * p.c_sb + h * p.c_sh + row * (16 * p.G) + EPC / 2 * c);
      s = bf2f(p.scale[k][b * p.s_sb + h * p.s_sh + row * p.G + c / (kGroup4 / EPC)]);
    }
    float x[8];
    decode4(w, s, x);
    Chunk v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (EPC == 8) v.w[j] = uint32_t(f2bf(x[2 * j])) | uint32_t(f2bf(x[2 * j + 1])) << 16;
      else v.w[j] = __float_as_uint(x[j]);
    }
    store_stream(reinterpret_cast<T*>(p.x[k]) + b * p.x_sb[k] + h * p.x_sh[k] + t * p.x_sr[k] + EPC * c, v);
  }
}

static int check_rows4(const mote_cache4_rows_args* a, const char* what) {
  if (!a) return set_error(MOTE_ERR_ARGUMENT, "%s: null args", what);
  if (a->dtype != MOTE_F32 && a->dtype != MOTE_BF16) return set_error(MOTE_ERR_ARGUMENT, "%s: bad dtype %d", what, a->dtype);
  if (a->D <= 0 || a->D > 128 || a->D % 8)
    return set_error(MOTE_ERR_SHAPE, "%s: head dim %d unsupported (need 8 <= D <= 128, D %% 8 == 0)", what, a->D);
  if (a->B < 0 || a->H < 0 || a->T < 0 || a->capacity <= 0) return set_error(MOTE_ERR_SHAPE, "%s: bad sizes", what);
  if (a->B == 0 || a->H == 0 || a->T == 0) return MOTE_OK;
  if (!a->p2.data || !a->info.data) return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  if (const char* bad = bad_cache4(a->cache)) return set_error(MOTE_ERR_ARGUMENT, "%s: %s", what, bad);
  const int64_t epc = a->dtype == MOTE_BF16 ? 8 : 4;
  for (const mote_view* v : {&a->p2, &a->info})
    if (reinterpret_cast<uintptr_t>(v->data) % 16 || v->stride_b % epc || v->stride_h % epc || v->stride_r % epc)
      return set_error(MOTE_ERR_ARGUMENT, "%s: rows must start on 16-byte boundaries", what);
  const int64_t octets = int64_t(a->T) * 4 * ((a->D + kGroup4 - 1) / kGroup4);
  if (octets >= (int64_t(1) << 30) || a->H > kMaxGrid4 || (octets / kRows4Threads + 1) * a->B * a->H >= (int64_t(1) << 31))
    return set_error(MOTE_ERR_SHAPE, "%s: too many rows for one launch", what);
  return MOTE_OK;
}

static int launch_rows4(const mote_cache4_rows_args* a, bool write, hipStream_t stream) {
  const char* what = write ? "cache4_write" : "cache4_read";
  if (const int rc = check_rows4(a, what)) return rc;
  if (a->B == 0 || a->H == 0 || a->T == 0) return MOTE_OK;
  if (write)
    if (const char* bad = shared_cache4(a->cache, a->B, a->H, a->capacity, (a->D + kGroup4 - 1) / kGroup4))
      return set_error(MOTE_ERR_ARGUMENT, "%s: %s", what, bad);
  Rows4Params p;
  const mote_view* v[2] = {&a->p2, &a->info};
  for (int k = 0; k < 2; ++k) {
    p.x[k] = reinterpret_cast<char*>(v[k]->data);
    p.x_sb[k] = v[k]->stride_b; p.x_sh[k] = v[k]->stride_h; p.x_sr[k] = v[k]->stride_r;
  }
  p.code[0] = reinterpret_cast<uint8_t*>(a->cache.p2); p.code[1] = reinterpret_cast<uint8_t*>(a->cache.info);
  p.scale[0] = reinterpret_cast<bf16_t*>(a->cache.p2_scale); p.scale[1] = reinterpret_cast<bf16_t*>(a->cache.info_scale);
  p.c_sb = a->cache.codes_sb; p.c_sh = a->cache.codes_sh; p.s_sb = a->cache.scale_sb; p.s_sh = a->cache.scale_sh;
  p.start = a->start; p.start_dev = a->start_dev; p.lens = write ? a->lens : nullptr;
  p.T = a->T; p.D = a->D; p.G = (a->D + kGroup4 - 1) / kGroup4; p.cap = a->capacity;
  const int chunks = a->D * (a->dtype == MOTE_BF16 ? 2 : 4) / 16;
  uint32_t bits = 0;
  while ((1 << bits) < chunks) ++bits;
  p.over_shift = 31 + bits;
  p.over_mul = uint32_t((uint64_t(1) << p.over_shift) / chunks) + 1;
  const int64_t tiles = (int64_t(a->T) * (write ? 4 * p.G : chunks) + kRows4Threads - 1) / kRows4Threads;
  // New rows that would push everything else out of the Infinity Cache (256 MB) pass it by, so that the codes
  // stay for the read behind them: write and read of 8 x 4984 rows (122 MB of them) 68 -> 61 us together; of
  // 16 x 5000 rows of head dim 48 (61 MB) 43 us, 46 so.
  const bool large = 2.0 * a->B * a->H * a->T * a->D * (a->dtype == MOTE_BF16 ? 2 : 4) >= 96e6;
  const dim3 block(kRows4Threads);
  for (int b0 = 0; b0 < a->B; b0 += kMaxGrid4) {
    const int nb = std::min(a->B - b0, kMaxGrid4);
    const dim3 grid(unsigned(tiles), unsigned(a->H), unsigned(nb));
    if (a->dtype == MOTE_BF16) {
      if (write && large) hipLaunchKernelGGL((cache4_write_kernel<bf16_t, true>), grid, block, 0, stream, p);
      else if (write) hipLaunchKernelGGL((cache4_write_kernel<bf16_t, false>), grid, block, 0, stream, p);
      else hipLaunchKernelGGL(cache4_read_kernel<bf16_t>, grid, block, 0, stream, p);
    } else {
      if (write && large) hipLaunchKernelGGL((cache4_write_kernel<float, true>), grid, block, 0, stream, p);
      else if (write) hipLaunchKernelGGL((cache4_write_kernel<float, false>), grid, block, 0, stream, p);
      else hipLaunchKernelGGL(cache4_read_kernel<float>, grid, block, 0, stream, p);
    }
    const int64_t e = a->dtype == MOTE_BF16 ? 2 : 4;
    for (int k = 0; k < 2; ++k) {
      p.x[k] += nb * p.x_sb[k] * e;
      p.code[k] += nb * p.c_sb;
      p.scale[k] += nb * p.s_sb;
    }
    if (p.start_dev) p.start_dev += nb;
    if (p.lens) p.lens += nb;
  }
  return check_launch(what);
}

int launch_cache4_write(const mote_cache4_rows_args* a, hipStream_t stream) { return launch_rows4(a, true, stream); }
int launch_cache4_read(const mote_cache4_rows_args* a, hipStream_t stream) { return launch_rows4(a, false, stream); }

}  // namespace mote
