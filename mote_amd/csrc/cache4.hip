// Rows of the {P2, I~} cache in 4 bits: written from a prompt's projections, read back for the prefix
// attention (mote_cache4_write / mote_cache4_read; the format stands in mote_relation.h).
//
// Both are one pass over memory, bound by it: 2 D e bytes a row and head on the wide side, D + 4 G on the
// narrow one. A thread holds one octet (eight values) of P2 and of I~, so a wave's wide accesses are
// 16 bytes a lane and its code accesses 4; a group's maximum is two DPP steps over its quad. Values read
// back pass the caches by (4407 rows, 17 MB: 6.5 -> 5.5 us; 8 x 4984 rows 26.6 -> 25.3 us).
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
  int H, T, D, G, cap, tiles;
};

constexpr int kRows4Threads = 256;

// the (sequence, head) of the workgroup and this thread's (row, octet) in it
struct Rows4At {
  int b, h, t, o;
  bool in;
};
__device__ __forceinline__ Rows4At rows4_at(const Rows4Params& p) {
  Rows4At a;
  const int bh = blockIdx.x / p.tiles;
  a.b = bh / p.H;
  a.h = bh % p.H;
  const int64_t i = int64_t(blockIdx.x % p.tiles) * kRows4Threads + threadIdx.x;
  a.t = int(i / (4 * p.G));
  a.o = int(i % (4 * p.G));
  a.in = a.t < p.T;
  return a;
}

template <typename T, bool STREAM>
__global__ void __launch_bounds__(kRows4Threads) cache4_write_kernel(const Rows4Params p) {
  const Rows4At a = rows4_at(p);
  const int64_t start = p.start_dev ? p.start_dev[a.b] : p.start;
  const int64_t len = p.lens ? p.lens[a.b] : p.T;
  const int64_t row = start + a.t;
  // quads are whole (4 G octets a row): a row is written by all of its lanes or by none
  const bool live = a.in && a.t < len && row >= 0 && row < p.cap;
  float x[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (live && 8 * a.o < p.D)
      load_octet<STREAM>(reinterpret_cast<const T*>(p.x[k]) + a.b * p.x_sb[k] + a.h * p.x_sh[k] + a.t * p.x_sr[k] + 8 * a.o, x[k]);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) x[k][j] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    bf16_t s;
    const uint32_t w = encode4(x[k], s);
    if (live) {
      *reinterpret_cast<uint32_t*>(p.code[k] + a.b * p.c_sb + a.h * p.c_sh + row * (16 * p.G) + 4 * a.o) = w;
      if ((a.o & 3) == 0) p.scale[k][a.b * p.s_sb + a.h * p.s_sh + row * p.G + (a.o >> 2)] = s;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kRows4Threads) cache4_read_kernel(const Rows4Params p) {
  const Rows4At a = rows4_at(p);
  if (!a.in || 8 * a.o >= p.D) return;
  const int64_t row = (p.start_dev ? p.start_dev[a.b] : p.start) + a.t;
  const bool held = row >= 0 && row < p.cap;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float x[8];
    uint32_t w = 0;
    float s = __builtin_nanf("");
    if (held) {
      w = *reinterpret_cast<const uint32_t*>(p.code[k] + a.b * p.c_sb + a.h * p.c_sh + row * (16 * p.G) + 4 * a.o);
      s = bf2f(p.scale[k][a.b * p.s_sb + a.h * p.s_sh + row * p.G + (a.o >> 2)]);
    }
    decode4(w, s, x);
    store_octet<T>(reinterpret_cast<T*>(p.x[k]) + a.b * p.x_sb[k] + a.h * p.x_sh[k] + a.t * p.x_sr[k] + 8 * a.o, x);
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
  if ((octets / kRows4Threads + 1) * a->B * a->H >= (int64_t(1) << 31))
    return set_error(MOTE_ERR_SHAPE, "%s: too many rows for one launch", what);
  return MOTE_OK;
}

static int launch_rows4(const mote_cache4_rows_args* a, bool write, hipStream_t stream) {
  const char* what = write ? "cache4_write" : "cache4_read";
  if (const int rc = check_rows4(a, what)) return rc;
  if (a->B == 0 || a->H == 0 || a->T == 0) return MOTE_OK;
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
  p.H = a->H; p.T = a->T; p.D = a->D; p.G = (a->D + kGroup4 - 1) / kGroup4; p.cap = a->capacity;
  p.tiles = int((int64_t(a->T) * 4 * p.G + kRows4Threads - 1) / kRows4Threads);
  const dim3 grid(unsigned(int64_t(p.tiles) * a->B * a->H)), block(kRows4Threads);
  // New rows that would push everything else out of the Infinity Cache (256 MB) pass it by, so that the codes
  // stay for the read behind them: write and read of 8 x 4984 rows (122 MB of them) 68 -> 61 us together; of
  // 16 x 5000 rows of head dim 48 (61 MB) 43 us, 46 so.
  const bool large = 2.0 * a->B * a->H * a->T * a->D * (a->dtype == MOTE_BF16 ? 2 : 4) >= 96e6;
  if (a->dtype == MOTE_BF16) {
    if (write && large) hipLaunchKernelGGL((cache4_write_kernel<bf16_t, true>), grid, block, 0, stream, p);
    else if (write) hipLaunchKernelGGL((cache4_write_kernel<bf16_t, false>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL(cache4_read_kernel<bf16_t>, grid, block, 0, stream, p);
  } else {
    if (write && large) hipLaunchKernelGGL((cache4_write_kernel<float, true>), grid, block, 0, stream, p);
    else if (write) hipLaunchKernelGGL((cache4_write_kernel<float, false>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL(cache4_read_kernel<float>, grid, block, 0, stream, p);
  }
  return check_launch(what);
}

int launch_cache4_write(const mote_cache4_rows_args* a, hipStream_t stream) { return launch_rows4(a, true, stream); }
int launch_cache4_read(const mote_cache4_rows_args* a, hipStream_t stream) { return launch_rows4(a, false, stream); }

}  // namespace mote
