// Rows of the paged {P2, I~} cache in 8 bits: appended from a prompt's projections, read back for the prefix
// attention (mote_cache8_write / mote_cache8_read; the format stands in mote_relation.h).
//
// Both are one pass over memory, bound by it: D e bytes a row, head and kind on the wide side, D + 1/16 on the
// narrow one. A workgroup has one block of one head and kind: the block's maximum needs all of it, and a page of
// 64 rows (6 KB at D = 96) is one round of loads for 256 threads. 8 sequences of up to 4984 rows, 8 heads of 96 in bf16:
// written in 29.3 us (5.5 TB/s of 161 MB), read back in 24.2 (6.6 TB/s); 311 rows in 4.7, 4407 in 6.5, each a block's
// chain of loads. In fp32 8 x 4984 whole rows 51.5 (5.9 TB/s of 306 MB) and 45.6 (6.7), 311 rows 5.4, 4407 7.6; the same
// whole rows in bf16 29.5 and 28.3.
#include <type_traits>

#include "common.hpp"
#include "device.hpp"
#include "fp8.hpp"

namespace mote {

struct Rows8Params {
  const void* p2;  // the new rows (write) or the results (read)
  const void* info;
  int64_t k_sb, k_sh, k_sr, v_sb, v_sh, v_sr;
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  void* kt;
  void* vt;
  const int32_t* table;
  int64_t codes_sp, scale_sp, tail_sb, table_sb;
  int64_t start, held;
  const int64_t* start_dev;
  const int64_t* held_dev;
  const int64_t* lens;
  int B, H, T, D, pages, blocks, nblk;
};

// workgroup -> block (fastest), kind, head, sequence
struct Place8 {
  int blk, kind, h, b;
};
__device__ __forceinline__ Place8 place8(const Rows8Params& p) {
  uint32_t i = blockIdx.x;
  Place8 r;
  r.blk = int(i % uint32_t(p.nblk));
  i /= uint32_t(p.nblk);
  r.kind = int(i & 1u);
  i >>= 1;
  r.h = int(i % uint32_t(p.H));
  r.b = int(i / uint32_t(p.H));
  return r;
}

// The first workgroup of a head and kind has the block that the sequence's old rows end in; the open block at the
// end goes into the tail that those are read from, so the same workgroup writes it, after it.
template <typename T, int C>
__global__ void __launch_bounds__(256) cache8_write_kernel(const Rows8Params p) {
  __shared__ __align__(16) uint8_t bytes[kBlockLds8];
  __shared__ uint32_t top[4];
  const Place8 at = place8(p);
  const int64_t n = p.start_dev ? p.start_dev[at.b] : p.start;
  int64_t len = p.lens ? p.lens[at.b] : p.T;
  len = len < p.T ? len : p.T;
  const int64_t most = int64_t(p.blocks) * kPage8;
  if (n < 0 || n > most || len <= 0) return;
  const int64_t end = n + len < most ? n + len : most;
  const int64_t j0 = n / kPage8, j = j0 + at.blk;
  if (j * kPage8 >= end) return;
  const int D = p.D;
  const T* src = reinterpret_cast<const T*>(at.kind ? p.info : p.p2) +
                 (at.kind ? at.b * p.v_sb + at.h * p.v_sh : at.b * p.k_sb + at.h * p.k_sh);
  const int64_t sr = at.kind ? p.v_sr : p.k_sr;
  T* tail = reinterpret_cast<T*>(at.kind ? p.vt : p.kt) + at.b * p.tail_sb + int64_t(at.h) * (kPage8 * D);
  // 16 dims of row `row` of block blk: new, or still in the tail (the second half past the head dim stays zero)
  auto from = [&](int64_t blk, int row, int ch, float* x) {
    const int64_t pos = blk * kPage8 + row;
    const T* s = (pos < n ? tail + row * D : src + (pos - n) * sr) + ch * 16;
    load_values<8>(s, x);
    if (ch * 16 + 8 < D) load_values<8>(s + 8, x + 8);
  };
  if ((j + 1) * kPage8 <= end) {
    const int32_t page = p.table[at.b * p.table_sb + j];
    const bool ok = page >= 0 && page < p.pages;
    if (ok) {  // the same for the whole workgroup
      uint8_t* dst = (at.kind ? p.vc : p.kc) + page * p.codes_sp + int64_t(at.h) * (kPage8 * 16 * C);
      float* sc = (at.kind ? p.vs : p.ks) + page * p.scale_sp + at.h;
      auto load = [&](int row, int ch, float* x) { from(j, row, ch, x); };
      if (at.kind) store_block8<C, true>(load, dst, sc, top, bytes);
      else store_block8<C, false>(load, dst, sc, top, bytes);
    }
  }
  // the open block, by the first workgroup alone: every tail row that it needed is in registers or stored by now
  const int64_t jl = end / kPage8;
  const int rest = int(end % kPage8);
  if (at.blk != 0 || rest == 0) return;
  __syncthreads();
  for (int it = threadIdx.x; it < kPage8 * C; it += 256) {
    const int row = it / C, ch = it % C;
    const int64_t pos = jl * kPage8 + row;
    if (row >= rest || pos < n) continue;
    const T* s = src + (pos - n) * sr + ch * 16;
    T* d = tail + row * D + ch * 16;
#pragma unroll
    for (int k = 0; k < int(sizeof(T)); ++k)
      if (ch * 16 + k * int(16 / sizeof(T)) < D) store_chunk(d + k * (16 / sizeof(T)), load_chunk(s + k * (16 / sizeof(T))));
  }
}

// A workgroup has the rows of one page: its codes come in 1 KB pieces and are laid out by rows in LDS, and the
// results leave in memory order, 16 bytes a thread.
template <typename T, typename TT, int C>
__global__ void __launch_bounds__(256) cache8_read_kernel(const Rows8Params p) {
  constexpr int PK = 16 * C + 16, PV = 16 * C + 4;  // LDS bytes between rows: whole-chunk and byte stores
  constexpr int PER = 16 / int(sizeof(T));          // values of a thread's piece
  __shared__ __align__(16) uint8_t rows[kPage8 * PK];
  const Place8 at = place8(p);
  constexpr int64_t kFar = int64_t(1) << 40;  // beyond every position that a table reaches
  int64_t s0 = p.start_dev ? p.start_dev[at.b] : p.start;
  s0 = s0 < -kFar ? -kFar : s0 > kFar ? kFar : s0;
  const int64_t held = p.held_dev ? p.held_dev[at.b] : p.held;
  const int64_t first = s0 >= 0 ? s0 / kPage8 : -((-s0 + kPage8 - 1) / kPage8);
  const int64_t j = first + at.blk, base = j * kPage8;  // the block's first position
  if (base >= s0 + p.T) return;
  const int D = p.D, tid = threadIdx.x;
  T* out = reinterpret_cast<T*>(const_cast<void*>(at.kind ? p.info : p.p2)) +
           (at.kind ? at.b * p.v_sb + at.h * p.v_sh : at.b * p.k_sb + at.h * p.k_sh);
  const int64_t sr = at.kind ? p.v_sr : p.k_sr;
  const TT* tail = reinterpret_cast<const TT*>(at.kind ? p.vt : p.kt) + at.b * p.tail_sb + int64_t(at.h) * (kPage8 * D);
  const bool whole = j >= 0 && held >= base + kPage8;
  float s = __builtin_nanf("");
  if (whole) {
    const int32_t page = j < p.blocks ? p.table[at.b * p.table_sb + j] : -1;
    if (page >= 0 && page < p.pages) {
      s = (at.kind ? p.vs : p.ks)[page * p.scale_sp + at.h];
      const uint8_t* src = (at.kind ? p.vc : p.kc) + page * p.codes_sp + int64_t(at.h) * (kPage8 * 16 * C);
#pragma unroll
      for (int it = tid; it < kPage8 * C; it += 256) {
        const Chunk c = load_chunk(src + it * 16);
        if (!at.kind) {
          store_chunk(rows + (it % kPage8) * PK + (it / kPage8) * 16, c);
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) rows[((it % 4) * 16 + k) * PV + it / 4] = uint8_t(c.w[k / 4] >> (8 * (k % 4)));
        }
      }
    } else {
      for (int it = tid; it < kPage8 * PK / 4; it += 256) reinterpret_cast<uint32_t*>(rows)[it] = 0;
    }
    __syncthreads();
  }
  const int per_row = D / PER;
  const uint32_t inv = (65536u + per_row - 1) / per_row;  // o / per_row for o < 2048, per_row <= 32
  for (int o = tid; o < kPage8 * per_row; o += 256) {
    const int row = int((uint32_t(o) * inv) >> 16), d = (o - row * per_row) * PER;
    const int64_t pos = base + row, t = pos - s0;
    if (t < 0 || t >= p.T) continue;
    float x[PER];
    if (pos < 0 || pos >= held) {
#pragma unroll
      for (int k = 0; k < PER; ++k) x[k] = 0.f;
    } else if (whole) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(rows + row * (at.kind ? PV : PK) + d);
#pragma unroll
      for (int k = 0; k < PER / 4; ++k) {
        const f32x2 a = codes8_f32<false>(w[k]), b = codes8_f32<true>(w[k]);
        x[4 * k] = a.x * s; x[4 * k + 1] = a.y * s; x[4 * k + 2] = b.x * s; x[4 * k + 3] = b.y * s;
      }
    } else if (base >= int64_t(p.blocks) * kPage8) {  // no such block
#pragma unroll
      for (int k = 0; k < PER; ++k) x[k] = __builtin_nanf("");
    } else {
#pragma unroll
      for (int k = 0; k < PER; ++k) x[k] = Elem<TT>::to_f(tail[row * D + d + k]);
    }
    Chunk c;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int k = 0; k < 4; ++k) c.w[k] = uint32_t(f2bf(x[2 * k])) | (uint32_t(f2bf(x[2 * k + 1])) << 16);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) c.w[k] = __float_as_uint(x[k]);
    }
    store_stream(out + t * sr + d, c);
  }
}

static const char* fill8(const mote_cache8_rows_args* a, Rows8Params& p, int row_bytes, int tail_bytes) {
  if (const char* bad = bad_cache8(a->cache, a->B, a->H, a->D, tail_bytes)) return bad;
  for (const mote_view* v : {&a->p2, &a->info}) {
    if (!v->data) return "null pointer";
    if (reinterpret_cast<uintptr_t>(v->data) % 16 || v->stride_b * row_bytes % 16 || v->stride_h * row_bytes % 16 ||
        v->stride_r * row_bytes % 16)
      return "rows must start on 16-byte boundaries";
  }
  p.p2 = a->p2.data; p.k_sb = a->p2.stride_b; p.k_sh = a->p2.stride_h; p.k_sr = a->p2.stride_r;
  p.info = a->info.data; p.v_sb = a->info.stride_b; p.v_sh = a->info.stride_h; p.v_sr = a->info.stride_r;
  const mote_cache8& c = a->cache;
  p.kc = reinterpret_cast<uint8_t*>(c.p2); p.vc = reinterpret_cast<uint8_t*>(c.info);
  p.ks = c.p2_scale; p.vs = c.info_scale;
  p.kt = c.p2_tail; p.vt = c.info_tail;
  p.table = c.table;
  p.codes_sp = c.codes_sp; p.scale_sp = c.scale_sp; p.tail_sb = c.tail_sb; p.table_sb = c.table_sb;
  p.start = a->start; p.start_dev = a->start_dev; p.held = a->held; p.held_dev = a->held_dev; p.lens = a->lens;
  p.B = a->B; p.H = a->H; p.T = a->T; p.D = a->D; p.pages = c.pages; p.blocks = c.blocks;
  // the blocks that T rows touch: one more than they fill where the first may begin inside one
  p.nblk = int((int64_t(a->T) + kPage8 - 1) / kPage8) + (a->start_dev || a->start % kPage8 ? 1 : 0);
  return nullptr;
}

static int rows8_sizes(const mote_cache8_rows_args* a, const char* what) {
  if (!a) return set_error(MOTE_ERR_ARGUMENT, "%s: null args", what);
  if ((a->dtype != MOTE_F32 && a->dtype != MOTE_BF16) || (a->tail_dtype != MOTE_F32 && a->tail_dtype != MOTE_BF16))
    return set_error(MOTE_ERR_ARGUMENT, "%s: bad dtype %d, %d", what, a->dtype, a->tail_dtype);
  if (a->D <= 0 || a->D > 128 || a->D % 8)
    return set_error(MOTE_ERR_SHAPE, "%s: head dim %d unsupported (need 8 <= D <= 128, D %% 8 == 0)", what, a->D);
  if (a->B < 0 || a->H < 0 || a->T < 0 || a->T >= (1 << 30)) return set_error(MOTE_ERR_SHAPE, "%s: bad sizes", what);
  return MOTE_OK;
}

static int grid8(const Rows8Params& p, const char* what, unsigned& grid) {
  const int64_t heads = int64_t(p.B) * p.H;
  if (heads > (int64_t(1) << 24) || !grid_fits(heads * 2 * p.nblk, 256))
    return set_error(MOTE_ERR_SHAPE, "%s: %d rows of %d sequences and %d heads are too many for one launch", what, p.T, p.B, p.H);
  grid = unsigned(heads * 2 * p.nblk);
  return MOTE_OK;
}

#define MOTE_C8(C_, ...)          \
  switch (C_) {                   \
    case 1: __VA_ARGS__(1); break; \
    case 2: __VA_ARGS__(2); break; \
    case 3: __VA_ARGS__(3); break; \
    case 4: __VA_ARGS__(4); break; \
    case 5: __VA_ARGS__(5); break; \
    case 6: __VA_ARGS__(6); break; \
    case 7: __VA_ARGS__(7); break; \
    default: __VA_ARGS__(8); break; \
  }

int launch_cache8_write(const mote_cache8_rows_args* a, hipStream_t stream) {
  const char* what = "cache8_write";
  if (int rc = rows8_sizes(a, what)) return rc;
  if (a->dtype != a->tail_dtype) return set_error(MOTE_ERR_ARGUMENT, "%s: rows and tails must share a dtype", what);
  if (a->B == 0 || a->H == 0 || a->T == 0) return MOTE_OK;
  Rows8Params p{};
  const int e = a->dtype == MOTE_F32 ? 4 : 2;
  if (const char* bad = fill8(a, p, e, e)) return set_error(MOTE_ERR_ARGUMENT, "%s: %s", what, bad);
  unsigned grid;
  if (int rc = grid8(p, what, grid)) return rc;
#define MOTE_W8(C_) hipLaunchKernelGGL((cache8_write_kernel<T, C_>), dim3(grid), dim3(256), 0, stream, p)
  if (a->dtype == MOTE_BF16) {
    using T = bf16_t;
    MOTE_C8(chunks8(a->D), MOTE_W8)
  } else {
    using T = float;
    MOTE_C8(chunks8(a->D), MOTE_W8)
  }
#undef MOTE_W8
  return check_launch(what);
}

int launch_cache8_read(const mote_cache8_rows_args* a, hipStream_t stream) {
  const char* what = "cache8_read";
  if (int rc = rows8_sizes(a, what)) return rc;
  if (a->B == 0 || a->H == 0 || a->T == 0) return MOTE_OK;
  Rows8Params p{};
  if (const char* bad = fill8(a, p, a->dtype == MOTE_F32 ? 4 : 2, a->tail_dtype == MOTE_F32 ? 4 : 2))
    return set_error(MOTE_ERR_ARGUMENT, "%s: %s", what, bad);
  unsigned grid;
  if (int rc = grid8(p, what, grid)) return rc;
#define MOTE_R8(C_) hipLaunchKernelGGL((cache8_read_kernel<T, TT, C_>), dim3(grid), dim3(256), 0, stream, p)
  auto launch = [&](auto t, auto tt) {
    using T = decltype(t);
    using TT = decltype(tt);
    MOTE_C8(chunks8(a->D), MOTE_R8)
  };
  if (a->dtype == MOTE_BF16) {
    if (a->tail_dtype == MOTE_BF16) launch(bf16_t{}, bf16_t{});
    else launch(bf16_t{}, 0.f);
  } else {
    if (a->tail_dtype == MOTE_BF16) launch(0.f, bf16_t{});
    else launch(0.f, 0.f);
  }
#undef MOTE_R8
  return check_launch(what);
}

}  // namespace mote
