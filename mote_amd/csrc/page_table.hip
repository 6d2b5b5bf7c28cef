// The pages of the cache in 8 bits: given out, shared, given back, and moved into another pool
// (mote_pages_reserve / _fork / _free / _compact; mote_relation.h has the table and the counts).
//
// Bookkeeping is integer work over tables of a few KB, bound by launches and by the chain of a scan; counts go by
// integer atomics, whose order does not matter. What moves bytes is the tails' copy of a fork and the copy of a
// compaction, both bound by memory: 15 forks of 4133 rows in 12 layers 6.8 us, 824 MB of pages moved in 313 (5.3
// TB/s of reads and writes); 16 x 73 entries reserved 4.7, freed 2.7. A reservation walks the whole table by one workgroup,
// 1024 entries a turn of 0.9 us, 2.1 where all of them need pages: 16 x 1024 entries 15 and 34 us, 2^20 0.9 and 2.1 ms.
#include <algorithm>

#include "common.hpp"
#include "device.hpp"
#include "fp8.hpp"

namespace mote {

constexpr int kSeqs = 256;  // sequences of one launch (a kernel argument of 1 KB)
struct SeqList {
  int32_t at[kSeqs];
};

struct PagesParams {
  int blocks, pages, n, src;
  int32_t* table;
  int64_t table_sb;
  int32_t* refs;
  int64_t* S;
  char* tails;
  int64_t tails_sp, tails_sb;  // bytes
  int row_bytes, H, planes, table_wgs;
};

__device__ __forceinline__ void release(const PagesParams& p, int32_t page) {
  if (page >= 0 && page < p.pages) atomicSub(p.refs + page, 1);
}

__global__ void __launch_bounds__(256) pages_free_kernel(const PagesParams p, const SeqList seqs) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= p.blocks) return;
  int32_t* t = p.table + seqs.at[blockIdx.y] * p.table_sb + j;
  release(p, *t);
  *t = -1;
}

// Workgroups [0, table_wgs): 256 entries of one sequence each; the others a (plane, sequence, head) of the tails.
// S[src], src's entries and its tail are only read: src is none of the sequences.
__global__ void __launch_bounds__(256) pages_fork_kernel(const PagesParams p, const SeqList seqs) {
  const int64_t s64 = p.S[p.src], most = int64_t(p.blocks) * kPage8;
  const int64_t rows = s64 < 0 ? 0 : s64 > most ? most : s64;
  if (int(blockIdx.x) < p.table_wgs) {
    const int per = (p.blocks + 255) / 256;
    const int seq = seqs.at[blockIdx.x / per], j = int(blockIdx.x % per) * 256 + threadIdx.x;
    if (j >= p.blocks) return;
    int32_t* t = p.table + seq * p.table_sb + j;
    release(p, *t);
    const int32_t page = j < rows / kPage8 ? p.table[p.src * p.table_sb + j] : -1;
    if (page >= 0 && page < p.pages) atomicAdd(p.refs + page, 1);
    *t = page;
    if (j == 0) p.S[seq] = s64;
    return;
  }
  uint32_t i = blockIdx.x - p.table_wgs;
  const int h = int(i % uint32_t(p.H));
  i /= uint32_t(p.H);
  const int seq = seqs.at[i % uint32_t(p.n)];
  const int64_t plane = i / uint32_t(p.n);
  char* base = p.tails + plane * p.tails_sp + int64_t(h) * kPage8 * p.row_bytes;
  const char* from = base + p.src * p.tails_sb;
  char* to = base + seq * p.tails_sb;
  const int bytes = int(rows % kPage8) * p.row_bytes;
  for (int o = threadIdx.x * 16; o < bytes; o += 256 * 16) store_chunk(to + o, load_chunk(from + o));
}

// ranks of the threads whose flag is set, in thread order, among a workgroup of 1024, and their number; waves'
// counts in `sum` (16 words of LDS). Every thread is here.
__device__ __forceinline__ int rank1024(bool flag, int* sum, int& total) {
  const uint64_t mask = __ballot(flag);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) sum[wave] = __popcll(mask);
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    before += w < wave ? sum[w] : 0;
    total += sum[w];
  }
  return before + __popcll(mask & ((uint64_t(1) << lane) - 1));
}

// One workgroup: free pages from the lowest number on into a list in LDS, then entries in order, each the next of
// the list; refilled until either end. (A list of all free pages in memory would need a workspace, and reads
// back what LDS holds.)
__global__ void __launch_bounds__(1024) pages_reserve_kernel(int32_t* table, int64_t table_sb, int32_t* refs, int B, int blocks,
                                                             int pages, int64_t rows, const int64_t* rows_dev, int32_t* missing) {
  constexpr int kList = 4096;
  __shared__ int32_t list[kList];
  __shared__ int sum[16];
  const int tid = threadIdx.x;
  const int64_t entries = int64_t(B) * blocks;
  int page0 = 0, head = 0, have = 0;  // the next pages to look at; the list's first unused entry and its length
  int lost = 0;
  for (int64_t e0 = 0; e0 < entries; e0 += 1024) {
    const int64_t e = e0 + tid;
    int32_t* t = nullptr;
    bool need = false;
    if (e < entries) {
      const int64_t b = e / blocks, j = e - b * blocks;
      const int64_t n = rows_dev ? rows_dev[b] : rows;
      t = table + b * table_sb + j;
      need = j < n / kPage8 && *t < 0;
    }
    int wanted;
    const int rank = rank1024(need, sum, wanted);
    if (wanted > have - head && page0 < pages) {  // refill: move what is left to the front, then add free pages
      const int left = have - head;
      int32_t keep = 0;
      if (tid < left) keep = list[head + tid];  // fewer than wanted, so fewer than 1024
      __syncthreads();
      if (tid < left) list[tid] = keep;
      head = 0;
      have = left;
      while (have + 1024 <= kList && page0 < pages) {
        const int q = page0 + tid;
        const bool open = q < pages && refs[q] == 0;
        int found;
        const int at = rank1024(open, sum, found);
        if (open) list[have + at] = q;
        have += found;
        page0 += 1024;
      }
      __syncthreads();
    }
    const int given = min(wanted, have - head);
    if (need && rank < given) {
      const int32_t q = list[head + rank];
      *t = q;
      refs[q] = 1;
    }
    head += given;
    lost += wanted - given;  // the list holds more than 1024 pages after a refill, or there are no more
    __syncthreads();
  }
  if (tid == 0) *missing = lost;
}

struct CompactParams {
  int planes, pages, pages2, H, B, blocks;
  int64_t page_bytes, codes_sp, scale_sp, table_sb, codes2_sp, scale2_sp;
  const char* codes;
  const float* scales;
  const int32_t* refs;
  const int32_t* table;
  char* codes2;
  float* scales2;
  int32_t* refs2;
  int32_t* table2;
  int32_t* missing;
  int32_t* map;
  int64_t copies;  // workgroups that copy: pages x planes
};

// One workgroup: the new number of every page (-1: not in use, or beyond the new pool), and the new counts.
__global__ void __launch_bounds__(1024) pages_plan_kernel(const CompactParams p) {
  __shared__ int sum[16];
  const int tid = threadIdx.x;
  int base = 0;
  for (int q0 = 0; q0 < p.pages; q0 += 1024) {
    const int q = q0 + tid;
    const int32_t n = q < p.pages ? p.refs[q] : 0;
    int live;
    const int at = base + rank1024(n > 0, sum, live);
    if (q < p.pages) p.map[q] = n > 0 && at < p.pages2 ? at : -1;
    if (n > 0 && at < p.pages2) p.refs2[at] = n;
    base += live;
  }
  for (int64_t q = base + int64_t(tid); q < p.pages2; q += 1024) p.refs2[q] = 0;
  if (tid == 0) *p.missing = 0;
}

// A page of a plane to its new number, by a workgroup of 256.
__device__ __forceinline__ void move_page(const CompactParams& p, int64_t plane, int page, int now) {
  const int tid = threadIdx.x;
  const char* from = p.codes + plane * p.codes_sp + page * p.page_bytes;
  char* to = p.codes2 + plane * p.codes2_sp + now * p.page_bytes;
  int64_t o = tid * 16;
  for (; o + 3 * 4096 < p.page_bytes; o += 4 * 4096) {
    Chunk c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = load_stream(from + o + k * 4096);
#pragma unroll
    for (int k = 0; k < 4; ++k) store_stream(to + o + k * 4096, c[k]);
  }
  for (; o < p.page_bytes; o += 4096) store_stream(to + o, load_stream(from + o));
  for (int h = tid; h < p.H; h += 256)
    p.scales2[plane * p.scale2_sp + int64_t(now) * p.H + h] = p.scales[plane * p.scale_sp + int64_t(page) * p.H + h];
}

// Workgroups [0, copies): a page of a plane each; the others 256 entries of the table.
__global__ void __launch_bounds__(256) pages_move_kernel(const CompactParams p) {
  const int64_t wg = blockIdx.x;
  if (wg >= p.copies) {
    const int64_t e = (wg - p.copies) * 256 + threadIdx.x;
    if (e >= int64_t(p.B) * p.blocks) return;
    const int64_t b = e / p.blocks, j = e - b * p.blocks;
    const int32_t t = p.table[b * p.table_sb + j];
    const int32_t now = t >= 0 && t < p.pages ? p.map[t] : -1;
    p.table2[e] = now;
    if (t >= 0 && now < 0) atomicAdd(p.missing, 1);
    return;
  }
  const int page = int(wg % p.pages);
  const int32_t now = p.map[page];
  if (now >= 0) move_page(p, wg / p.pages, page, now);
}

// Plan and copies in one launch for a small pool: every workgroup makes a bit per page and their prefix counts in LDS,
// and from them the new numbers that it needs. The last workgroup has the table and the counts (a pool of 300 pages, 28
// MB of them moved: two launches 9.9 us, one 8.8).
constexpr int kFewPages = 4096, kFewEntries = 16384;
__global__ void __launch_bounds__(256) pages_compact_few_kernel(const CompactParams p) {
  __shared__ uint64_t used[kFewPages / 64];
  __shared__ int before[kFewPages / 64], lost[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool table = blockIdx.x == p.copies;
  const int page = table ? p.pages - 1 : int(blockIdx.x % p.pages);
  if (!table && p.refs[page] <= 0) return;  // the same for the whole workgroup
  for (int q0 = wave * 64; q0 < p.pages; q0 += 256) {
    const uint64_t mask = __ballot(q0 + lane < p.pages && p.refs[min(q0 + lane, p.pages - 1)] > 0);
    if (lane == 0) used[q0 / 64] = mask;
  }
  __syncthreads();
  const int words = (p.pages + 63) / 64;
  if (wave == 0) {  // at most 64 words: a lane each
    const int n = lane < words ? __popcll(used[lane]) : 0;
    int sum = n;
    for (int d = 1; d < 64; d *= 2) {
      const int up = __shfl_up(sum, d);
      sum += lane >= d ? up : 0;
    }
    before[lane] = sum - n;
  }
  __syncthreads();
  auto number = [&](int q) {  // the new number of a page (-1: not in use, or beyond the new pool)
    const uint64_t m = used[q / 64], bit = uint64_t(1) << (q % 64);
    const int at = before[q / 64] + __popcll(m & (bit - 1));
    return (m & bit) && at < p.pages2 ? at : -1;
  };
  if (!table) {
    const int now = number(page);
    if (now >= 0) move_page(p, blockIdx.x / p.pages, page, now);
    return;
  }
  for (int q = tid; q < p.pages; q += 256) {
    const int now = number(q);
    if (now >= 0) p.refs2[now] = p.refs[q];
  }
  const int live = before[words - 1] + __popcll(used[words - 1]);
  for (int q = live + tid; q < p.pages2; q += 256) p.refs2[q] = 0;
  int gone = 0;
  for (int e = tid; e < p.B * p.blocks; e += 256) {
    const int b = e / p.blocks, j = e - b * p.blocks;
    const int32_t t = p.table[b * p.table_sb + j];
    const int now = t >= 0 && t < p.pages ? number(t) : -1;
    p.table2[e] = now;
    gone += t >= 0 && now < 0;
  }
  for (int d = 32; d > 0; d >>= 1) gone += __shfl_xor(gone, d);
  if (lane == 0) lost[wave] = gone;
  __syncthreads();
  if (tid == 0) *p.missing = lost[0] + lost[1] + lost[2] + lost[3];
}

static int pages_sizes(const mote_pages_args* a, const char* what) {
  if (!a) return set_error(MOTE_ERR_ARGUMENT, "%s: null args", what);
  if (a->B < 1 || a->blocks < 1 || a->blocks > (1 << 24) || a->pages < 1)
    return set_error(MOTE_ERR_SHAPE, "%s: bad sizes of the pool or the table", what);
  if (!a->table || !a->refs) return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  if (a->B > 1 && a->table_sb < a->blocks) return set_error(MOTE_ERR_ARGUMENT, "%s: sequences lie over one another", what);
  return MOTE_OK;
}
// The listed sequences: each in the table, none of them `src`, and each once in a launch (in two launches one may come
// twice: the second finds what the first left).
static int pages_seqs(const mote_pages_args* a, int src, const char* what) {
  if (a->n < 0 || (a->n > 0 && !a->seqs)) return set_error(MOTE_ERR_ARGUMENT, "%s: bad list of sequences", what);
  for (int i = 0; i < a->n; i += kSeqs) {
    int32_t sorted[kSeqs];
    const int n = std::min(kSeqs, a->n - i);
    std::copy(a->seqs + i, a->seqs + i + n, sorted);
    std::sort(sorted, sorted + n);
    for (int k = 0; k < n; ++k) {
      if (sorted[k] < 0 || sorted[k] >= a->B) return set_error(MOTE_ERR_ARGUMENT, "%s: no sequence %d of %d", what, sorted[k], a->B);
      if (sorted[k] == src) return set_error(MOTE_ERR_ARGUMENT, "%s: sequence %d is the source", what, src);
      if (k > 0 && sorted[k] == sorted[k - 1]) return set_error(MOTE_ERR_ARGUMENT, "%s: sequence %d twice", what, sorted[k]);
    }
  }
  return MOTE_OK;
}
static PagesParams pages_params(const mote_pages_args* a) {
  PagesParams p{};
  p.blocks = a->blocks; p.pages = a->pages; p.src = a->src;
  p.table = a->table; p.table_sb = a->table_sb; p.refs = a->refs; p.S = a->S;
  return p;
}

int launch_pages_free(const mote_pages_args* a, hipStream_t stream) {
  const char* what = "pages_free";
  if (int rc = pages_sizes(a, what)) return rc;
  if (int rc = pages_seqs(a, -1, what)) return rc;
  for (int i = 0; i < a->n; i += kSeqs) {
    PagesParams p = pages_params(a);
    SeqList list{};
    const int n = std::min(kSeqs, a->n - i);
    std::copy(a->seqs + i, a->seqs + i + n, list.at);
    hipLaunchKernelGGL(pages_free_kernel, dim3((a->blocks + 255) / 256, n), dim3(256), 0, stream, p, list);
  }
  return a->n ? check_launch(what) : MOTE_OK;
}

int launch_pages_fork(const mote_pages_args* a, hipStream_t stream) {
  const char* what = "pages_fork";
  if (int rc = pages_sizes(a, what)) return rc;
  if (a->src < 0 || a->src >= a->B) return set_error(MOTE_ERR_ARGUMENT, "%s: no sequence %d of %d", what, a->src, a->B);
  if (int rc = pages_seqs(a, a->src, what)) return rc;
  if (!a->S) return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  int64_t row = 0;
  if (a->tails) {
    if (a->planes < 1 || a->H < 1 || a->D < 8 || a->D > 128 || a->D % 8 || (a->elem_bytes != 2 && a->elem_bytes != 4))
      return set_error(MOTE_ERR_SHAPE, "%s: bad sizes of the tails", what);
    row = int64_t(a->D) * a->elem_bytes;
    if (reinterpret_cast<uintptr_t>(a->tails) % 16 || a->tails_sp * a->elem_bytes % 16 || a->tails_sb * a->elem_bytes % 16)
      return set_error(MOTE_ERR_ARGUMENT, "%s: tails must start on 16-byte boundaries", what);
  }
  for (int i = 0; i < a->n; i += kSeqs) {
    PagesParams p = pages_params(a);
    SeqList list{};
    p.n = std::min(kSeqs, a->n - i);
    std::copy(a->seqs + i, a->seqs + i + p.n, list.at);
    p.table_wgs = p.n * ((a->blocks + 255) / 256);
    int64_t copies = 0;
    if (a->tails) {
      p.tails = reinterpret_cast<char*>(a->tails);
      p.tails_sp = a->tails_sp * a->elem_bytes; p.tails_sb = a->tails_sb * a->elem_bytes;
      p.row_bytes = int(row); p.H = a->H; p.planes = a->planes;
      copies = int64_t(p.n) * a->planes * a->H;
    }
    if (copies > (int64_t(1) << 31) || !grid_fits(p.table_wgs + copies, 256))
      return set_error(MOTE_ERR_SHAPE, "%s: %d planes of %d heads are too many for one launch", what, a->planes, a->H);
    hipLaunchKernelGGL(pages_fork_kernel, dim3(unsigned(p.table_wgs + copies)), dim3(256), 0, stream, p, list);
  }
  return a->n ? check_launch(what) : MOTE_OK;
}

int launch_pages_reserve(const mote_pages_args* a, hipStream_t stream) {
  const char* what = "pages_reserve";
  if (int rc = pages_sizes(a, what)) return rc;
  if (!a->missing) return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  if (a->pages > (1 << 30)) return set_error(MOTE_ERR_SHAPE, "%s: %d pages (at most 2^30)", what, a->pages);
  hipLaunchKernelGGL(pages_reserve_kernel, dim3(1), dim3(1024), 0, stream, a->table, a->table_sb, a->refs, a->B, a->blocks,
                     a->pages, a->rows, a->rows_dev, a->missing);
  return check_launch(what);
}

static bool few_pages(const mote_pages_compact_args* a) {
  return a->pages <= kFewPages && int64_t(a->B) * a->blocks <= kFewEntries;
}

size_t pages_compact_workspace_bytes(const mote_pages_compact_args* a) {
  return a->pages > 0 && !few_pages(a) ? (size_t(a->pages) * sizeof(int32_t) + 15) / 16 * 16 : 0;
}

int launch_pages_compact(const mote_pages_compact_args* a, hipStream_t stream) {
  const char* what = "pages_compact";
  if (!a) return set_error(MOTE_ERR_ARGUMENT, "%s: null args", what);
  if (a->planes < 1 || a->pages < 1 || a->pages2 < 1 || a->H < 1 || a->B < 1 || a->blocks < 1 || a->pages > (1 << 30) ||
      a->pages2 > (1 << 30))
    return set_error(MOTE_ERR_SHAPE, "%s: bad sizes", what);
  if (!a->codes || !a->scales || !a->refs || !a->table || !a->codes2 || !a->scales2 || !a->refs2 || !a->table2 || !a->missing)
    return set_error(MOTE_ERR_ARGUMENT, "%s: null pointer", what);
  const uintptr_t both = reinterpret_cast<uintptr_t>(a->codes) | reinterpret_cast<uintptr_t>(a->codes2);
  if (both % 16 || a->page_bytes < 16 || a->page_bytes % 16 || a->codes_sp % 16 || a->codes2_sp % 16)
    return set_error(MOTE_ERR_ARGUMENT, "%s: pages must start on 16-byte boundaries", what);
  if ((a->planes > 1 && (a->codes_sp < a->pages * a->page_bytes || a->codes2_sp < a->pages2 * a->page_bytes ||
                         a->scale_sp < int64_t(a->pages) * a->H || a->scale2_sp < int64_t(a->pages2) * a->H)) ||
      (a->B > 1 && a->table_sb < a->blocks))
    return set_error(MOTE_ERR_ARGUMENT, "%s: planes or sequences lie over one another", what);
  const size_t need = pages_compact_workspace_bytes(a);
  if (need && (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return set_error(MOTE_ERR_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes, %zu needed", what, a->workspace_bytes, need);
  CompactParams p{};
  p.planes = a->planes; p.pages = a->pages; p.pages2 = a->pages2; p.H = a->H; p.B = a->B; p.blocks = a->blocks;
  p.page_bytes = a->page_bytes; p.codes_sp = a->codes_sp; p.scale_sp = a->scale_sp; p.table_sb = a->table_sb;
  p.codes2_sp = a->codes2_sp; p.scale2_sp = a->scale2_sp;
  p.codes = reinterpret_cast<const char*>(a->codes); p.scales = a->scales; p.refs = a->refs; p.table = a->table;
  p.codes2 = reinterpret_cast<char*>(a->codes2); p.scales2 = a->scales2; p.refs2 = a->refs2; p.table2 = a->table2;
  p.missing = a->missing; p.map = reinterpret_cast<int32_t*>(a->workspace);
  p.copies = int64_t(a->pages) * a->planes;
  const int64_t entries = (int64_t(a->B) * a->blocks + 255) / 256;
  if (!grid_fits(p.copies + entries, 256))
    return set_error(MOTE_ERR_SHAPE, "%s: %d pages of %d planes are too many for one launch", what, a->pages, a->planes);
  if (!need) {
    hipLaunchKernelGGL(pages_compact_few_kernel, dim3(unsigned(p.copies + 1)), dim3(256), 0, stream, p);
    return check_launch(what);
  }
  hipLaunchKernelGGL(pages_plan_kernel, dim3(1), dim3(1024), 0, stream, p);
  if (int rc = check_launch(what)) return rc;
  hipLaunchKernelGGL(pages_move_kernel, dim3(unsigned(p.copies + entries)), dim3(256), 0, stream, p);
  return check_launch(what);
}

}  // namespace mote
