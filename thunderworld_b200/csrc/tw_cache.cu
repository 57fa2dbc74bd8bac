// Pages of a key-value cache, managed on the device so that a captured step can allocate: which pages a sequence has (table, -1 behind
// them), how many tokens (lengths), and how many sequences hold a page (refs, 0: free).
//   append   rows of new tokens behind their sequences; pages are taken from the lowest free numbers, in the order of the entries
//   fork     children share their parents' full pages; a partly filled last page is copied, so that only its owner ever writes it
//   free     a sequence's pages lose a reference each
//   compact  the live pages with the highest numbers move into the lowest free ones, until the live ones are numbers 0 ... live - 1
// append, fork and compact are two launches: a plan by one CTA (a few kilobytes of counts and, only where a page is needed,
// one pass over refs: block-wide prefix sums give every request its page, so the result does not depend on any order of execution),
// then the copies by the whole device, which is what takes the time where there is much to copy (HBM-bound, 16 bytes a lane). A call whose
// append or fork does not work out (a slot, length or page outside, a slot twice, a full pool) changes nothing and reports it in the status
// word; compact leaves table entries outside the pool as they are and reports them.
// Measured (B200, kernels alone): compact 5.6 us + 25.2 us for copies of 91 MB of pages (64 tokens, 8 heads of 128, bf16; 7 TB/s read and written, some
// of it in L2); append of 64 tokens 7.0 + 4.7 us, of 48 x 1 ... 200 rows 7.0 + 10.0 us, E4M3 13.9; fork of 32 sequences 8.6 + 7.1 us, of 1000 10.0 + 17.0;
// free of 32 4.7 us. Append and fork of tens of sequences copy a microsecond or two: they are held by their two launches.
#include "tw_common.cuh"
#include "../../include/twb200.h"

namespace {

constexpr int PLAN = 1024;                       // threads of the planning CTA
constexpr int MOST_SEQUENCES = 65536;

struct Cache {
  uint8_t *k, *v; long long k_page, k_head, v_page, v_head;          // strides in bytes
  int* table; long long table_stride;
  int *lengths, *refs, *status;
  int sequences, max_pages, pages, hk, page_shift, row;               // row: bytes
};
struct Plan { int ok, count, live, unused; };                         // head of the workspace

__device__ __forceinline__ int pages_of(const Cache& c, int tokens) { return (tokens + (1 << c.page_shift) - 1) >> c.page_shift; }
__device__ __forceinline__ void report(const Cache& c, int code) { if (c.status) atomicMax(c.status, code); }
__device__ __forceinline__ bool outside(const Cache& c, int page) { return page < 0 || page >= c.pages; }
__device__ __forceinline__ long long capacity(const Cache& c) { return (long long)c.max_pages << c.page_shift; }

// Exclusive prefix sum of one value per thread of the planning CTA; returns the sum of all in `total`.
__device__ __forceinline__ int block_scan(int value, int& total) {
  __shared__ int warps[PLAN / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int sum = value;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += x; }
  __syncthreads();                               // of the call before, everyone has read `warps`
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int w = warps[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += x; }
    warps[lane] = w;
  }
  __syncthreads();
  total = warps[PLAN / 32 - 1];
  return sum - value + (warp ? warps[warp - 1] : 0);
}
// Calls take(rank, page) for the pages of [from, to) that `want(refs)` holds for, in ascending order of their numbers, until `most`
// of them are found; returns how many were.
template <typename Want, typename Take>
__device__ __forceinline__ int rank_pages(const Cache& c, int from, int to, int most, Want want, Take take) {
  int found = 0;
  for (int base = from; base < to && found < most; base += PLAN * 4) {
    const int first = base + threadIdx.x * 4;
    int mine = 0, total;
    bool is[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) { is[j] = first + j < to && want(c.refs[first + j]); mine += is[j]; }
    int rank = found + block_scan(mine, total);
#pragma unroll
    for (int j = 0; j < 4; ++j) if (is[j]) { if (rank < most) take(rank, first + j); ++rank; }
    found += total;
  }
  return found < most ? found : most;
}
// Marks sequence s; true if it was marked before.
__device__ __forceinline__ bool twice(unsigned* seen, int s) { return atomicOr(seen + (s >> 5), 1u << (s & 31)) >> (s & 31) & 1u; }

// ---- append -----------------------------------------------------------------------------------------------------------
struct Append {
  const __nv_bfloat16 *k, *v; long long k_row, k_head, v_row, v_head;
  const int *slots, *cu;
  const float *k_scale, *v_scale;
  Plan* plan; int *base, *offset, *fresh;        // per entry: tokens before, first request; per request: its page
  int batch, rows, most_fresh, dim;
};
__device__ __forceinline__ int slot_of(const Append& a, int i) { return a.slots ? a.slots[i] : i; }

__global__ void __launch_bounds__(PLAN) append_plan_kernel(const __grid_constant__ Cache c, const __grid_constant__ Append a) {
  __shared__ unsigned seen[MOST_SEQUENCES / 32];
  __shared__ int error;
  for (int i = threadIdx.x; i < (c.sequences + 31) / 32; i += PLAN) seen[i] = 0;
  if (threadIdx.x == 0) error = 0;
  __syncthreads();
  int needed = 0;
  for (int first = 0; first < a.batch; first += PLAN) {
    const int i = first + threadIdx.x;
    int need = 0;
    if (i < a.batch) {
      const int s = slot_of(a, i), from = a.cu ? a.cu[i] : i, to = a.cu ? a.cu[i + 1] : i + 1;
      int wrong = 0;
      if (s < 0 || s >= c.sequences || from < 0 || to < from || to > a.rows) wrong = TW_ERR_PAGE;
      else if (twice(seen, s)) wrong = TW_ERR_PAGE;
      else {
        const int before = c.lengths[s];
        if (before < 0 || before > capacity(c)) wrong = TW_ERR_PAGE;
        else if (before + (long long)(to - from) > capacity(c)) wrong = TW_ERR_CACHE_FULL;
        else if (to > from && before & ((1 << c.page_shift) - 1) && outside(c, c.table[s * c.table_stride + (before >> c.page_shift)])) wrong = TW_ERR_PAGE;
        else { need = pages_of(c, before + to - from) - pages_of(c, before); a.base[i] = before; }
      }
      if (wrong) { atomicMax(&error, wrong); need = 0; }
    }
    int total;
    const int rank = block_scan(need, total);
    if (i < a.batch) a.offset[i] = needed + rank;
    needed = min(needed + total, a.most_fresh + 1);
  }
  __syncthreads();
  // requests are bounded by the rows, whatever the lengths: most_fresh is what the workspace holds
  if (!error && needed > 0) {
    const int got = needed > a.most_fresh ? 0 : rank_pages(c, 0, c.pages, needed, [](int refs) { return refs == 0; }, [&](int rank, int page) { a.fresh[rank] = page; });
    if (threadIdx.x == 0 && got < needed) error = TW_ERR_CACHE_FULL;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (error) report(c, error);
    a.plan->ok = !error;
  }
  if (error) return;
  for (int r = threadIdx.x; r < needed; r += PLAN) {
    int low = 0, high = a.batch - 1;             // the last entry whose requests begin at or before r
    while (low < high) { const int mid = (low + high + 1) >> 1; if (a.offset[mid] <= r) low = mid; else high = mid - 1; }
    const int s = slot_of(a, low), page = a.fresh[r];
    c.table[s * c.table_stride + pages_of(c, a.base[low]) + r - a.offset[low]] = page;
    c.refs[page] = 1;
  }
  for (int i = threadIdx.x; i < a.batch; i += PLAN) c.lengths[slot_of(a, i)] = a.base[i] + (a.cu ? a.cu[i + 1] - a.cu[i] : 1);
}

__device__ __forceinline__ uint2 to_e4m3(const uint4& x, float scale) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t out[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = __fdiv_rn(tw::bf16_bits_to_float(w[i] & 0xffffu), scale), hi = __fdiv_rn(tw::bf16_bits_to_float(w[i] >> 16), scale);
    uint16_t two;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(hi), "f"(lo));
    out[i >> 1] |= (uint32_t)two << (i & 1) * 16;
  }
  return make_uint2(out[0], out[1]);
}

template <bool FP8>
__global__ void __launch_bounds__(256) append_rows_kernel(const __grid_constant__ Cache c, const __grid_constant__ Append a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!a.plan->ok) return;
  const int chunks = a.dim / 8, per_row = c.hk * chunks;               // 8 values a thread
  const long long all = (long long)a.rows * per_row;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < all; e += (long long)gridDim.x * 256) {
    const int r = (int)(e / per_row), inside = (int)(e - (long long)r * per_row), head = inside / chunks, at = (inside - head * chunks) * 8;
    int i = r;
    if (a.cu) {
      int low = 0, high = a.batch - 1;           // the last entry that begins at or before r
      while (low < high) { const int mid = (low + high + 1) >> 1; if (a.cu[mid] <= r) low = mid; else high = mid - 1; }
      i = low;
      if (r < a.cu[i] || r >= a.cu[i + 1]) continue;                   // rows of no entry
    }
    const int pos = a.base[i] + (a.cu ? r - a.cu[i] : 0), page = c.table[slot_of(a, i) * c.table_stride + (pos >> c.page_shift)];
    if (outside(c, page)) { report(c, TW_ERR_PAGE); continue; }        // not after the plan, unless somebody changes the table meanwhile
    const uint4 k = *reinterpret_cast<const uint4*>(a.k + r * a.k_row + head * a.k_head + at), v = *reinterpret_cast<const uint4*>(a.v + r * a.v_row + head * a.v_head + at);
    const long long row = (long long)(pos & ((1 << c.page_shift) - 1)) * c.row + at * (FP8 ? 1 : 2);
    uint8_t *ko = c.k + page * c.k_page + head * c.k_head + row, *vo = c.v + page * c.v_page + head * c.v_head + row;
    if (FP8) {
      *reinterpret_cast<uint2*>(ko) = to_e4m3(k, a.k_scale ? a.k_scale[head] : 1.f);
      *reinterpret_cast<uint2*>(vo) = to_e4m3(v, a.v_scale ? a.v_scale[head] : 1.f);
    } else {
      *reinterpret_cast<uint4*>(ko) = k;
      *reinterpret_cast<uint4*>(vo) = v;
    }
  }
}

// ---- fork -------------------------------------------------------------------------------------------------------------
struct Fork {
  const int *parents, *children;
  Plan* plan; int *tokens, *fresh;               // per pair: the parent's tokens, the page for its partly filled one or -1
  int count;
};

__global__ void __launch_bounds__(PLAN) fork_plan_kernel(const __grid_constant__ Cache c, const __grid_constant__ Fork f) {
  __shared__ unsigned seen[MOST_SEQUENCES / 32];
  __shared__ int error;
  for (int i = threadIdx.x; i < (c.sequences + 31) / 32; i += PLAN) seen[i] = 0;
  if (threadIdx.x == 0) error = 0;
  __syncthreads();
  int needed = 0;
  for (int first = 0; first < f.count; first += PLAN) {
    const int i = first + threadIdx.x;
    int need = 0;
    if (i < f.count) {
      const int parent = f.parents[i], child = f.children[i];
      bool wrong = parent < 0 || parent >= c.sequences || child < 0 || child >= c.sequences;
      if (!wrong) wrong = twice(seen, child) || c.lengths[child] != 0;
      const int tokens = wrong ? 0 : c.lengths[parent];
      wrong = wrong || tokens < 0 || tokens > capacity(c);
      if (wrong) atomicMax(&error, (int)TW_ERR_PAGE);
      else { need = (tokens & ((1 << c.page_shift) - 1)) != 0; f.tokens[i] = tokens; }
    }
    int total;
    const int rank = block_scan(need, total);
    if (i < f.count) f.fresh[i] = need ? -2 - (needed + rank) : -1;      // the request, until its page is known
    needed += total;
  }
  __syncthreads();
  if (!error) {
    // the parents' pages have to be pages: as many threads look through one's as there are for each
    int each = PLAN;
    while (each > 1 && each * f.count > PLAN) each >>= 1;
    bool wrong = false;
    for (int i = threadIdx.x / each; i < f.count; i += PLAN / each) {
      const int* row = c.table + f.parents[i] * c.table_stride;
      const int pages = pages_of(c, f.tokens[i]);
#pragma unroll 4
      for (int j = threadIdx.x % each; j < pages; j += each) wrong = wrong | outside(c, row[j]);
    }
    if (wrong) atomicMax(&error, (int)TW_ERR_PAGE);
  }
  __syncthreads();
  int* free_pages = f.fresh + f.count;
  if (!error && needed > 0) {
    const int got = rank_pages(c, 0, c.pages, needed, [](int refs) { return refs == 0; }, [&](int rank, int page) { free_pages[rank] = page; });
    if (threadIdx.x == 0 && got < needed) error = TW_ERR_CACHE_FULL;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (error) report(c, error);
    f.plan->ok = !error;
  }
  if (error) return;
  for (int i = threadIdx.x; i < f.count; i += PLAN) {
    if (f.fresh[i] != -1) {
      const int page = free_pages[-2 - f.fresh[i]];
      f.fresh[i] = page;
      c.refs[page] = 1;
    }
    c.lengths[f.children[i]] = f.tokens[i];      // every parent's has been read
  }
}

__device__ __forceinline__ void copy_bytes(uint8_t* to, const uint8_t* from, int bytes, int thread, int threads) {   // multiples of 16
  int at = thread * 16;
  for (; at + 3 * threads * 16 < bytes; at += 4 * threads * 16) {
    uint4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __ldcs(reinterpret_cast<const uint4*>(from + at + j * threads * 16));
#pragma unroll
    for (int j = 0; j < 4; ++j) __stcs(reinterpret_cast<uint4*>(to + at + j * threads * 16), x[j]);
  }
  for (; at < bytes; at += threads * 16) *reinterpret_cast<uint4*>(to + at) = *reinterpret_cast<const uint4*>(from + at);
}

// Block (pair, part): part 0 also writes the child's table row; part 2 h and 2 h + 1 copy what the parent's last page holds of head h.
__global__ void __launch_bounds__(128) fork_copy_kernel(const __grid_constant__ Cache c, const __grid_constant__ Fork f) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!f.plan->ok) return;
  const int i = blockIdx.x, tokens = f.tokens[i], full = tokens >> c.page_shift, part = tokens & ((1 << c.page_shift) - 1), fresh = f.fresh[i];
  const int* from = c.table + f.parents[i] * c.table_stride;
  int* to = c.table + f.children[i] * c.table_stride;
  if (blockIdx.y == 0) {
    for (int j = threadIdx.x; j < full; j += 128) {
      const int page = from[j];
      to[j] = page;
      if (outside(c, page)) report(c, TW_ERR_PAGE); else atomicAdd(c.refs + page, 1);       // as above
    }
    if (threadIdx.x == 0 && part) to[full] = fresh;
  }
  if (!part) return;
  const int old = from[full];
  if (outside(c, old)) { if (threadIdx.x == 0) report(c, TW_ERR_PAGE); return; }
  for (int p = blockIdx.y; p < 2 * c.hk; p += gridDim.y) {
    const int head = p >> 1;
    const long long page = p & 1 ? c.v_page : c.k_page, at = head * (p & 1 ? c.v_head : c.k_head);
    uint8_t* pool = p & 1 ? c.v : c.k;
    copy_bytes(pool + fresh * page + at, pool + old * page + at, part * c.row, threadIdx.x, 128);
  }
}

// ---- free -------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(128) free_kernel(const __grid_constant__ Cache c, const int* slots) {
  const int s = slots[blockIdx.x];
  __shared__ int tokens;
  if (s < 0 || s >= c.sequences) { if (threadIdx.x == 0) report(c, TW_ERR_PAGE); return; }
  if (threadIdx.x == 0) tokens = atomicExch(c.lengths + s, 0);           // a slot named twice is empty the second time
  __syncthreads();
  int* row = c.table + s * c.table_stride;
  const int pages = tokens < 0 ? 0 : tokens > capacity(c) ? c.max_pages : pages_of(c, tokens);
  if ((tokens < 0 || tokens > capacity(c)) && threadIdx.x == 0) report(c, TW_ERR_PAGE);
  for (int j = threadIdx.x; j < pages; j += 128) {
    const int page = row[j];
    row[j] = -1;
    if (outside(c, page)) report(c, TW_ERR_PAGE);
    else if (atomicSub(c.refs + page, 1) <= 0) { atomicAdd(c.refs + page, 1); report(c, TW_ERR_PAGE); }     // nobody held it
  }
}

// ---- compact ----------------------------------------------------------------------------------------------------------
struct Compact { Plan* plan; int *source, *target, *number; int* live; };        // number: the new one of a page that moves

__global__ void __launch_bounds__(PLAN) compact_plan_kernel(const __grid_constant__ Cache c, const __grid_constant__ Compact m) {
  int live = 0, total;
  for (int base = 0; base < c.pages; base += PLAN * 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) { const int p = base + j * PLAN + threadIdx.x; live += p < c.pages && c.refs[p] > 0; }
  }
  block_scan(live, total);
  live = total;
  for (int p = live + threadIdx.x; p < c.pages; p += PLAN) m.number[p] = -1;
  const int away = rank_pages(c, live, c.pages, c.pages, [](int refs) { return refs > 0; }, [&](int rank, int page) { m.source[rank] = page; });
  rank_pages(c, 0, live, away, [](int refs) { return refs <= 0; }, [&](int rank, int page) { m.target[rank] = page; });
  __syncthreads();
  for (int r = threadIdx.x; r < away; r += PLAN) {
    const int from = m.source[r], to = m.target[r];
    m.number[from] = to;
    c.refs[to] = c.refs[from];
    c.refs[from] = 0;
  }
  if (threadIdx.x == 0) { m.plan->count = away; m.plan->live = live; if (m.live) *m.live = live; }
}

__global__ void __launch_bounds__(256) compact_move_kernel(const __grid_constant__ Cache c, const __grid_constant__ Compact m) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int away = m.plan->count, live = m.plan->live;
  if (!away) return;
  // table entries of pages that moved; a page number at or above `live` held pages before, and those moved
  const long long entries = (long long)c.sequences * c.max_pages;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < entries; e += (long long)gridDim.x * 256) {
    const int s = (int)(e / c.max_pages), j = (int)(e - (long long)s * c.max_pages), tokens = c.lengths[s];
    if (tokens <= 0 || (long long)j << c.page_shift >= tokens) continue;
    int* at = c.table + s * c.table_stride + j;
    const int page = *at;
    if (outside(c, page)) report(c, TW_ERR_PAGE);
    else if (page >= live) {
      const int to = m.number[page];
      if (to >= 0 && to < live) *at = to; else report(c, TW_ERR_PAGE);
    }
  }
  const int bytes = c.row << c.page_shift;
  const long long items = (long long)away * 2 * c.hk;
  for (long long e = blockIdx.x; e < items; e += gridDim.x) {
    const int r = (int)(e / (2 * c.hk)), p = (int)(e - (long long)r * 2 * c.hk), head = p >> 1;
    const long long page = p & 1 ? c.v_page : c.k_page, at = head * (p & 1 ? c.v_head : c.k_head);
    uint8_t* pool = p & 1 ? c.v : c.k;
    copy_bytes(pool + m.target[r] * page + at, pool + m.source[r] * page + at, bytes, threadIdx.x, 256);
  }
}

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

int cache_of(const TwCache* a, Cache& c, bool pools) {
  if (!a || !a->table || !a->lengths || !a->refs || a->sequences <= 0 || a->max_pages <= 0 || a->pages <= 0 || a->page <= 0) return TW_ERR_ARGUMENT;
  if (a->page & (a->page - 1)) return TW_ERR_SHAPE;
  if (a->sequences > MOST_SEQUENCES || a->page > (1 << 20) || (long long)a->max_pages * a->page > (1LL << 30)) return TW_ERR_TOO_LARGE;
  if (pools) {
    if (!a->k_pages || !a->v_pages || a->hk <= 0) return TW_ERR_ARGUMENT;
    if (a->dim != 64 && a->dim != 128) return TW_ERR_SHAPE;
    const int bytes = a->fp8 ? 1 : 2;
    if (misaligned(a->k_pages, 16) || misaligned(a->v_pages, 16) ||
        ((a->k_stride_page | a->k_stride_head | a->v_stride_page | a->v_stride_head) * bytes) % 16)
      return TW_ERR_ALIGNMENT;
    if ((long long)a->page * a->dim * bytes > (1LL << 30) || a->hk > 65536) return TW_ERR_TOO_LARGE;
    c.k = static_cast<uint8_t*>(a->k_pages); c.v = static_cast<uint8_t*>(a->v_pages);
    c.k_page = a->k_stride_page * bytes; c.k_head = a->k_stride_head * bytes;
    c.v_page = a->v_stride_page * bytes; c.v_head = a->v_stride_head * bytes;
    c.row = a->dim * bytes;
  }
  c.table = a->table; c.table_stride = a->table_stride; c.lengths = a->lengths; c.refs = a->refs; c.status = a->status;
  c.sequences = a->sequences; c.max_pages = a->max_pages; c.pages = a->pages; c.hk = a->hk;
  while ((1 << c.page_shift) < a->page) ++c.page_shift;
  return TW_OK;
}

// The second launch of an operation: overlaps the first one's end, waits for it before it reads anything.
template <typename... Args>
int launch_after(void (*kernel)(Args...), dim3 grid, int threads, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  if (cudaLaunchKernelEx(&config, kernel, args...) != cudaSuccess) { (void)cudaGetLastError(); return TW_ERR_LAUNCH; }
  return TW_OK;
}

}  // namespace

extern "C" size_t tw_cache_append_workspace(int batch, int rows) {
  return batch <= 0 || rows < 0 ? 0 : sizeof(Plan) + ((size_t)2 * batch + rows) * 4;
}
extern "C" size_t tw_cache_fork_workspace(int count) { return count <= 0 ? 0 : sizeof(Plan) + (size_t)3 * count * 4; }
extern "C" size_t tw_cache_compact_workspace(int pages) { return pages <= 0 ? 0 : sizeof(Plan) + (size_t)3 * pages * 4; }

extern "C" int tw_cache_append(const TwCache* cache, const TwAppendArgs* a, void* workspace, void* stream_) {
  Cache c = {};
  if (const int status = cache_of(cache, c, true)) return status;
  if (!a || !a->k || !a->v || !workspace || a->batch <= 0 || a->rows < 0 || (!a->cu && a->rows != a->batch) || (!a->slots && a->batch > c.sequences))
    return TW_ERR_ARGUMENT;
  if (a->batch > MOST_SEQUENCES) return TW_ERR_TOO_LARGE;
  if (misaligned(a->k, 16) || misaligned(a->v, 16) || (a->k_stride_row | a->k_stride_head | a->v_stride_row | a->v_stride_head) % 8 || misaligned(workspace, 16))
    return TW_ERR_ALIGNMENT;
  Append p = {};
  p.k = static_cast<const __nv_bfloat16*>(a->k); p.v = static_cast<const __nv_bfloat16*>(a->v);
  p.k_row = a->k_stride_row; p.k_head = a->k_stride_head; p.v_row = a->v_stride_row; p.v_head = a->v_stride_head;
  p.slots = a->slots; p.cu = a->cu; p.k_scale = a->k_scale; p.v_scale = a->v_scale;
  p.plan = static_cast<Plan*>(workspace);
  p.base = reinterpret_cast<int*>(p.plan + 1); p.offset = p.base + a->batch; p.fresh = p.offset + a->batch;
  p.batch = a->batch; p.rows = a->rows; p.most_fresh = a->rows; p.dim = cache->dim;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  append_plan_kernel<<<1, PLAN, 0, stream>>>(c, p);
  if (cudaGetLastError() != cudaSuccess) return TW_ERR_LAUNCH;
  const long long blocks = ((long long)a->rows * c.hk * (cache->dim / 8) + 255) / 256;
  if (!blocks) return TW_OK;
  const dim3 grid((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8));
  return cache->fp8 ? launch_after(append_rows_kernel<true>, grid, 256, stream, c, p) : launch_after(append_rows_kernel<false>, grid, 256, stream, c, p);
}

extern "C" int tw_cache_fork(const TwCache* cache, const int32_t* parents, const int32_t* children, int count, void* workspace, void* stream_) {
  Cache c = {};
  if (const int status = cache_of(cache, c, true)) return status;
  if (!parents || !children || !workspace || count <= 0) return TW_ERR_ARGUMENT;
  if (count > MOST_SEQUENCES) return TW_ERR_TOO_LARGE;
  if (misaligned(workspace, 16)) return TW_ERR_ALIGNMENT;
  Fork f = {};
  f.parents = parents; f.children = children; f.count = count;
  f.plan = static_cast<Plan*>(workspace);
  f.tokens = reinterpret_cast<int*>(f.plan + 1); f.fresh = f.tokens + count;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  fork_plan_kernel<<<1, PLAN, 0, stream>>>(c, f);
  if (cudaGetLastError() != cudaSuccess) return TW_ERR_LAUNCH;
  return launch_after(fork_copy_kernel, dim3(count, 2 * c.hk < 64 ? 2 * c.hk : 64), 128, stream, c, f);
}

extern "C" int tw_cache_free(const TwCache* cache, const int32_t* slots, int count, void* stream) {
  Cache c = {};
  if (const int status = cache_of(cache, c, false)) return status;
  if (!slots || count <= 0) return TW_ERR_ARGUMENT;
  free_kernel<<<count, 128, 0, static_cast<cudaStream_t>(stream)>>>(c, slots);
  return cudaGetLastError() == cudaSuccess ? TW_OK : TW_ERR_LAUNCH;
}

extern "C" int tw_cache_compact(const TwCache* cache, int32_t* live, void* workspace, void* stream_) {
  Cache c = {};
  if (const int status = cache_of(cache, c, true)) return status;
  if (!workspace) return TW_ERR_ARGUMENT;
  if (misaligned(workspace, 16)) return TW_ERR_ALIGNMENT;
  Compact m = {};
  m.plan = static_cast<Plan*>(workspace);
  m.source = reinterpret_cast<int*>(m.plan + 1); m.target = m.source + c.pages; m.number = m.target + c.pages;
  m.live = live;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  compact_plan_kernel<<<1, PLAN, 0, stream>>>(c, m);
  if (cudaGetLastError() != cudaSuccess) return TW_ERR_LAUNCH;
  return launch_after(compact_move_kernel, dim3(148 * 8), 256, stream, c, m);
}
