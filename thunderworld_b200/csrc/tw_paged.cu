// Attention of one new token per sequence over a paged key-value cache:
//   o[b, h] = sum_t softmax_t(scale q[b, h] . k_t) v_t,  t < lengths[slot b],  k_t = k_pages[table[slot, t / page], h / G, t % page]
// for G = hq / hk query heads per key head, head dimension 64 or 128, pages in bf16 or in E4M3 with a scale per key head.
//
// What bounds it is the read of the keys and values, once. The work is cut into units of 64 tokens of one (sequence, key head), 128
// where a row is shorter than 256 bytes, in that order, and the units are shared evenly by the CTAs that run beside each other,
// whatever the lengths (which only the device knows; putting the warps' parts of a sequence together is counted as a few more): a
// CTA's run may begin and end inside a sequence, and what it has of such a one goes to the workspace, unnormalised, with its
// maximum and sum; a second small launch joins these in their order. A call needs no zeroed state and no counter, so calls
// on several streams, and captured ones, do not meet.
// A warp takes 16 (32) of a unit's tokens: it copies their rows (two units ahead) to a ring of its own, multiplies q (the group's heads,
// padded to 16 rows) by the keys, keeps its own running maximum and sum in 32 bits, base 2, and multiplies the probabilities
// by the values on the tensor cores (m16n8k16, 32-bit sums); warps meet only at the end of a sequence. With bf16 pages a
// probability is two bf16 values (8 bits each, off by at most 2^-16 of it), so that rounding it adds nothing to the result's own rounding.
// Both are positive (the first is truncated, the second has 2^-24 of the first added), so that an infinite value gives that infinity, as its
// product with the probability does (NaN where that is below 2^-109 of the warp's running maximum). With E4M3 pages both
// products are in f16, which holds E4M3 exactly, and q is scaled by a power of two per head to the range of f16. There a probability is
// one f16 value, 2^15 times itself: rounded by 2^-12 of itself, a sixteenth of the result's own rounding (a second value would double the
// products of values), and of what lies 2^-29 and more below the warp's running maximum by 2^-40 of that; without the factor everything
// 2^-25 below was lost, where a key with all the weight and a value of zero leaves the result to such tokens.
// Tokens behind a sequence's end, and those of a table entry outside the pool (reported in the status word), are masked
// and read as zeros, whatever lies there.
//
// Measured (B200, pages from HBM, graph replay; both launches; 32 heads on 8 or 4, dim 128): 24 sequences of 0 ... 8192 tokens in pages
// of 16 69.7 us (5.4 TB/s of keys and values), of 4 95 us, of 1 107 us; 48 of up to 16384 with E4M3 pages 67.7 us (4.2 TB/s); one of 100000 tokens
// 76.7 us (5.3 TB/s); 32 of 4096 41.7 us (4.5 TB/s); one of 3840 tokens 13.7 us; 32 of up to 8192 with 32 heads on 2 30.5 us (3.1 TB/s), E4M3 27.3 us;
// 16 of up to 4096 with 32 heads on 32 71.8 us (5.4 TB/s). The large bf16 cases are held by memory (12 warps per SM wait for it, long scoreboard the
// first stall); E4M3 ones by latency: half the bytes per tile for the same chain of products, maxima and exponentials, 1.65 instructions per
// cycle and SM of four; wide groups of 128 channels by two warps per scheduler; small calls by their chain of start, lengths, table, pages,
// warps' join, second launch. The narrow kernels of 128 channels spill 92 and 114 bytes at 168 registers. Three times as many smaller runs, an earlier launch of the join and branch hints changed nothing.
#include <atomic>
#include "tw_common.cuh"
#include "../../include/twb200.h"

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int SMS = 148;
// CTAs per SM: three, so of at most 168 registers a thread; two where 16 query rows of 128 channels need more than that (up to 252;
// 32 sequences of 8192 tokens, 32 heads on 2: 47.9 us with three, 38.4 with two; E4M3 39.8, 31.0). 16 rows of 64 channels fit
// (64 sequences 34.9 us with three, 37.7 with two).
__host__ __device__ constexpr int ctas_per_sm(int dim, bool wide) { return wide && dim == 128 ? 2 : 3; }
// Tokens of a warp's tile: 16 of 256-byte rows, 32 of shorter ones: the instructions beside the products are per tile (48 sequences of
// E4M3 pages 82.4 us with 16, 77.3 us with 32), and 32 of 256 bytes would take the shared memory of a CTA.
__host__ __device__ constexpr int tile_tokens(int row_bytes) { return row_bytes >= 256 ? 16 : 32; }
constexpr int JOIN_ROWS = 4;        // query rows that a CTA's warps put together at a time
// Steps, of a unit each, that putting the warps' parts of a sequence together is counted as: the more rows and channels, the more. 1, 2,
// 3, 6 steps: 24 ragged sequences, 4 rows per key head 75.3, 69.0, 69.8, 70.1 us; 48 E4M3 ones of 8 rows 79.1, 69.1, 67.0, 69.4; 32 of up
// to 8192 tokens and 16 rows 39.9, 38.5, 37.9, 30.2, with 64 channels (64 of them) 38.7, 35.6, 33.7, 34.2.
constexpr int MOST_JOINING = 6;
inline int joining_of(int rows, int dim) { return rows <= JOIN_ROWS ? 2 : rows <= 2 * JOIN_ROWS || dim == 64 ? 3 : MOST_JOINING; }

struct Params {
  const __nv_bfloat16* q; long long q_batch, q_head;
  const uint8_t *k, *v; long long k_page, k_head, v_page, v_head;     // strides in bytes
  const int *table; long long table_stride;
  const int *lengths, *slots;
  const float *k_scale, *v_scale;
  __nv_bfloat16* out; float* lse;
  int4* borders;                    // [grid] what to join where a CTA's run begins: number of parts (0: nothing), first part, head, rows
  float *part_o, *part_ml;          // [grid][2][rows][dim], [grid][2][rows][2]
  int* status;
  float scale_log2;
  int batch, sequences, hk, group, tiles, heads, page_shift, pages, max_pages, rows, joining, grid;   // tiles of 16 query rows per key head; heads = hk * tiles
};

__device__ __forceinline__ void report(const Params& p) { if (p.status) atomicMax(p.status, (int)TW_ERR_PAGE); }
// Tokens of batch entry b.
__device__ __forceinline__ int tokens_of(const Params& p, int b, int& slot) {
  slot = p.slots ? __ldg(p.slots + b) : b;
  if (slot < 0 || slot >= p.sequences) { report(p); slot = 0; return 0; }
  const int n = __ldg(p.lengths + slot);
  const long long most = (long long)p.max_pages << p.page_shift;
  if (n < 0 || n > most) { report(p); return n < 0 ? 0 : (int)most; }
  return n;
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t e4m3_to_f16(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  return h;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// What probabilities and their sums are multiplied by, as a power of two; the sums of parts carry it to the end, where it cancels.
__host__ __device__ constexpr int p_shift(bool fp8) { return fp8 ? 15 : 0; }
// Weight of a part whose maximum is m among parts whose largest is top; nothing is left of a part without tokens.
__device__ __forceinline__ float weight_of(float m, float top) { return m == -INFINITY ? 0.f : exp2_fast(m - top); }

// Natural log of a softmax's sum, from the maximum and the sum in base 2.
template <bool FP8>
__device__ __forceinline__ float lse_of(float top, float sum) {
  return sum == 0.f ? -INFINITY : (top + log2f(sum * (1.f / (1 << p_shift(FP8))))) * 0.693147180559945f;
}

// Place of 16-byte chunk c of row r in a tile of rows of CHUNKS chunks: what eight lanes read at once lies in different banks.
template <int CHUNKS> __device__ __forceinline__ int swizzled(int c, int r) { return CHUNKS == 4 ? c ^ (r >> 1 & 3) : c ^ (r & 7); }

// Shares of `all` steps: the first all % owners owners have a step more than the others.
// An owner per SM before any has two steps, then no more owners than have two: a second CTA on an SM for one step, and its part to join,
// cost more than they take off the others (1 x 3840 tokens, 8 key heads, 15.2 with an owner per step, 14.2 us; 1 x 30000, one key head
// of 64 channels, 17.0, 13.8; 1 x 16384, 32 heads on one, 29.0, 24.5; at least four steps: 14.5, 14.7, 26.2).
struct Shares {
  int all, owners, per, more;
  __device__ __forceinline__ Shares(int all_, int grid) : all(all_), owners(min(max(all_ - all_ / 2, min(all_, SMS)), grid)) { per = owners ? all / owners : 0; more = all - per * owners; }
  __device__ __forceinline__ int begin(int c) const { return c * per + min(c, more); }
  __device__ __forceinline__ int owner(int u) const { return u < more * (per + 1) ? u / (per + 1) : more + (u - more * (per + 1)) / per; }
};
// Where a warp is in its CTA's run: one cursor fetches, one multiplies. A sequence's steps are its units and, last, the joining of
// its parts. What changes with the sequence only is kept in shared memory (every lane writes the same): registers are what
// the kernel has least of.
struct Sequence { int b, h, kv, slot, tokens; };
struct Cursor {
  int left, tile, units;                           // steps left of the run; tile of the sequence's units
  Sequence* of;
};

// WIDE: more than 8 query heads per key head; else the upper 8 of a tile's 16 rows do not exist, and nothing is computed for them
// (maxima, exponentials and sums are half of a tile's arithmetic).
template <int D, bool FP8, bool WIDE>
__global__ void __launch_bounds__(THREADS, ctas_per_sm(D, WIDE)) paged_attention_kernel(const __grid_constant__ Params p) {
  constexpr int ROW = D * (FP8 ? 1 : 2), CHUNKS = ROW / 16, TOK = tile_tokens(ROW), SUBS = TOK / 16, UNIT = WARPS * TOK;
  constexpr int SUB = 16 * ROW, TILE = SUBS * SUB;         // bytes of 16 tokens' rows, of a tile's
  constexpr uint32_t ALL = TOK == 32 ? 0xffffffffu : 0xffffu;
  constexpr int STAGES = 2, HALVES = WIDE ? 2 : 1;
  constexpr float LESS = -1.f + 1.f / (1 << 24);           // x + LESS hi: what is left of x, and 2^-24 hi
  extern __shared__ __align__(128) uint8_t dynamic[];                             // [WARPS][STAGES][K, V][TOK rows], from a multiple of 256
  __shared__ float gather[WARPS * JOIN_ROWS * D];
  __shared__ float part_m[WARPS][16], part_l[WARPS][16];
  __shared__ float2 joined[16];
  __shared__ int sums[WARPS + 1], start_b, start_offset;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  auto units_of = [](int tokens) { return (tokens + UNIT - 1) / UNIT; };
  if (threadIdx.x == 0) start_b = start_offset = 0;

  // ---- this CTA's run: the lengths' prefix sums, in units -----------------------------------------------------------
  const int per = (p.batch + THREADS - 1) / THREADS, first_b = min(threadIdx.x * per, p.batch), last_b = min(first_b + per, p.batch);
  int mine = 0, slot_unused;
  for (int b = first_b; b < last_b; ++b) { const int n = units_of(tokens_of(p, b, slot_unused)); mine += n ? n + p.joining : 0; }
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += x; }
  if (lane == 31) sums[warp] = before;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) { if (w == warp) before += total - mine; total += sums[w]; }
  const Shares shares(total * p.heads, p.grid);
  // rows of empty sequences, dealt out over the CTAs
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (tokens_of(p, b, slot_unused)) continue;
    const long long head0 = (long long)b * p.hk * p.group, heads = p.hk * p.group;
    for (long long e = threadIdx.x; e < heads * D; e += THREADS) p.out[head0 * D + e] = __float2bfloat16_rn(0.f);
    if (p.lse) for (int e = threadIdx.x; e < heads; e += THREADS) p.lse[head0 + e] = -INFINITY;
  }
  if ((int)blockIdx.x >= shares.owners) {
    if (threadIdx.x == 0) p.borders[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  const int step0 = shares.begin(blockIdx.x);
  for (int b = first_b, at = before * p.heads; b < last_b; ++b) {
    const int n = units_of(tokens_of(p, b, slot_unused)), steps = n ? (n + p.joining) * p.heads : 0;
    if (at <= step0 && step0 < at + steps) { start_b = b; start_offset = step0 - at; }
    at += steps;
  }
  __syncthreads();

  __shared__ Sequence sequences[2][WARPS];
  // To the next sequence, if the cursor is behind the units of its own. Every lane finds it in registers and writes what it found once,
  // the same as the others: between two warp barriers, so that no lane reads what another has yet to write, or writes what another reads.
  auto settle = [&](Cursor& c) {
    if (c.tile < c.units) return;
    c.left -= c.units + p.joining - c.tile;          // the joining steps, or what the run has of them
    c.tile = 0;
    int b = c.of->b, h = c.of->h + 1, slot = 0, tokens = 0;
    const bool enters = h == p.heads && c.left > 0;
    if (h == p.heads) h = 0;
    if (enters) {
      // (the bounds matter only if somebody changes the lengths meanwhile)
      do c.units = units_of(tokens = tokens_of(p, b = min(b + 1, p.batch - 1), slot)); while (c.units == 0 && b + 1 < p.batch);
    }
    __syncwarp();
    if (enters) {
      c.of->b = b;
      c.of->slot = slot;
      c.of->tokens = tokens;
    }
    c.of->h = h;
    c.of->kv = h / p.tiles;
    __syncwarp();
  };
  auto advance = [&](Cursor& c) { --c.left; ++c.tile; settle(c); };

  // ---- copies: a tile's rows of K and of V to the warp's ring ---------------------------------------------
  // rows begin at multiples of 256, so that a chunk's place in its row can be had by exclusive or
  const uint32_t ring = ((tw::smem_u32(dynamic) + 255) & ~255u) + warp * STAGES * 2 * TILE;
  constexpr int LANES = CHUNKS, STEP = 32 / LANES, COPIES = 16 / STEP;            // lanes per row, rows per instruction
  constexpr int PLACES = STEP >= 8 ? 1 : 8 / STEP;                                // different swizzles of a lane's chunks
  const int copy_row = lane / LANES, copy_chunk = lane % LANES;
  uint32_t place[PLACES];
#pragma unroll
  for (int i = 0; i < PLACES; ++i) place[i] = copy_row * ROW + swizzled<CHUNKS>(copy_chunk, i * STEP + copy_row) * 16;
  Cursor in;
  in.left = shares.begin(blockIdx.x + 1) - step0;
  in.of = &sequences[0][warp];
  int start_slot;
  const int start_tokens = tokens_of(p, start_b, start_slot);
  in.units = units_of(start_tokens);
  const int start_h = min(start_offset / (in.units + p.joining), p.heads - 1);       // below it, unless the lengths have changed
  in.tile = start_offset - start_h * (in.units + p.joining);
  *in.of = Sequence{start_b, start_h, start_h / p.tiles, start_slot, start_tokens};
  __syncwarp();
  settle(in);                          // a run that begins with a joining step leaves it to the owner of the sequence's last unit
  Cursor at = in;
  at.of = &sequences[1][warp];
  *at.of = *in.of;
  __syncwarp();
  if (threadIdx.x == 0) {
    // A run that begins inside a sequence, the first one to: the parts are the last of the run before (its first, if that begins
    // with the sequence, or with the joining step before it), and the first of every run from this one to the owner of the sequence's last unit.
    int4 border = make_int4(0, 0, 0, 0);
    if (in.left > 0 && in.tile > 0) {
      const int begin = step0 - in.tile, previous = shares.begin((int)blockIdx.x - 1), row0 = (in.of->h - in.of->kv * p.tiles) * 16;
      if (previous <= begin)
        border = make_int4(min(shares.owner(begin + in.units - 1), p.grid - 1) - (int)blockIdx.x + 2, ((int)blockIdx.x - 1) * 2 + (previous < begin - p.joining ? 1 : 0),
                           (in.of->b * p.hk + in.of->kv) * p.group + row0, min(p.group - row0, 16));
    }
    p.borders[blockIdx.x] = border;
  }
  const int in_page = (1 << p.page_shift) - 1;
  int next_page[SUBS];                 // where the tokens lie that are fetched next: looked up a tile ahead
  auto look_up = [&]() {
    const int t0 = (in.tile * WARPS + warp) * TOK;
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      next_page[u] = 0;
      if (p.page_shift >= 4 && t0 + u * 16 < in.of->tokens)
        next_page[u] = __ldg(p.table + in.of->slot * p.table_stride + ((t0 + u * 16) >> p.page_shift));
    }
  };
  look_up();
  // the queries of the sequence entered, to where they are had quickly when its turn comes: a line per lane
  auto warm = [&]() {
    const int kv = in.of->kv, row = (in.of->h - kv * p.tiles) * 16 + (lane >> 1);
    if (row < p.group && (D == 128 || !(lane & 1)))
      asm volatile("prefetch.global.L1 [%0];" ::"l"(p.q + in.of->b * p.q_batch + (long long)(kv * p.group + row) * p.q_head + (lane & 1) * 64));
  };
  // Starts the copies of the next tile; returns which of its tokens count.
  auto fetch = [&](uint32_t to) -> uint32_t {
    uint32_t all_mask = 0;
    const int t0 = (in.tile * WARPS + warp) * TOK;
    if (in.left > 0 && t0 < in.of->tokens) {
      const int kv = in.of->kv, left = in.of->tokens - t0;
#pragma unroll
      for (int u = 0; u < SUBS; ++u) {
        const int live = min(left - u * 16, 16);
        uint32_t mask = 0;
        const uint32_t sub = to + u * SUB;
        if (p.page_shift >= 4) {       // 16 tokens lie in one page, one behind the other
          const bool inside = next_page[u] >= 0 && next_page[u] < p.pages;
          if (!inside && lane == 0) report(p);
          const long long page = inside ? next_page[u] : 0, row = (long long)((t0 + u * 16) & in_page) * ROW + lane * 16;
          const uint8_t *k = p.k + page * p.k_page + kv * p.k_head + row, *v = p.v + page * p.v_page + kv * p.v_head + row;
          if (inside && live > 0) mask = 0xffffu >> (16 - live);
          if (mask == 0xffffu) {
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
              copy16(sub + place[i % PLACES] + i * 512, k + i * 512);
              copy16(sub + TILE + place[i % PLACES] + i * 512, v + i * 512);
            }
          } else {
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
              const bool valid = mask >> (i * STEP + copy_row) & 1u;
              copy16(sub + place[i % PLACES] + i * 512, valid ? k + i * 512 : p.k, valid ? 16 : 0);
              copy16(sub + TILE + place[i % PLACES] + i * 512, valid ? v + i * 512 : p.v, valid ? 16 : 0);
            }
          }
        } else {
          const int* entries = p.table + in.of->slot * p.table_stride;
#pragma unroll
          for (int i = 0; i < COPIES; ++i) {
            const int r = i * STEP + copy_row, token = t0 + u * 16 + r;
            bool valid = r < live;
            const long long page = valid ? __ldg(entries + (token >> p.page_shift)) : 0;
            if (page < 0 || page >= p.pages) { report(p); valid = false; }
            // one bit per row, from the first lane of each row
            const uint32_t votes = __ballot_sync(0xffffffffu, valid);
#pragma unroll
            for (int j = 0; j < STEP; ++j) mask |= (votes >> (j * LANES) & 1u) << (i * STEP + j);
            const long long row = (long long)(token & in_page) * ROW + copy_chunk * 16;
            copy16(sub + place[i % PLACES] + i * 512, valid ? p.k + page * p.k_page + kv * p.k_head + row : p.k, valid ? 16 : 0);
            copy16(sub + TILE + place[i % PLACES] + i * 512, valid ? p.v + page * p.v_page + kv * p.v_head + row : p.v, valid ? 16 : 0);
          }
        }
        all_mask |= mask << (u * 16);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (in.left > 0) {
      advance(in);
      if (in.left > 0) {
        look_up();
        if (in.tile == 0) warm();
      }
    }
    return all_mask;
  };
  if (in.left > 0) warm();
  uint32_t stage = ring, mask = fetch(ring), next_mask = fetch(ring + 2 * TILE);

  // ---- products -----------------------------------------------------------------------------------------------------
  uint32_t q[D / 16][4];               // A fragments; with E4M3 pages lane t holds channels 4 t ... 4 t + 3 of each 16
  float o[D / 8][4], m[2], l[2], score_scale[2];
  bool first_segment = true, fresh = true;
  const bool begins_inside = at.tile != 0;
  // Lane addresses of the fragment loads, of a tile at address 0; chunk 2 j of a row is 32 j further, by exclusive or.
  // keys: tokens 0-7 and 8-15 (lane / 16) of channels 16 j ... + 7 and + 8 ... + 15 (lane / 8 % 2); values: tokens 0-7 and 8-15
  // (lane / 8 % 2) of chunks 2 c and 2 c + 1 (lane / 16)
  const int key_row = (lane & 7) + (lane >> 4) * 8, value_row = lane & 15;
  const uint32_t key_lane = key_row * ROW + swizzled<CHUNKS>(lane >> 3 & 1, key_row) * 16;
  const uint32_t value_lane = value_row * ROW + swizzled<CHUNKS>(lane >> 4, value_row) * 16;
  const uint32_t fp8_lane = g * ROW + swizzled<CHUNKS>(0, g) * 16 + t * 4;       // row g + 8 has the same swizzle
  while (at.left > 0) {
      if (fresh) {
        fresh = false;
        const int kv = at.of->kv, row0 = (at.of->h - kv * p.tiles) * 16;
        const __nv_bfloat16* base = p.q + at.of->b * p.q_batch + (long long)(kv * p.group + row0) * p.q_head;
        const bool low = row0 + g < p.group, high = row0 + g + 8 < p.group;
        const __nv_bfloat16 *r0 = base + g * p.q_head, *r1 = base + (g + 8) * p.q_head;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          const int c = FP8 ? j * 16 + t * 4 : j * 16 + t * 2, d = FP8 ? 2 : 8;
          q[j][0] = low ? __ldg(reinterpret_cast<const uint32_t*>(r0 + c)) : 0u;
          q[j][1] = high ? __ldg(reinterpret_cast<const uint32_t*>(r1 + c)) : 0u;
          q[j][2] = low ? __ldg(reinterpret_cast<const uint32_t*>(r0 + c + d)) : 0u;
          q[j][3] = high ? __ldg(reinterpret_cast<const uint32_t*>(r1 + c + d)) : 0u;
        }
        const float k_scale = p.k_scale ? __ldg(p.k_scale + kv) : 1.f;
        score_scale[0] = score_scale[1] = p.scale_log2 * k_scale;
        if (FP8) {
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {              // rows g and g + 8 to the range of f16, as the largest finite value says
            unsigned top = 0;
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t w = q[j][h + 2 * i], lo = (w & 0x7fffu) << 16, hi = w & 0x7fff0000u;
                top = max(top, max(lo < 0x7f800000u ? lo : 0u, hi < 0x7f800000u ? hi : 0u));
              }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int shift = top ? min(14 - ((int)(top >> 23) - 127), 126) : 0;
            const float up = __uint_as_float((unsigned)(127 + shift) << 23);
            score_scale[h] *= __uint_as_float((unsigned)(127 - shift) << 23);
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t w = q[j][h + 2 * i];
                q[j][h + 2 * i] = pack_f16(tw::bf16_bits_to_float(w & 0xffffu) * up, tw::bf16_bits_to_float(w >> 16) * up);
              }
          }
        }
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
      }

      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      __syncwarp();
      if (mask) {
        float s[TOK / 8][4];
#pragma unroll
        for (int n = 0; n < TOK / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          if (FP8) {
#pragma unroll
            for (int n = 0; n < TOK / 8; ++n) {
              uint32_t w;
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(((stage + fp8_lane) ^ (j * 16)) + n * 8 * ROW) : "memory");
              mma<true>(s[n], q[j], e4m3_to_f16(w & 0xffffu), e4m3_to_f16(w >> 16));
            }
          } else {
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
              uint32_t b[4];
              ldsm4(b, ((stage + key_lane) ^ (j * 32)) + u * SUB);
              mma<false>(s[u * 2], q[j], b[0], b[1]);
              mma<false>(s[u * 2 + 1], q[j], b[2], b[3]);
            }
          }
        }
        // scores in base 2; row g in elements 0 and 1, row g + 8 in 2 and 3; tokens 8 n + 2 t and the next
        float top[2] = {m[0], m[1]};
#pragma unroll
        for (int n = 0; n < TOK / 8; ++n)
#pragma unroll
          for (int i = 0; i < 2 * HALVES; ++i) s[n][i] *= score_scale[i >> 1];
        if (mask != ALL) {
#pragma unroll
          for (int n = 0; n < TOK / 8; ++n)
#pragma unroll
            for (int i = 0; i < 2 * HALVES; ++i)
              if (!(mask >> (n * 8 + t * 2 + (i & 1)) & 1u)) s[n][i] = -INFINITY;
        }
        bool higher = false;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
#pragma unroll
          for (int n = 0; n < TOK / 8; ++n) top[h] = fmaxf(top[h], fmaxf(s[n][2 * h], s[n][2 * h + 1]));
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
          higher = higher || top[h] > m[h];
        }
        if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            const float a = weight_of(m[h], top[h]);
            m[h] = top[h];
            l[h] *= a;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) { o[n][2 * h] *= a; o[n][2 * h + 1] *= a; }
          }
        }
        const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0] - p_shift(FP8), m[1] == -INFINITY ? 0.f : m[1] - p_shift(FP8)};
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
          uint32_t hi[4] = {}, lo[4] = {};                // probabilities as an A fragment: rows g, g + 8; tokens 2 t, 2 t + 8
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int h = i & 1, n = u * 2 + (i >> 1);
            if (h < HALVES) {
              const float x = exp2_fast(s[n][h * 2] - ref[h]), y = exp2_fast(s[n][h * 2 + 1] - ref[h]);
              l[h] += x + y;
              if (FP8) {
                hi[i] = pack_f16(x, y);
              } else {
                const uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
                hi[i] = __byte_perm(xb, yb, 0x7632);
                lo[i] = pack_bf16(__fmaf_rn(__uint_as_float(xb & 0xffff0000u), LESS, x), __fmaf_rn(__uint_as_float(yb & 0xffff0000u), LESS, y));
              }
            }
          }
#pragma unroll
          for (int c = 0; c < CHUNKS / 2; ++c) {
            uint32_t b[4];
            ldsm4_trans(b, ((stage + TILE + value_lane) ^ (c * 32)) + u * SUB);
            if (FP8) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {               // a chunk's 16 channels: the even ones and the odd ones
                const uint32_t x = b[2 * h], y = b[2 * h + 1];
                mma<true>(o[c * 4 + h * 2], hi, e4m3_to_f16(__byte_perm(x, 0, 0x4420)), e4m3_to_f16(__byte_perm(y, 0, 0x4420)));
                mma<true>(o[c * 4 + h * 2 + 1], hi, e4m3_to_f16(__byte_perm(x, 0, 0x4431)), e4m3_to_f16(__byte_perm(y, 0, 0x4431)));
              }
            } else {
              mma<false>(o[c * 2], hi, b[0], b[1]);
              mma<false>(o[c * 2], lo, b[0], b[1]);
              mma<false>(o[c * 2 + 1], hi, b[2], b[3]);
              mma<false>(o[c * 2 + 1], lo, b[2], b[3]);
            }
          }
        }
      }
      __syncwarp();
      mask = next_mask;
      next_mask = fetch(stage);
      stage = 2 * ring + 2 * TILE - stage;               // the other one

      const bool last = at.tile + 1 == at.units;
      if (last || at.left == 1) {
        // ---- the sequence's, or the run's, end: the warps' parts together -------------------------------------------
        const bool whole = last && !(first_segment && begins_inside);
        const int kv = at.of->kv, row0 = (at.of->h - kv * p.tiles) * 16, rows = min(p.group - row0, 16);
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
          l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
          if (t == 0) { part_m[warp][g + 8 * h] = m[h]; part_l[warp][g + 8 * h] = l[h]; }
        }
        __syncthreads();
        float own[HALVES];                                // weight of this warp's part
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          const int r = g + 8 * h;
          const float top = fmaxf(fmaxf(part_m[0][r], part_m[1][r]), fmaxf(part_m[2][r], part_m[3][r]));
          own[h] = weight_of(m[h], top);
          if (warp == 0 && t == 0) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) sum += weight_of(part_m[w][r], top) * part_l[w][r];
            joined[r] = make_float2(top, sum);
          }
        }
        const float v_scale = p.v_scale ? __ldg(p.v_scale + kv) : 1.f;
        for (int r0 = 0; r0 < rows; r0 += JOIN_ROWS) {
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            const int r = g + 8 * h - r0;
            if (r >= 0 && r < JOIN_ROWS) {
              float* to = gather + (warp * JOIN_ROWS + r) * D;
#pragma unroll
              for (int n = 0; n < D / 8; ++n) {
                // E4M3: tiles 2 c and 2 c + 1 hold the even and odd channels of chunk c
                const int d0 = FP8 ? (n >> 1) * 16 + t * 4 + (n & 1) : n * 8 + t * 2, d1 = d0 + (FP8 ? 2 : 1);
                to[d0] = o[n][2 * h] * own[h];
                to[d1] = o[n][2 * h + 1] * own[h];
              }
            }
          }
          __syncthreads();
#pragma unroll 1
          for (int e = threadIdx.x; e < min(rows - r0, JOIN_ROWS) * D; e += THREADS) {
            const int r = r0 + e / D, d = e % D;
            const float2 ml = joined[r];
            float y = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) y += gather[w * JOIN_ROWS * D + e];
            if (whole) {
              const long long head = (long long)at.of->b * p.hk * p.group + kv * p.group + row0 + r;
              p.out[head * D + d] = __float2bfloat16_rn(ml.y == 0.f ? 0.f : y * v_scale / ml.y);
              if (p.lse && d == 0) p.lse[head] = lse_of<FP8>(ml.x, ml.y);
            } else {
              const long long slot = ((long long)blockIdx.x * 2 + (first_segment ? 0 : 1)) * p.rows + r;
              p.part_o[slot * D + d] = y;
              if (d == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = ml;
            }
          }
          __syncthreads();
        }
        first_segment = false;
        fresh = true;
      }
      advance(at);
  }
}

// Joins what several CTAs have of one (sequence, head tile): a block per border between two runs and query row, whose warps take the
// parts in turn. (One row and eight warps a block: 1 x 3840 tokens 14.7 us in all; four rows and four warps each 15.6, sixteen warps 14.8.)
constexpr int JOIN_WARPS = 8;
template <int D, bool FP8>
__global__ void __launch_bounds__(JOIN_WARPS * 32) paged_join_kernel(const __grid_constant__ Params p) {
  constexpr int VEC = D / 32;                              // channels of a lane
  struct __align__(VEC * 4) Channels { float v[VEC]; };
  __shared__ Channels sums[JOIN_WARPS][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");       // the parts are written
  const int4 border = p.borders[blockIdx.x + 1];
  const int share = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.y, parts = border.x;
  if (parts == 0 || r >= border.w) return;
  // the first part is border.y, the others are the first ones of the runs that follow
  auto slot_of = [&](int i) { return ((long long)(i == 0 ? border.y : (border.y | 1) + 2 * i - 1) * p.rows + r); };
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  float top = -INFINITY, sum = 0.f;
  for (int i = lane; i < parts; i += 32) {
    const float2 x = ml[slot_of(i)];
    const float higher = fmaxf(top, x.x);
    sum = sum * weight_of(top, higher) + x.y * weight_of(x.x, higher);
    top = higher;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, top, o), more = __shfl_xor_sync(0xffffffffu, sum, o), higher = fmaxf(top, other);
    sum = sum * weight_of(top, higher) + more * weight_of(other, higher);
    top = higher;
  }
  Channels y = {};
#pragma unroll 8
  for (int i = share; i < parts; i += JOIN_WARPS) {
    const Channels o = *reinterpret_cast<const Channels*>(p.part_o + slot_of(i) * D + lane * VEC);
    const float w = weight_of(ml[slot_of(i)].x, top);
#pragma unroll
    for (int j = 0; j < VEC; ++j) y.v[j] += w * o.v[j];
  }
  sums[share][lane] = y;
  __syncthreads();
  if (share) return;
#pragma unroll
  for (int q = 1; q < JOIN_WARPS; ++q)
#pragma unroll
    for (int j = 0; j < VEC; ++j) y.v[j] += sums[q][lane].v[j];
  const long long head = border.z + r;
  const int kv = (border.z / p.group) % p.hk;
  const float scale = p.v_scale ? __ldg(p.v_scale + kv) : 1.f;
#pragma unroll
  for (int j = 0; j < VEC; j += 2)
    *reinterpret_cast<uint32_t*>(p.out + head * D + lane * VEC + j) = sum == 0.f ? 0u : pack_bf16(y.v[j] * scale / sum, y.v[j + 1] * scale / sum);
  if (p.lse && lane == 0) p.lse[head] = lse_of<FP8>(top, sum);
}

int part_rows(int hq, int hk) { return hq / hk < 16 ? hq / hk : 16; }
// CTAs that run beside each other, or as many as there may be units.
int grid_of(int batch, int hq, int hk, int dim, long long tokens) {
  const long long tiles = (hq / hk + 15) / 16, unit = WARPS * tile_tokens(256);          // the shortest unit
  const long long most = (long long)batch * hk * tiles * ((tokens + unit - 1) / unit + joining_of(part_rows(hq, hk), dim)), fit = SMS * ctas_per_sm(dim, hq / hk > 8);
  return (int)(most < 1 ? 1 : most < fit ? most : fit);
}

template <int D, bool FP8, bool WIDE>
int launch(const Params& p, cudaStream_t stream) {
  constexpr int ROW = D * (FP8 ? 1 : 2), SMEM = WARPS * 2 * 2 * tile_tokens(ROW) * ROW + 256;
  static std::atomic<bool> configured[64];            // the shared-memory opt-in is a per-device attribute of the function
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) { (void)cudaGetLastError(); return TW_ERR_LAUNCH; }
  if (device >= 64 || !configured[device].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(paged_attention_kernel<D, FP8, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) {
      (void)cudaGetLastError();
      return TW_ERR_LAUNCH;
    }
    if (device < 64) configured[device].store(true, std::memory_order_relaxed);
  }
  paged_attention_kernel<D, FP8, WIDE><<<p.grid, THREADS, SMEM, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return TW_ERR_LAUNCH;
  if (p.grid == 1) return TW_OK;
  // the join's launch overlaps the end of the first kernel; it waits for it before it reads anything
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(p.grid - 1, p.rows);
  config.blockDim = dim3(JOIN_WARPS * 32);
  config.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  if (cudaLaunchKernelEx(&config, paged_join_kernel<D, FP8>, p) != cudaSuccess) { (void)cudaGetLastError(); return TW_ERR_LAUNCH; }
  return TW_OK;
}

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

}  // namespace

extern "C" size_t tw_paged_attention_workspace(int batch, int hq, int hk, int dim, long long tokens) {
  if (batch <= 0 || hk <= 0 || hq <= 0 || hq % hk || dim <= 0 || tokens < 0) return 0;
  return (size_t)grid_of(batch, hq, hk, dim, tokens) * (16 + 2 * part_rows(hq, hk) * (dim + 2) * 4);
}

extern "C" int tw_paged_attention(const TwPagedAttentionArgs* a, void* stream) {
  if (!a || !a->q || !a->k_pages || !a->v_pages || !a->table || !a->lengths || !a->out || !a->workspace || a->batch <= 0 || a->sequences <= 0 ||
      a->hq <= 0 || a->hk <= 0 || a->hq % a->hk || a->page <= 0 || a->pages <= 0 || a->max_pages <= 0)
    return TW_ERR_ARGUMENT;
  if ((a->dim != 64 && a->dim != 128) || (a->page & (a->page - 1))) return TW_ERR_SHAPE;
  const long long tokens = (long long)a->max_pages * a->page;
  const int tiles = (a->hq / a->hk + 15) / 16, heads = a->hk * tiles;
  if (a->page > (1 << 20) || tokens > (1LL << 30) || (long long)a->batch * heads > (1 << 30) ||
      (long long)a->batch * heads * (tokens / (WARPS * tile_tokens(256)) + 1 + MOST_JOINING) > (1LL << 31) - 1)
    return TW_ERR_TOO_LARGE;
  const int bytes = a->fp8 ? 1 : 2;
  if (misaligned(a->q, 4) || (a->q_stride_batch | a->q_stride_head) & 1 || misaligned(a->k_pages, 16) || misaligned(a->v_pages, 16) ||
      ((a->k_stride_page | a->k_stride_head | a->v_stride_page | a->v_stride_head) * bytes) % 16 || misaligned(a->workspace, 16) ||
      misaligned(a->out, 4) || misaligned(a->table, 4) || misaligned(a->lengths, 4))
    return TW_ERR_ALIGNMENT;
  Params p = {};
  p.q = static_cast<const __nv_bfloat16*>(a->q); p.q_batch = a->q_stride_batch; p.q_head = a->q_stride_head;
  p.k = static_cast<const uint8_t*>(a->k_pages); p.v = static_cast<const uint8_t*>(a->v_pages);
  p.k_page = a->k_stride_page * bytes; p.k_head = a->k_stride_head * bytes;
  p.v_page = a->v_stride_page * bytes; p.v_head = a->v_stride_head * bytes;
  p.table = a->table; p.table_stride = a->table_stride; p.lengths = a->lengths; p.slots = a->slots;
  p.k_scale = a->k_scale; p.v_scale = a->v_scale;
  p.out = static_cast<__nv_bfloat16*>(a->out); p.lse = a->lse; p.status = a->status;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.batch = a->batch; p.sequences = a->sequences; p.hk = a->hk; p.group = a->hq / a->hk; p.tiles = tiles; p.heads = heads;
  p.pages = a->pages; p.max_pages = a->max_pages; p.rows = part_rows(a->hq, a->hk); p.joining = joining_of(p.rows, a->dim);
  p.grid = grid_of(a->batch, a->hq, a->hk, a->dim, tokens);
  while ((1 << p.page_shift) < a->page) ++p.page_shift;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.borders = reinterpret_cast<int4*>(ws);
  p.part_ml = reinterpret_cast<float*>(p.borders + p.grid);
  p.part_o = p.part_ml + (size_t)p.grid * 2 * p.rows * 2;                 // 16-byte aligned, as part_ml
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.rows <= 8) {
    if (a->dim == 128) return a->fp8 ? launch<128, true, false>(p, st) : launch<128, false, false>(p, st);
    return a->fp8 ? launch<64, true, false>(p, st) : launch<64, false, false>(p, st);
  }
  if (a->dim == 128) return a->fp8 ? launch<128, true, true>(p, st) : launch<128, false, true>(p, st);
  return a->fp8 ? launch<64, true, true>(p, st) : launch<64, false, true>(p, st);
}
