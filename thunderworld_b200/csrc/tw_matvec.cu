// Products of a few rows with packed NVFP4 weights: y[r, n] = factor * sum_k bf16(x[r, k] d[k]) W[n, k] + bias[n], the form a
// token at a time needs (tw_fused works on M128 tiles and quantizes its activation; here the rows stay bf16).
//
// W is code * group scale, W0 plus the W1 tiles of the bank. A code has 2 significant bits and a scale 4, so their product is
// exact in f16 (2^-10 ... 2688), and the tensor cores multiply f16 exactly into 32-bit sums: m16n8k16 with 16 weight rows as A and
// up to 8 rows of x as B. x is bf16, whose exponents f16 does not have: every CTA scales its part of a row by a power of two
// that brings the largest value to [2^14, 2^15). That is exact but for values 2^29 below the largest, whose last
// bits are rounded away, at most 2^-39 of the largest each: far below the 2^-24 of the sums, unless all weights that the largest meets
// are zero (a second f16 value for the rest would double the products). The sums are scaled back.
//
// What bounds it is the read of the weights, 9/16 byte each, once. A lane loads 16 bytes of codes (32 of k) of two rows and the two
// scales of each; four lanes cover a K128 block of a row, and each lane's 32 k-values may sit in any k-slot of the
// instruction, because x is laid out alike. A byte of codes is one conversion to two f16 (cvt.rn.f16x2.e2m1x2,
// one per cycle and scheduler measured; masks and shifts take 2.4 times as long) and one packed multiplication by the scale.
// A warp owns 16 rows and runs over its CTA's part of K in quads of four blocks, which it copies to a ring of its own in shared
// memory, two quads of 4.6 KB, across the borders of its tiles: two CTAs of eight warps have up to 148 KB per SM on the way. A lane
// copies what it reads itself, so that the copies have immediate offsets: the instructions beside the decoding count (the
// conversions and all integer work share a half-rate pipe). Rows and x columns that do not exist repeat the last one; their
// sums are never read. The CTAs of a cluster hold the parts of K: each stages (and scales) only its part of x, and sends
// its sums of 128 rows to their owners through distributed shared memory, one cluster barrier per 128 rows, waited for after the
// next 128 rows' products. No workspace, no atomics on sums: the order is fixed.
//
// Measured (B200, weights from HBM, graph replay; bytes of the weights over time): 1 x 24576 x 6144 23.3 us (3.7 TB/s), 1 x 12288 x
// 4096 12.6 us, 8 x 16384 x 4096 16.8 us, 16 and 32 rows 21.9 and 35.8 us (a prescale adds 0.5, 1.2, 1.2 and 2.6 us), 5 x 6144 x 24576 with a
// quarter repaired 36 us (3.0 TB/s), 1 x 2048 x 2048 4.9 us. What bounds it: of the 23 us of 24576 x 6144, some 7 are start (launch, instructions from L2, x to f16)
// and join (cluster barriers, cold code); then the decoding and the stream of the weights hide each other in part only: without the
// decoding, or without the copies, it takes 2 us and 1 us less, without both products and decoding 5 us. More warps (24 or 32
// per SM), a third quad on the way, chains of products and x loaded ahead change nothing, the next block's codes ahead cost 1 us.
#include <atomic>
#include "tw_common.cuh"
#include "../../include/twb200.h"

namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int SCALE_PITCH = 40;     // bytes per row of a quad's scales: 32, in up to five aligned words; a load's banks are all different
constexpr int QUAD = 16 * 256 + 16 * SCALE_PITCH;    // bytes of a ring slot: codes by lane, then scales
constexpr int MAX_ROUNDS = 32;      // N128 blocks per cluster; bounds the shared-memory lists of bank tiles
constexpr int MOST_SMEM = 224 * 1024, PAIR_SMEM = 112 * 1024;      // of one CTA on an SM, of each of two

struct Params {
  const __nv_bfloat16* x; long long x_stride;
  const float* prescale;
  const uint8_t *codes, *scales;
  const float* factor;
  const __nv_bfloat16* bias;
  const uint8_t *wr, *wrs;
  const int *off, *wi, *wloc;
  void* out;
  int rows, n, k, kb, nb, groups, ksplit, k_share, k_more, n_share, n_more, slots, entries, shared, dense, out_f32;
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// The first `bytes` (0 ... 8) from global memory, zeros behind them.
__device__ __forceinline__ void copy8(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
// Eight codes -> four f16 pairs, low nibble first.
__device__ __forceinline__ void decode8(uint32_t w, __half2 scale, uint32_t (&o)[4]) {
  asm("{ .reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %4;\n cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d; }"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]) : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&o[i]), scale);
    o[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}
// Two E4M3 bytes -> two f16 pairs, each with one scale in both halves.
__device__ __forceinline__ void decode_scales(uint32_t bytes, __half2& s0, __half2& s1) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)bytes));
  const __half2 h = *reinterpret_cast<const __half2*>(&h2);
  s0 = __low2half2(h);
  s1 = __high2half2(h);
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void peer_store(float* own, uint32_t rank, float v) {      // at the same place of another CTA of the cluster
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(tw::smem_u32(own)), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// Floats of a buffer for a round's sums: as many shares of them as there are ranks, rounded up; even.
__device__ __host__ __forceinline__ int sum_floats(int rows, int ksplit) { return (rows * 128 + ksplit * ksplit + 1) & ~1; }
// Bytes of a row of x in shared memory: a block's 64 chunks of 16 bytes by word of codes and lane, and 64 bytes that put the
// eight rows that a warp reads at once into different banks.
__device__ __host__ __forceinline__ int x_pitch(int blocks) { return blocks * 256 + 64; }
// Where chunk c (8 values: word c & 3 of lane (c & 15) / 4 of block c / 16) of a row lies.
__device__ __forceinline__ int x_chunk(int c) { return (c >> 4) * 256 + (c & 3) * 64 + ((c & 15) >> 2) * 16; }

template <int MT, bool BANK>     // MT: groups of 8 x rows
__global__ void __launch_bounds__(THREADS, 2) matvec_kernel(const __grid_constant__ Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");       // launched while the kernel before it drains; nothing is read until that is through
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ unsigned peak[32];
  __shared__ float unscale[32];
  __shared__ int counts[MAX_ROUNDS];               // bank blocks of a round
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = p.ksplit > 1 ? (int)cluster_rank() : 0, group = p.ksplit > 1 ? (blockIdx.x - rank) / p.ksplit : blockIdx.x;
  // even shares, the first ones one larger: of K by rank, of the N128 blocks by cluster
  const int kb0 = rank * p.k_share + min(rank, p.k_more), nkb = p.k_share + (rank < p.k_more), max_kb = p.k_share + (p.k_more > 0);
  const int nb0 = group * p.n_share + min(group, p.n_more), rounds = p.n_share + (group < p.n_more);
  const int pitch = x_pitch(max_kb);
  uint8_t* ring = dynamic + warp * 2 * QUAD;                                                     // [WARPS][2][QUAD]
  uint8_t* xs = dynamic + WARPS * 2 * QUAD;                                                      // [rows][pitch]
  float* landing = reinterpret_cast<float*>(xs + p.rows * pitch);                                // [2][ranks][rows * 128 / ranks]
  int2* list = reinterpret_cast<int2*>(landing + 2 * sum_floats(p.rows, p.ksplit));              // [rounds][max_kb], only with a bank

  if (p.ksplit > 1) cluster_arrive();              // waited for before the first store to a peer: it has to be running
  // This CTA's part of x on its way to shared memory while the weights' first blocks are fetched. Half a warp takes a K128 block of
  // a row at a time, 8 values a lane, and an even share of them that lie one behind the other, so that rows change seldom.
  const int units = p.rows * nkb, half = threadIdx.x >> 4, chunk = threadIdx.x & 15;
  const int unit0 = half * units / (THREADS / 16), unit_count = (half + 1) * units / (THREADS / 16) - unit0;
  const int first_row = unit0 / nkb, first_kb = unit0 - first_row * nkb;
  auto each_unit = [&](auto&& body) {              // (row, block, last of this share in its row)
    int r = first_row, b = first_kb;
#pragma unroll 1
    for (int u = unit_count; u > 0; --u) {
      const bool last = u == 1 || b + 1 == nkb;
      body(r, b, last);
      if (++b == nkb) { b = 0; ++r; }
    }
  };
  auto x_at = [&](int r, int b) { return reinterpret_cast<uint4*>(xs + r * pitch + b * 256 + x_chunk(chunk)); };
  each_unit([&](int r, int b, bool) {
    const int kk = (kb0 + b) * 128 + chunk * 8;
    if (kk < p.k) copy16(tw::smem_u32(x_at(r, b)), p.x + r * p.x_stride + kk);
    else *x_at(r, b) = make_uint4(0, 0, 0, 0);                                    // k % 32 == 0; zeros behind it
  });
  asm volatile("cp.async.commit_group;" ::: "memory");
  if (threadIdx.x < 32) peak[threadIdx.x] = 0;
  if (BANK) {
    // the bank tiles of this cluster's N128 blocks that lie in this CTA's part of K: {block, bank position}
    for (int j = warp; j < rounds; j += WARPS) {
      const int nb = nb0 + j;
      int filled = 0;
      const int begin = p.dense ? nb * p.kb : max(__ldg(p.off + nb), 0);
      const int end = p.dense ? begin + p.kb : min(__ldg(p.off + nb + 1), p.entries);
      for (int s0 = begin; s0 < end; s0 += 32) {
        const int s = s0 + lane;
        int block = -1, loc = -1;
        if (s < end) {
          block = (p.dense ? s - begin : __ldg(p.wi + s)) - kb0;
          loc = p.shared && !p.dense ? __ldg(p.wloc + s) : s;
        }
        const bool take = block >= 0 && block < nkb && loc >= 0 && loc < p.slots;
        const unsigned who = __ballot_sync(0xffffffffu, take);
        const int slot = filled + __popc(who & ((1u << lane) - 1u));
        if (take && slot < max_kb) list[(size_t)j * max_kb + slot] = make_int2(block, loc);
        filled += __popc(who);
      }
      if (lane == 0) counts[j] = filled < max_kb ? filled : max_kb;
    }
  }
  __syncthreads();

  // ---- the stream of weight blocks: W0's of this part of K, then the bank's, then the next round ----------------------
  // Two cursors run over it quad by quad: one fetches, one, two quads behind, multiplies.
  const size_t code_pitch = p.k / 2, scale_pitch = p.k / 16;
  struct Cursor { int round, at, w0, bank; };      // blocks fetched or multiplied of the round's w0 + bank
  auto open = [&](Cursor& c) {
    c.w0 = c.round < rounds && (nb0 + c.round) * 128 + warp * 16 < p.n ? nkb : 0;
    c.bank = BANK && c.w0 ? counts[c.round] : 0;
    c.at = 0;
  };
  // blocks of the quad that the cursor is at: four, or what is left of W0's or of the bank's
  auto width = [&](const Cursor& c) { return min((!BANK || c.at < c.w0 ? c.w0 : c.w0 + c.bank) - c.at, 4); };
  Cursor in{0, 0, 0, 0};
  // a lane copies the 16 bytes of each block and row that it will read; the scales as the aligned words that hold a row's: words
  // 2 (lane & 1) and one more of row lane / 2, and, where rows do not begin on one, the fifth word of row lane
  const uint32_t ring_at = tw::smem_u32(ring), code_to = ring_at + lane * 16;
  const uint32_t scale_to = ring_at + 4096 + (lane >> 1) * SCALE_PITCH + (lane & 1) * 16, fifth_to = ring_at + 4096 + lane * SCALE_PITCH + 32;
  const bool fifth = scale_pitch % 8 && lane < 16;
  // lanes whose 32 k of the last block lie behind K repeat the block's first 32 (x is zero there)
  const int last_block = p.kb - 1 - kb0, tail = last_block < nkb && (kb0 + last_block) * 128 + t * 32 >= p.k ? t * 16 : 0;
  // quads before this block have all their words within their rows: four blocks, and where there is a fifth word, another that it lies in
  const int whole = last_block - (scale_pitch % 8 ? 4 : 3);
  const uint8_t *c0, *c8, *s0, *s32;               // where the round's next quad begins for this lane
  auto aligned = [](const uint8_t* at) { return reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(at) & ~(uintptr_t)7); };
  auto point = [&]() {
    const int row0 = (nb0 + in.round) * 128 + warp * 16;
    c0 = p.codes + min(row0 + g, p.n - 1) * code_pitch + kb0 * 64 + t * 16;
    c8 = p.codes + min(row0 + g + 8, p.n - 1) * code_pitch + kb0 * 64 + t * 16;
    s0 = aligned(p.scales + min(row0 + (lane >> 1), p.n - 1) * scale_pitch + kb0 * 8) + (lane & 1) * 16;
    s32 = aligned(p.scales + min(row0 + (lane & 15), p.n - 1) * scale_pitch + kb0 * 8) + 32;
  };
  auto fetch = [&](int slot) {
    const int n = width(in);
    const uint32_t offset = slot * QUAD;
    if (n > 0 && (!BANK || in.at < in.w0)) {
      if (n == 4 && in.at < whole) {                                 // the usual quad
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          copy16(code_to + offset + j * 1024, c0 + j * 64);
          copy16(code_to + offset + j * 1024 + 512, c8 + j * 64);
        }
        copy8(scale_to + offset, s0, 8);
        copy8(scale_to + offset + 8, s0 + 8, 8);
        if (fifth) copy8(fifth_to + offset, s32, 8);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j < n) {
            const int back = in.at + j == last_block ? tail : 0;
            copy16(code_to + offset + j * 1024, c0 + j * 64 - back);
            copy16(code_to + offset + j * 1024 + 512, c8 + j * 64 - back);
          }
        }
        // what lies behind the row's end is zero
        const int row0 = (nb0 + in.round) * 128 + warp * 16;
        auto word = [&](uint32_t to, const uint8_t* from, int r) {
          const long long rest = p.scales + (min(row0 + r, p.n - 1) + 1) * scale_pitch - from;
          const int size = (int)(rest < 0 ? 0 : rest > 8 ? 8 : rest);
          copy8(to + offset, size ? from : p.scales, size);
        };
        word(scale_to, s0, lane >> 1);
        word(scale_to + 8, s0 + 8, lane >> 1);
        if (fifth) word(fifth_to, s32, lane);
      }
      c0 += 256; c8 += 256; s0 += 32; s32 += 32;
    } else if (BANK && n > 0) {                    // n and k are multiples of 128; a bank tile's rows lie one behind the other
      const int2* entry = list + (size_t)in.round * max_kb + in.at - in.w0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j < n) {
          const size_t row = (size_t)entry[j].y * 128 + warp * 16;
          copy16(code_to + offset + j * 1024, p.wr + (row + g) * 64 + t * 16);
          copy16(code_to + offset + j * 1024 + 512, p.wr + (row + g + 8) * 64 + t * 16);
          if (lane < 16) copy8(ring_at + offset + 4096 + lane * SCALE_PITCH + j * 8, p.wrs + (row + lane) * 8, 8);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    in.at += n;
    if (in.at >= in.w0 + in.bank) {    // a round without a block for this warp takes one empty quad all the same
      ++in.round;
      open(in);
      if (in.w0 > 0) point();
    }
  };
  open(in);
  if (in.w0 > 0) point();

  // x d, rounded to bf16, in the order the lanes read it; then scaled f16 in place
  auto stage_x = [&]() {
    float4 d0 = make_float4(1.f, 1.f, 1.f, 1.f), d1 = d0;
    auto load_d = [&](int b) {
      const int kk = (kb0 + b) * 128 + chunk * 8;
      if (kk < p.k) { d0 = __ldg(reinterpret_cast<const float4*>(p.prescale + kk)); d1 = __ldg(reinterpret_cast<const float4*>(p.prescale + kk) + 1); }
    };
    if (p.prescale && unit_count > 0) load_d(first_kb);
    asm volatile("cp.async.wait_group 1;" ::: "memory");         // a thread's own chunks: nobody else reads them before the barrier
    uint32_t top = 0;                    // sizes of two bf16 values
    each_unit([&](int r, int b, bool last) {
      uint4* to = x_at(r, b);
      const uint4 v = *to;
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
      if (p.prescale) {
        const float d[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __nv_bfloat162 b2 = __floats2bfloat162_rn(__fmul_rn(tw::bf16_bits_to_float(w[j] & 0xffffu), d[2 * j]),
                                                          __fmul_rn(tw::bf16_bits_to_float(w[j] >> 16), d[2 * j + 1]));
          w[j] = *reinterpret_cast<const uint32_t*>(&b2);
        }
        *to = make_uint4(w[0], w[1], w[2], w[3]);
        load_d(b + 1 == nkb ? 0 : b + 1);          // the next unit's
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) top = __vmaxu2(top, w[j] & 0x7fff7fffu);
      if (last) {
        // The largest size, infinity among them: a row that holds one is infinite or NaN whatever becomes of its other values. Bits
        // of sizes order like integers; NaN, which would come out on top, counts as infinity.
        const uint32_t most = min(max(top << 16, top & 0xffff0000u), 0x7f800000u);
        if (most) atomicMax(&peak[r], most);
        top = 0;
      }
    });
    __syncthreads();
    int known = -1;
    float up = 0.f;
    each_unit([&](int r, int b, bool) {
      if (r != known) {
        // 2^shift brings the largest value to [2^14, 2^15); an all-zero row stays, and 2^shift stays a normal number
        const int shift = peak[r] ? min(14 - ((int)(peak[r] >> 23) - 127), 126) : 0;
        up = __uint_as_float((unsigned)(127 + shift) << 23);
        if (b == 0 && chunk == 0) unscale[r] = __uint_as_float((unsigned)(127 - shift) << 23);
        known = r;
      }
      uint4* to = x_at(r, b);
      const uint4 v = *to;
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __half2 h = __floats2half2_rn(tw::bf16_bits_to_float(w[j] & 0xffffu) * up, tw::bf16_bits_to_float(w[j] >> 16) * up);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
      *to = make_uint4(w[0], w[1], w[2], w[3]);
    });
    __syncthreads();
  };

  // ---- products --------------------------------------------------------------------------------------------------
  const float factor = __ldg(p.factor);
  constexpr int CHAINS = MT == 1 ? 2 : 1;          // of dependent additions: one per x group, two where there is one group
  float acc[MT][CHAINS][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < CHAINS; ++h) acc[m][h][0] = acc[m][h][1] = acc[m][h][2] = acc[m][h][3] = 0.f;
  const uint8_t* x_lane[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) x_lane[m] = xs + min(m * 8 + g, p.rows - 1) * pitch + t * 16;
  auto multiply = [&](const uint8_t* codes, const uint8_t* low, const uint8_t* high, int block) {
    const uint4 first = *reinterpret_cast<const uint4*>(codes), second = *reinterpret_cast<const uint4*>(codes + 512);
    __half2 sc[2][2];
    decode_scales(*reinterpret_cast<const uint16_t*>(low), sc[0][0], sc[0][1]);
    decode_scales(*reinterpret_cast<const uint16_t*>(high), sc[1][0], sc[1][1]);
    const uint32_t w[2][4] = {{first.x, first.y, first.z, first.w}, {second.x, second.y, second.z, second.w}};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a[2][4];
      decode8(w[0][i], sc[0][i >> 1], a[0]);
      decode8(w[1][i], sc[1][i >> 1], a[1]);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint4 b = *reinterpret_cast<const uint4*>(x_lane[m] + block * 256 + i * 64);
        mma_f16(acc[m][0], a[0][0], a[1][0], a[0][1], a[1][1], b.x, b.y);
        mma_f16(acc[m][CHAINS - 1], a[0][2], a[1][2], a[0][3], a[1][3], b.z, b.w);
      }
    }
  };
  // A round's sums over this CTA's part of K are in `landing`, its owners' share of them from every rank; rank q adds its share,
  // elements (x row, weight row) q * share ..., in the order of the ranks.
  const int elements = p.rows * 128, share = (elements + p.ksplit - 1) / p.ksplit, floats = sum_floats(p.rows, p.ksplit);
  const float per_share = 1.f / (float)share;
  auto join = [&](int done) {
    const float* from = landing + (done & 1) * floats;
    for (int j = threadIdx.x; j < share && rank * share + j < elements; j += THREADS) {
      const int e = rank * share + j, col = e >> 7, row = (nb0 + done) * 128 + (e & 127);
      if (row >= p.n) continue;
      float y = 0.f;
      for (int q = 0; q < p.ksplit; ++q) y += from[q * share + j];
      y *= factor;
      if (p.bias) y += __bfloat162float(p.bias[row]);
      const size_t to = (size_t)col * p.n + row;
      if (p.out_f32) static_cast<float*>(p.out)[to] = y;
      else static_cast<__nv_bfloat16*>(p.out)[to] = __float2bfloat16_rn(y);
    }
  };
  Cursor at{0, 0, 0, 0};
  open(at);
  // One copy of everything: the first two passes only fetch (and stage x between), the others multiply what was fetched two passes
  // before. Code that runs once costs its way from L2, some 7 cycles an instruction.
  for (int pass = 0; rounds > at.round; ++pass) {
    const int slot = pass & 1;
    int n = 0;
    if (pass >= 2) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      n = width(at);
      const uint8_t* codes = ring + slot * QUAD + lane * 16;
      const uint8_t *low = ring + slot * QUAD + 4096 + t * 2 + g * SCALE_PITCH, *high = low + 8 * SCALE_PITCH;
      const bool base = !BANK || at.at < at.w0;
      if (base && scale_pitch % 8) {     // where a row's scales begin within their first aligned word
        const int row = (nb0 + at.round) * 128 + warp * 16 + g;
        low += (min(row, p.n - 1) * (uint32_t)scale_pitch) & 7;
        high += (min(row + 8, p.n - 1) * (uint32_t)scale_pitch) & 7;
      }
      const int2* entry = list + (size_t)at.round * max_kb + at.at - at.w0;
#pragma unroll 1
      for (int j = 0; j < n; ++j, codes += 1024, low += 8, high += 8) multiply(codes, low, high, base ? at.at + j : entry[j].x);
      __syncwarp();
    }
    fetch(slot);
    if (pass == 0) stage_x();
    if (pass < 2) continue;
    at.at += n;
    if (at.at >= at.w0 + at.bank) {
      if (p.ksplit > 1) {                // the barrier of the round before; at first, the one that says that all ranks run
        cluster_wait();
        if (at.round > 0) join(at.round - 1);
      } else if (at.round > 0) {
        __syncthreads();
        join(at.round - 1);
      }
      float* mine = landing + (at.round & 1) * floats;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int col = m * 8 + 2 * t + (h & 1), e = col * 128 + warp * 16 + g + (h >> 1) * 8;
          const float y = CHAINS == 1 ? acc[m][0][h] : acc[m][0][h] + acc[m][CHAINS - 1][h];
          if (col < p.rows) {
            if (p.ksplit > 1) { const int owner = (int)(((float)e + .5f) * per_share); peer_store(mine + rank * share + e - owner * share, owner, y * unscale[col]); }
            else mine[e] = y * unscale[col];
          }
        }
#pragma unroll
        for (int h = 0; h < CHAINS; ++h) acc[m][h][0] = acc[m][h][1] = acc[m][h][2] = acc[m][h][3] = 0.f;
      }
      // the other buffer's readers are through before anyone passes the barrier that follows
      __syncwarp();
      if (p.ksplit > 1) cluster_arrive();
      ++at.round;
      open(at);
    }
  }
  if (p.ksplit > 1) cluster_wait(); else __syncthreads();
  if (rounds > 0) join(rounds - 1);
}

// Clusters of `ksplit` CTAs, one or two CTAs per SM, that run beside each other: asked once per kind, the query takes longer
// than a launch.
int fitting_clusters(int ksplit, int per_sm) {
  static std::atomic<int> known[9][3];
  int n = known[ksplit][per_sm].load(std::memory_order_relaxed);
  if (n) return n;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(148 * 2 * ksplit);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = per_sm == 2 ? PAIR_SMEM : MOST_SMEM;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = ksplit;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = 1;
  if (cudaFuncSetAttribute(matvec_kernel<1, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_SMEM) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, matvec_kernel<1, false>, &config) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    n = 148 * per_sm * 7 / 8 / ksplit;
  }
  known[ksplit][per_sm].store(n, std::memory_order_relaxed);
  return n;
}

size_t smem_bytes(int rows, int kb, int ksplit, int rounds) {        // rounds: with a bank, else 0
  const int kbs = (kb + ksplit - 1) / ksplit;
  return (size_t)WARPS * 2 * QUAD + (size_t)rows * x_pitch(kbs) + (size_t)2 * sum_floats(rows, ksplit) * 4 + (size_t)rounds * kbs * 8;
}

template <int MT, bool BANK>
int launch(Params p, cudaStream_t stream) {
  auto kernel = matvec_kernel<MT, BANK>;
  static std::atomic<bool> configured[64];            // the shared-memory opt-in is a per-device attribute of the function
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) { (void)cudaGetLastError(); return TW_ERR_LAUNCH; }
  if (device >= 64 || !configured[device].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_SMEM) != cudaSuccess) {
      (void)cudaGetLastError();
      return TW_ERR_LAUNCH;
    }
    if (device < 64) configured[device].store(true, std::memory_order_relaxed);
  }
  // The cluster size that leaves a warp the fewest blocks: rounds of 128 rows times blocks per round, a round's barrier and
  // sums counted as MT blocks, the staging of a block of 8 rows of x as one (8 x 16384 x 4096 17.3 us with the barrier as 2 MT, 16.9
  // with MT; 32 x 16384 x 4096 42.4 us with 4 MT, 36.1 with MT). More clusters than run beside each other would wait for the others;
  // one CTA on an SM instead of two has half the warps to hide its latencies.
  int best = 0, best_cost = 1 << 30;
  size_t smem = 0;
  for (int ksplit = 1; ksplit <= 8 && ksplit <= p.kb; ++ksplit) {
    const int kbs = (p.kb + ksplit - 1) / ksplit;
    for (int per_sm = 2; per_sm >= 1; --per_sm) {
      int groups = ksplit == 1 ? 148 * per_sm : fitting_clusters(ksplit, per_sm);
      if (groups > p.nb) groups = p.nb;
      if (groups < (p.nb + MAX_ROUNDS - 1) / MAX_ROUNDS) groups = (p.nb + MAX_ROUNDS - 1) / MAX_ROUNDS;
      const int rounds = (p.nb + groups - 1) / groups;
      const size_t need = smem_bytes(p.rows, p.kb, ksplit, BANK ? rounds : 0);
      if (need > (size_t)(per_sm == 2 ? PAIR_SMEM : MOST_SMEM)) continue;
      const int cost = 8 * rounds * (kbs + MT) + p.rows * kbs;
      if (cost < best_cost) { best = ksplit; best_cost = cost; p.groups = groups; smem = need; }
      break;
    }
  }
  if (!best) return TW_ERR_TOO_LARGE;
  p.ksplit = best;
  p.k_share = p.kb / best; p.k_more = p.kb % best;
  p.n_share = p.nb / p.groups; p.n_more = p.nb % p.groups;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(p.groups * p.ksplit);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = p.ksplit;
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  config.attrs = attributes;
  config.numAttrs = best > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, p);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? TW_OK : TW_ERR_LAUNCH;
}

// Rows of each launch: the fewest even shares of the rows that fit a cluster of 8, since each reads all weights; at most 29 rows of a K of
// 16384, 21 of 24576, 16 of 32768; with a bank 28, 20, 15. (20 x 4096 x 16384 48.6 us as two halves, 41.8 at once; 21 x 6144 x 24576
// 86.1, 77.7; 17 with a quarter repaired 105.3, 90.5.)
int rows_at_once(int rows, int kb, bool bank) {
  int passes = 1, step = rows;
  while (step > 1 && smem_bytes(step, kb, kb < 8 ? kb : 8, bank ? MAX_ROUNDS : 0) > MOST_SMEM) { ++passes; step = (rows + passes - 1) / passes; }
  return step;
}

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

}  // namespace

extern "C" int tw_matvec_launches(int rows, int k, int bank) {
  if (rows <= 0 || rows > 32 || k <= 0 || k % 32 || k > 32768) return 0;
  const int step = rows_at_once(rows, (k + 127) / 128, bank != 0);
  return (rows + step - 1) / step;
}

extern "C" int tw_matvec(const TwMatvecArgs* a, void* stream) {
  if (!a || !a->x || !a->codes || !a->scales || !a->factor || !a->out || a->rows <= 0 || a->n <= 0 || a->k <= 0) return TW_ERR_ARGUMENT;
  const bool bank = a->slots > 0;
  if (a->slots < 0 || a->entries < 0 || (bank && (!a->wr || !a->wrs))) return TW_ERR_ARGUMENT;
  if (bank && !a->dense && (!a->off || !a->wi || (a->shared && !a->wloc))) return TW_ERR_ARGUMENT;
  if (a->k % 32 || (bank && (a->n % 128 || a->k % 128))) return TW_ERR_SHAPE;
  if (a->rows > 32 || a->k > 32768) return TW_ERR_TOO_LARGE;
  if (misaligned(a->x, 16) || a->x_stride % 8 || misaligned(a->codes, 16) || misaligned(a->scales, 8) || misaligned(a->factor, 4) ||
      misaligned(a->prescale, 16) || misaligned(a->bias, 2) || misaligned(a->wr, 16) || misaligned(a->wrs, 8) ||
      misaligned(a->out, a->out_f32 ? 4 : 2))
    return TW_ERR_ALIGNMENT;
  Params p = {};
  p.x = static_cast<const __nv_bfloat16*>(a->x); p.x_stride = a->x_stride;
  p.prescale = a->prescale; p.codes = a->codes; p.scales = a->scales; p.factor = a->factor;
  p.bias = static_cast<const __nv_bfloat16*>(a->bias);
  p.wr = a->wr; p.wrs = a->wrs; p.off = a->off; p.wi = a->wi; p.wloc = a->wloc; p.out = a->out;
  p.rows = a->rows; p.n = a->n; p.k = a->k; p.kb = (a->k + 127) / 128; p.nb = (a->n + 127) / 128;
  p.slots = a->slots; p.entries = a->entries; p.shared = a->shared; p.dense = a->dense; p.out_f32 = a->out_f32;
  const int step = rows_at_once(a->rows, p.kb, bank);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int row = 0; row < a->rows; row += step) {
    p.rows = a->rows - row < step ? a->rows - row : step;
    p.x = static_cast<const __nv_bfloat16*>(a->x) + row * a->x_stride;
    p.out = static_cast<uint8_t*>(a->out) + (size_t)row * a->n * (a->out_f32 ? 4 : 2);
    const int status = p.rows <= 8 ? (bank ? launch<1, true>(p, st) : launch<1, false>(p, st))
                     : p.rows <= 16 ? (bank ? launch<2, true>(p, st) : launch<2, false>(p, st))
                                    : (bank ? launch<4, true>(p, st) : launch<4, false>(p, st));
    if (status) return status;
  }
  return TW_OK;
}
