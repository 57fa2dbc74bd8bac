// Products of a few rows with packed NVFP4 weights: y[r, n] = factor * sum_k bf16(x[r, k] d[k]) W[n, k] + bias[n], the form a
// token at a time needs (tw_fused works on M128 tiles and quantizes its activation; here the rows stay bf16).
//
// W is code * group scale, W0 plus the W1 tiles of the bank. A code has 2 significant bits and a scale 4, so their product is
// exact in f16 (2^-10 ... 2688), and the tensor cores multiply f16 exactly into 32-bit sums: m16n8k16 with 16 weight rows as A and
// up to 8 rows of x as B. x is bf16, whose exponents f16 does not have: every CTA scales its part of a row by a power of two
// that brings the largest finite value to [2^14, 2^15). That is exact but for values 2^29 below the largest, whose last
// bits, 2^-39 of the largest, are rounded away, far below the 2^-24 of the sums; the sums are scaled back.
//
// What bounds it is the read of the weights, 9/16 byte each, once. A lane loads 16 bytes of codes (32 of k) of two rows and the two
// scales of each; four lanes cover a K128 block of a row, and each lane's 32 k-values may sit in any k-slot of the
// instruction, because x is laid out alike. A byte of codes is one conversion to two f16 (cvt.rn.f16x2.e2m1x2,
// one per cycle and scheduler measured; masks and shifts take 2.4 times as long) and one packed multiplication by the scale.
// The eight warps of a CTA take the K128 blocks of a 16-row tile in turn, four blocks of each warp in flight, and add
// up in shared memory; a CTA owns consecutive tiles and loads across their borders. Where there are fewer tiles than CTAs fit, or x is too
// large for a CTA's shared memory, the CTAs of a cluster split K and add up through distributed shared memory: no workspace, and
// sums of a fixed order.
#include "tw_common.cuh"
#include "../../include/twb200.h"

namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32, DEPTH = 4;
constexpr int COL_PITCH = 20;       // floats per x row of a warp's 16-row partial tile: bank = 8 t + g, no conflicts
constexpr int MAX_TILES = 64;       // 16-row tiles per CTA; bounds the shared-memory lists of bank tiles

struct Params {
  const __nv_bfloat16* x; long long x_stride;
  const float* prescale;
  const uint8_t *codes, *scales;
  const float* factor;
  const __nv_bfloat16* bias;
  const uint8_t *wr, *wrs;
  const int *off, *wi, *wloc;
  void* out;
  int rows, n, k, kb, tiles, groups, ksplit, slots, entries, shared, dense, out_f32, list_blocks;
};

__device__ __forceinline__ uint4 load_codes(const uint8_t* p) {          // read once: keep it out of L1
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
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
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_load(const float* own, uint32_t rank) {
  uint32_t addr;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(tw::smem_u32(own)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Where a warp is in its sequence of K128 blocks: all W0 blocks of a tile, then the tile's bank blocks, then the next tile.
struct Cursor {
  int tile, at;
};

template <int MT, bool BANK>     // MT: groups of 8 x rows
__global__ void __launch_bounds__(THREADS, 2) matvec_kernel(Params p) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ unsigned peak[32];
  __shared__ float unscale[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = p.ksplit > 1 ? (int)cluster_rank() : 0, group = blockIdx.x / p.ksplit;
  const int kb0 = (int)((long long)p.kb * rank / p.ksplit), nkb = (int)((long long)p.kb * (rank + 1) / p.ksplit) - kb0;
  const int max_kb = (p.kb + p.ksplit - 1) / p.ksplit;
  const int tile0 = (int)((long long)p.tiles * group / p.groups), tile1 = (int)((long long)p.tiles * (group + 1) / p.groups);
  uint4* xs = reinterpret_cast<uint4*>(dynamic);                                  // [max_kb][4 words][rows][4 lanes]
  float* red = reinterpret_cast<float*>(xs + (size_t)max_kb * 16 * p.rows);       // [2][WARPS][8 MT][COL_PITCH]
  float* part = red + 2 * WARPS * 8 * MT * COL_PITCH;                             // [2][8 MT][16], only with ksplit > 1
  int2* list = reinterpret_cast<int2*>(part + (p.ksplit > 1 ? 2 * 8 * MT * 16 : 0));   // [list_blocks][max_kb], only with a bank
  int* counts = reinterpret_cast<int*>(list + (BANK ? (size_t)p.list_blocks * max_kb : 0));
  const int nb0 = tile0 >> 3;

  if (BANK) {
    // the bank tiles of this CTA's N128 blocks that lie in its part of K: {x block, bank position}
    const int last = tile1 > tile0 ? (tile1 - 1) >> 3 : nb0 - 1;
    for (int nb = nb0 + warp; nb <= last; nb += WARPS) {
      int2* mine = list + (size_t)(nb - nb0) * max_kb;
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
        if (take && slot < max_kb) mine[slot] = make_int2(block, loc);
        filled += __popc(who);
      }
      if (lane == 0) counts[nb - nb0] = filled < max_kb ? filled : max_kb;
    }
    __syncthreads();
  }

  // ---- the stream of weight blocks: registers hold DEPTH of them --------------------------------------------------
  uint4 code[DEPTH][2];
  uint32_t scale[DEPTH][2];
  int block_of[DEPTH];                 // x block, or -1 for nothing to add
  bool ends[DEPTH];                    // the warp's last block of the tile
  const int own = nkb > warp ? (nkb - warp + WARPS - 1) / WARPS : 0;              // this warp's W0 blocks of a tile
  Cursor cur{tile0, 0};
  auto fetch = [&](int slot) {
    code[slot][0] = code[slot][1] = make_uint4(0, 0, 0, 0);
    scale[slot][0] = scale[slot][1] = 0;
    block_of[slot] = -1;
    ends[slot] = true;
    if (cur.tile >= tile1) return;
    int steps = own;
    if (BANK) {
      const int count = counts[(cur.tile >> 3) - nb0];
      steps += count > warp ? (count - warp + WARPS - 1) / WARPS : 0;
    }
    if (cur.at < steps) {
      const int row0 = cur.tile * 16 + g;
      if (!BANK || cur.at < own) {
        const int block = warp + cur.at * WARPS, kk = (kb0 + block) * 128 + t * 32;
        block_of[slot] = block;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = row0 + 8 * h;
          if (row < p.n && kk < p.k) {
            code[slot][h] = load_codes(p.codes + (size_t)row * (p.k / 2) + kk / 2);
            scale[slot][h] = __ldg(reinterpret_cast<const uint16_t*>(p.scales + (size_t)row * (p.k / 16) + kk / 16));
          }
        }
      } else {
        const int2 e = list[(size_t)((cur.tile >> 3) - nb0) * max_kb + warp + (cur.at - own) * WARPS];
        block_of[slot] = e.x;
#pragma unroll
        for (int h = 0; h < 2; ++h) {                 // n and k are multiples of 128 with a bank
          const size_t row = (size_t)e.y * 128 + ((row0 + 8 * h) & 127);
          code[slot][h] = load_codes(p.wr + row * 64 + t * 16);
          scale[slot][h] = __ldg(reinterpret_cast<const uint16_t*>(p.wrs + row * 8 + t * 2));
        }
      }
    }
    if (++cur.at >= steps) { ++cur.tile; cur.at = 0; } else ends[slot] = false;
  };
#pragma unroll
  for (int s = 0; s < DEPTH; ++s) fetch(s);

  // ---- x: bf16(x d) to shared memory in the order the lanes read it, then to scaled f16 in place --------------------
  if (threadIdx.x < 32) peak[threadIdx.x] = 0;
  __syncthreads();
  const int chunks = nkb * 16;                                                    // of 8 values
  for (int r = 0; r < p.rows; ++r) {
    unsigned top = 0;
    for (int c = threadIdx.x; c < chunks; c += THREADS) {
      const int kk = kb0 * 128 + c * 8;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (kk < p.k) {                                                             // k % 32 == 0
        v = __ldg(reinterpret_cast<const uint4*>(p.x + r * p.x_stride + kk));
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (p.prescale) {
            const float2 d = __ldg(reinterpret_cast<const float2*>(p.prescale + kk + 2 * i));
            const __nv_bfloat162 b = __floats2bfloat162_rn(__fmul_rn(tw::bf16_bits_to_float(w[i] & 0xffffu), d.x),
                                                           __fmul_rn(tw::bf16_bits_to_float(w[i] >> 16), d.y));
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
          }
          const unsigned lo = (w[i] & 0x7fffu) << 16, hi = w[i] & 0x7fff0000u;
          if (lo < 0x7f800000u) top = max(top, lo);                               // finite values only
          if (hi < 0x7f800000u) top = max(top, hi);
        }
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
      // chunk c of a block: lane t = (c & 15) / 4 holds k 32 t ... 32 t + 31, word i = c & 3 of its 16 bytes of codes
      xs[(size_t)(((c >> 4) * 4 + (c & 3)) * p.rows + r) * 4 + ((c & 15) >> 2)] = v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0 && top) atomicMax(&peak[r], top);
  }
  __syncthreads();
  for (int r = 0; r < p.rows; ++r) {
    // 2^shift brings the largest value to [2^14, 2^15); an all-zero row stays, and 2^shift stays a normal number
    const int shift = peak[r] ? min(14 - ((int)(peak[r] >> 23) - 127), 126) : 0;
    const float up = __uint_as_float((unsigned)(127 + shift) << 23);
    if (threadIdx.x == 0) unscale[r] = __uint_as_float((unsigned)(127 - shift) << 23);
    for (int c = threadIdx.x; c < chunks; c += THREADS) {
      uint4* at = xs + (size_t)(((c >> 4) * 4 + (c & 3)) * p.rows + r) * 4 + ((c & 15) >> 2);
      const uint4 v = *at;
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(tw::bf16_bits_to_float(w[i] & 0xffffu) * up, tw::bf16_bits_to_float(w[i] >> 16) * up);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
      *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __syncthreads();

  // ---- products --------------------------------------------------------------------------------------------------
  const float factor = __ldg(p.factor);
  float acc[MT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
  int tile = tile0, buffer = 0;
  while (tile < tile1) {
#pragma unroll
    for (int s = 0; s < DEPTH; ++s) {
      if (tile < tile1) {
        if (block_of[s] >= 0) {
          __half2 sc[2][2];
          decode_scales(scale[s][0], sc[0][0], sc[0][1]);
          decode_scales(scale[s][1], sc[1][0], sc[1][1]);
          const uint32_t w[2][4] = {{code[s][0].x, code[s][0].y, code[s][0].z, code[s][0].w},
                                    {code[s][1].x, code[s][1].y, code[s][1].z, code[s][1].w}};
          const uint4* xb = xs + (size_t)block_of[s] * 16 * p.rows + lane;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a[2][4];
            decode8(w[0][i], sc[0][i >> 1], a[0]);
            decode8(w[1][i], sc[1][i >> 1], a[1]);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const uint4 b = m * 8 + g < p.rows ? xb[i * 4 * p.rows + m * 32] : make_uint4(0, 0, 0, 0);
              mma_f16(acc[m], a[0][0], a[1][0], a[0][1], a[1][1], b.x, b.y);
              mma_f16(acc[m], a[0][2], a[1][2], a[0][3], a[1][3], b.z, b.w);
            }
          }
        }
        const bool end = ends[s];
        fetch(s);
        if (end) {
          float* mine = red + ((size_t)buffer * WARPS + warp) * 8 * MT * COL_PITCH;
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            float* c = mine + (m * 8 + 2 * t) * COL_PITCH + g;
            c[0] = acc[m][0]; c[COL_PITCH] = acc[m][1]; c[8] = acc[m][2]; c[COL_PITCH + 8] = acc[m][3];
            acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
          }
          __syncthreads();               // the other buffer is written next: one barrier per tile is enough
          float sum[(MT * 128 + THREADS - 1) / THREADS];
#pragma unroll
          for (int o = 0; o < (MT * 128 + THREADS - 1) / THREADS; ++o) {
            const int e = threadIdx.x + o * THREADS, col = e >> 4, row = e & 15;
            sum[o] = 0.f;
            if (col < p.rows) {
              const float* from = red + (size_t)buffer * WARPS * 8 * MT * COL_PITCH + col * COL_PITCH + row;
#pragma unroll
              for (int w8 = 0; w8 < WARPS; ++w8) sum[o] += from[w8 * 8 * MT * COL_PITCH];
              sum[o] *= unscale[col];
              if (p.ksplit > 1) part[buffer * 8 * MT * 16 + e] = sum[o];
            }
          }
          if (p.ksplit > 1) cluster_sync();
#pragma unroll
          for (int o = 0; o < (MT * 128 + THREADS - 1) / THREADS; ++o) {
            const int e = threadIdx.x + o * THREADS, col = e >> 4, row = tile * 16 + (e & 15);
            if (col < p.rows && row < p.n && (p.ksplit == 1 || col % p.ksplit == rank)) {
              float y = sum[o];
              if (p.ksplit > 1) {        // the ranks' sums in their order, whoever adds them
                y = 0.f;
                for (int q = 0; q < p.ksplit; ++q) y += peer_load(part + buffer * 8 * MT * 16 + e, q);
              }
              y *= factor;
              if (p.bias) y += __bfloat162float(p.bias[row]);
              const size_t at = (size_t)col * p.n + row;
              if (p.out_f32) static_cast<float*>(p.out)[at] = y;
              else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
            }
          }
          buffer ^= 1;
          ++tile;
        }
      }
    }
  }
  if (p.ksplit > 1) cluster_sync();      // nobody leaves while its sums may still be read
}

template <int MT, bool BANK>
int launch(const Params& p, size_t smem, cudaStream_t stream) {
  auto kernel = matvec_kernel<MT, BANK>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
    (void)cudaGetLastError();
    return TW_ERR_LAUNCH;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(p.groups * p.ksplit);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = p.ksplit;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = p.ksplit > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, p);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? TW_OK : TW_ERR_LAUNCH;
}

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

}  // namespace

extern "C" int tw_matvec(const TwMatvecArgs* a, void* stream) {
  if (!a || !a->x || !a->codes || !a->scales || !a->factor || !a->out || a->rows <= 0 || a->n <= 0 || a->k <= 0) return TW_ERR_ARGUMENT;
  const bool bank = a->slots > 0;
  if (a->slots < 0 || a->entries < 0 || (bank && (!a->wr || !a->wrs))) return TW_ERR_ARGUMENT;
  if (bank && !a->dense && (!a->off || !a->wi || (a->shared && !a->wloc))) return TW_ERR_ARGUMENT;
  if (a->k % 32 || (bank && (a->n % 128 || a->k % 128))) return TW_ERR_SHAPE;
  if (a->rows > 32 || a->k > 32768) return TW_ERR_TOO_LARGE;
  if (misaligned(a->x, 16) || a->x_stride % 8 || misaligned(a->codes, 16) || misaligned(a->scales, 2) || misaligned(a->factor, 4) ||
      misaligned(a->prescale, 8) || misaligned(a->bias, 2) || misaligned(a->wr, 16) || misaligned(a->wrs, 2) ||
      misaligned(a->out, a->out_f32 ? 4 : 2))
    return TW_ERR_ALIGNMENT;
  Params p = {};
  p.x = static_cast<const __nv_bfloat16*>(a->x); p.x_stride = a->x_stride;
  p.prescale = a->prescale; p.codes = a->codes; p.scales = a->scales; p.factor = a->factor;
  p.bias = static_cast<const __nv_bfloat16*>(a->bias);
  p.wr = a->wr; p.wrs = a->wrs; p.off = a->off; p.wi = a->wi; p.wloc = a->wloc; p.out = a->out;
  p.rows = a->rows; p.n = a->n; p.k = a->k; p.kb = (a->k + 127) / 128; p.tiles = (a->n + 15) / 16;
  p.slots = a->slots; p.entries = a->entries; p.shared = a->shared; p.dense = a->dense; p.out_f32 = a->out_f32;
  // K is split over a cluster until a CTA's part of x leaves room for a second CTA on its SM, and further while the CTAs
  // still fit beside each other and every warp keeps two K128 blocks of a tile
  constexpr int ROOM = 104 * 1024, MOST = 220 * 1024;
  auto bytes = [&](int ksplit, int list_blocks) {
    const int mt = p.rows <= 8 ? 1 : p.rows <= 16 ? 2 : 4;
    const size_t kbs = (p.kb + ksplit - 1) / ksplit;
    return kbs * 256 * p.rows + (size_t)2 * WARPS * 8 * mt * COL_PITCH * 4 + (ksplit > 1 ? (size_t)2 * 8 * mt * 16 * 4 : 0) +
           (bank ? (size_t)list_blocks * (kbs * 8 + 4) : 0);
  };
  if (bytes(8, MAX_TILES / 8 + 2) > MOST) p.rows = 16;       // K > 21 k: more rows go in passes of 16, which always fit
  const int step = p.rows;
  for (int row = 0; row < a->rows; row += step) {
    p.rows = a->rows - row < step ? a->rows - row : step;
    p.x = static_cast<const __nv_bfloat16*>(a->x) + row * a->x_stride;
    p.out = static_cast<uint8_t*>(a->out) + (size_t)row * a->n * (a->out_f32 ? 4 : 2);
    int ksplit = 1;
    while (ksplit < 8 && (bytes(ksplit, MAX_TILES / 8 + 2) > ROOM ||
                          (p.tiles * ksplit * 2 <= 148 * 2 && p.kb >= ksplit * 2 * 2 * WARPS))) ksplit *= 2;
    int groups = 148 * 2 / ksplit;
    if (groups > p.tiles) groups = p.tiles;
    if (groups < (p.tiles + MAX_TILES - 1) / MAX_TILES) groups = (p.tiles + MAX_TILES - 1) / MAX_TILES;
    p.ksplit = ksplit; p.groups = groups;
    p.list_blocks = bank ? ((p.tiles + groups - 1) / groups + 7) / 8 + 1 : 0;
    const size_t smem = bytes(ksplit, p.list_blocks);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int status = p.rows <= 8 ? (bank ? launch<1, true>(p, smem, st) : launch<1, false>(p, smem, st))
                     : p.rows <= 16 ? (bank ? launch<2, true>(p, smem, st) : launch<2, false>(p, smem, st))
                                    : (bank ? launch<4, true>(p, smem, st) : launch<4, false>(p, smem, st));
    if (status) return status;
  }
  return TW_OK;
}
