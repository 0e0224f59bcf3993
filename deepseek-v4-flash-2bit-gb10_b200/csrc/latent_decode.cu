// K8 latent attention, absorbed form: attention of T new tokens a sequence over the 4-bit latent
// cache. For the query row (t, h) of sequence b, with cached rows j = 0 .. kv_len[b] - 1,
//   z_j = scale * (q_c . c_j + q_r . r_j),  j <= kv_len[b] - T + t;   out = sum_j softmax(z)_j c_j
// H is symmetric and H H = I, so q_c . c_j = (H q_c) . (n s)_j and out = H sum_j p_j (n s)_j: the
// kernel rotates the query and the result, never a cached row.
//
// Both products run on tcgen05 with the cached rows as the wide operand and NQ = 16, 32 or 64 query
// rows (heads x tokens of one sequence) as the narrow one, so few heads waste little:
//   S^T [64 cached x NQ] = K Q^T       K tile in shared memory, rows = cached rows (K-major)
//   O^T [L x NQ]        += V^T P^T     the same tile read along the other direction (MN-major): the
//                                      latent is key and value, expanded from 4 bits once for both
// A row is held as n s in fp16, which is exact (|n| <= 7, s has 8 significant bits), q in fp16 with a
// power-of-two scale a row, P in fp16 with its largest values between 2^10 and 2^15, so that values down to
// 2^-34 of the largest still count; sums are fp32 in tensor memory.
//
// Work: the (sequence, block of NQ query rows, tile of 64 cached rows) triples in order, split evenly over one
// block an SM. A block that holds all tiles of a query block writes the result; otherwise it
// leaves its unnormalised sum, maximum and denominator, and the join kernel adds up the parts in order.
// Roles: 8 worker warps load 64 rows ahead into registers, expand them into one of two tiles, and do the softmax
// of the tile before with a thread per cached row and column group; one thread of a ninth warp issues
// S of a tile before P V of the tile before it, so the products run under expansion and softmax.
#include "vq2_common.cuh"

namespace vq2 {

constexpr int LD_TILE = 64;             // cached rows a tile
constexpr int LD_WORKERS = 256, LD_WARPS = LD_WORKERS / 32;
constexpr int LD_THREADS = LD_WORKERS + 128;     // 168 registers each at launch: 256 x 200 + 128 x 104 afterwards
constexpr int LD_UNIT = LD_TILE * 128;  // bytes of a unit of the tile: 64 rows of 64 fp16 values
constexpr int LD_UNITS = 9;             // 8 for the latent, 1 for the rotary part (P takes its place once S is done)
constexpr int LD_KBYTES = LD_UNITS * LD_UNIT;
constexpr float LD_BIAS = 10.f, LD_RAISE = 5.f;    // P = 2^(z - m + BIAS); m is raised when z exceeds it by RAISE

struct LdArgs {
  vq2_latent_decode_args a;
  int rb;               // bytes of a cached row
  int nrb;              // blocks of NQ query rows a sequence
  int grid;             // blocks that share the tiles
  long long capacity;   // cached rows
  uint32_t page_mul, page_shift;   // j / page_size = (j * mul) >> 32 >> shift (or j >> shift where mul is 0)
  int* start;           // [B + 1] first position of each sequence
  float2* ml;           // [2 grid][NQ] maximum and denominator of a part
  float* part;          // [2 grid][NQ][L]
};

template <int NQ>
struct LdShared {
  uint64_t kfull[2], sfull[2], pfull[2], kfree[2], drain;      // by tile buffer
  uint32_t tmem;
  int abort, b0, rb0, tile0;
  long long rows[4][LD_TILE];        // byte offset of a cached row, -1: not there (written two tiles ahead, read until the softmax)
  int bad[2][LD_TILE];               // number of the tile in which this row held a non-finite scale
  float red[4][NQ];
  float fac[NQ];                     // log2-scaled factor of a query row's logits
  float ref[NQ], down[NQ];           // maximum that P and O are relative to; factor of its last change
  float lsum[4][NQ];
  int lim[NQ];                       // cached rows a query row sees
  int scan[LD_WARPS];
};
template <int NQ>
constexpr size_t ld_smem() { return (size_t)2 * LD_KBYTES + (size_t)LD_UNITS * NQ * 128 + sizeof(LdShared<NQ>) + 1024; }
static_assert(ld_smem<64>() <= 227 * 1024, "latent decode shared memory");

// Wait that ends early once any thread of the block has given up; it never leaves the caller's loop,
// so every thread keeps to the same sequence of block barriers.
__device__ __forceinline__ bool ld_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  for (uint32_t i = 0; i < VQ2_WAIT_LIMIT; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63) == 63 && *abort) return false;
  }
  set_status(VQ2_ERR_TIMEOUT);
  *abort = 1;
  return false;
}
__device__ __forceinline__ void ld_sync_workers() { asm volatile("barrier.cta.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void ld_sync_group(int g) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(2 + g) : "memory"); }
__device__ __forceinline__ bool ld_any_group(int g, bool p) {
  uint32_t r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n barrier.cta.red.or.pred q, %1, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
               : "=r"(r) : "r"(2 + g), "r"((uint32_t)p) : "memory");
  return r != 0;
}
template <int N>
__device__ __forceinline__ void ld_tmem_load(uint32_t t, float* v) {
  if (N == 32) tmem_ld32(t, v);
  else if (N == 16) tmem_ld16(t, v);
  else tmem_ld8(t, v);
}
// Position of a tile: sequence, block of query rows, tile; the order is sequence, block, tile.
struct LdPos {
  int b, rb, tile, len, tiles;
  __device__ __forceinline__ void at(const LdArgs& g, int sequence) {
    b = sequence;
    const int most = (int)min((long long)g.a.max_pages * g.a.page_size, 0x7FFFFF00LL);
    len = b < g.a.B ? min(max(g.a.kv_len[b], 0), most) : 0;
    tiles = (len + LD_TILE - 1) / LD_TILE;
  }
  __device__ __forceinline__ void next(const LdArgs& g) {
    if (++tile < tiles) return;
    tile = 0;
    if (++rb < g.nrb) return;
    rb = 0;
    do at(g, b + 1);
    while (tiles == 0 && b < g.a.B);
  }
};

// D += A B with both descriptors at constant offsets from their bases (added in place: otherwise
// the compiler keeps a register for each of the unrolled products).
template <uint32_t A_OFF, uint32_t B_OFF, uint32_t B_HI, uint32_t ID>
__device__ __forceinline__ void umma_at(uint32_t d, uint32_t a, uint32_t b, uint32_t acc) {
  asm volatile("{\n .reg .pred p;\n .reg .b64 x, y;\n .reg .b32 u, v;\n setp.ne.b32 p, %7, 0;\n add.u32 u, %1, %3;\n add.u32 v, %2, %4;\n"
               " mov.b64 x, {u, %5};\n mov.b64 y, {v, %6};\n tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %8, p;\n}"
               ::"r"(d), "r"(a), "r"(b), "n"(A_OFF), "n"(B_OFF), "n"(LP_DESC_HI), "n"(B_HI), "r"(acc), "r"(ID));
}

// The products of a tile, unrolled for each number of units: issued by one thread, with nothing but
// constants added to two addresses, a product takes about 15 cycles to issue (with run-time loops and branches in
// between about 50, which is more than the product itself takes).
template <int NQ, int SU, int I = 0>
__device__ __forceinline__ void ld_scores_n(uint32_t d, uint32_t k, uint32_t q) {
  constexpr uint32_t id = (1u << 4) | ((uint32_t)(NQ >> 3) << 17) | ((uint32_t)(LD_TILE >> 4) << 24);
  constexpr int s = I / 4, ks = I % 4;
  umma_at<s * (LD_UNIT >> 4) + 2 * ks, s * (NQ * 8) + 2 * ks, LP_DESC_HI, id>(d, k, q, I != 0);
  if constexpr (I + 1 < SU * 4) ld_scores_n<NQ, SU, I + 1>(d, k, q);
}
template <int NQ>
__device__ __forceinline__ void ld_scores(int su, uint32_t d, uint32_t k, uint32_t q) {
  k |= 1u << 16;
  q |= 1u << 16;
  switch (su) {
    case 1: return ld_scores_n<NQ, 1>(d, k, q);
    case 2: return ld_scores_n<NQ, 2>(d, k, q);
    case 3: return ld_scores_n<NQ, 3>(d, k, q);
    case 4: return ld_scores_n<NQ, 4>(d, k, q);
    case 5: return ld_scores_n<NQ, 5>(d, k, q);
    case 6: return ld_scores_n<NQ, 6>(d, k, q);
    case 7: return ld_scores_n<NQ, 7>(d, k, q);
    case 8: return ld_scores_n<NQ, 8>(d, k, q);
    default: return ld_scores_n<NQ, 9>(d, k, q);
  }
}
// O^T += V^T P^T: M = 128 latent values a block (the second unit of the last block may be P itself, where the latent has an
// odd number of units: its rows of O^T are not read). P lies as rows of 2 NQ bytes in the swizzle of that width.
template <int NQ, int NB, int I = 0>
__device__ __forceinline__ void ld_values_n(uint32_t d, uint32_t v, uint32_t p, uint32_t acc) {
  constexpr uint32_t id = (1u << 4) | (1u << 15) | (1u << 16) | ((uint32_t)(NQ >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t p_hi = (uint32_t)(16 * NQ >> 4) | 1u << 14 | (NQ == 64 ? 2u : NQ == 32 ? 4u : 6u) << 29;
  constexpr int ks = I / NB, m = I % NB;
  umma_at<m * (2 * LD_UNIT >> 4) + ks * 128, ks * (2 * NQ), p_hi, id>(d + m * NQ, v, p, ks > 0 ? 1 : acc);
  if constexpr (I + 1 < NB * (LD_TILE / 16)) ld_values_n<NQ, NB, I + 1>(d, v, p, acc);
}
template <int NQ>
__device__ __forceinline__ void ld_values(int nblk, uint32_t d, uint32_t tile, int nl, uint32_t acc) {
  const uint32_t v = tile | (LD_UNIT >> 4) << 16, p = (tile + nl * (LD_UNIT >> 4)) | 1u << 16;
  switch (nblk) {
    case 1: return ld_values_n<NQ, 1>(d, v, p, acc);
    case 2: return ld_values_n<NQ, 2>(d, v, p, acc);
    case 3: return ld_values_n<NQ, 3>(d, v, p, acc);
    default: return ld_values_n<NQ, 4>(d, v, p, acc);
  }
}

template <int DT, int NQ>
__global__ void __launch_bounds__(LD_THREADS, 1) latent_decode_kernel(LdArgs g) {
  constexpr int CPT = NQ / 2, CPH = NQ / 4;     // columns of S^T (query rows) a column group has, a softmax thread takes
  constexpr uint32_t COLS = NQ == 64 ? 512 : NQ == 32 ? 256 : 128;    // tensor memory: O^T 4 x NQ columns, S^T 2 x NQ
  extern __shared__ __align__(1024) uint8_t ld_smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)ld_smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t kb = smem_u32(smem), qb = kb + 2 * LD_KBYTES;
  LdShared<NQ>* sh = (LdShared<NQ>*)(smem + 2 * LD_KBYTES + LD_UNITS * NQ * 128);
  const vq2_latent_decode_args& a = g.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int L = a.latent_dim, R = a.rope_dim, nl = L / 64, nblk = (nl + 1) / 2;
  volatile int* abort = &sh->abort;
  pdl_launch_dependents();

  if (tid == 0) {
    for (int k = 0; k < 2; ++k) {
      mbar_init(&sh->kfull[k], 1);
      mbar_init(&sh->sfull[k], 1);
      mbar_init(&sh->pfull[k], 1);
      mbar_init(&sh->kfree[k], 1);
    }
    mbar_init(&sh->drain, 1);
    sh->abort = 0;
    fence_mbar_init();
  }
  if (warp == LD_WARPS) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem)), "r"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid < 2 * LD_TILE) sh->bad[tid >> 6][tid & 63] = -1;

  // ---------------- this block's share of the tiles. Each worker sums a run of sequences, a scan gives
  // the runs' first positions, and the worker whose run holds the block's first tile walks to it.
  const int B = a.B, run = (B + LD_WORKERS - 1) / LD_WORKERS;
  const int r0 = min(B, tid * run), r1 = tid < LD_WORKERS ? min(B, r0 + run) : r0;
  LdPos pos;
  int mine = 0;
  for (int b = r0; b < r1; ++b) {
    pos.at(g, b);
    mine += pos.tiles * g.nrb;
  }
  int inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31 && warp < LD_WARPS) sh->scan[warp] = inc;
  __syncthreads();
  int before = inc - mine, total = 0;
  for (int w = 0; w < LD_WARPS; ++w) {
    if (w < warp) before += sh->scan[w];
    total += sh->scan[w];
  }
  const int quota = max(1, (total + g.grid - 1) / g.grid);
  const int begin = (int)min((long long)blockIdx.x * quota, (long long)total), count = min(quota, total - begin);
  if (blockIdx.x == 0) {
    int p = before;
    for (int b = r0; b < r1; ++b) {
      g.start[b] = p;
      pos.at(g, b);
      p += pos.tiles * g.nrb;
    }
    if (tid == 0) g.start[B] = total;
  }
  if (count > 0 && begin >= before && begin < before + mine) {
    int p = before, b = r0;
    for (;; ++b) {
      pos.at(g, b);
      if (begin < p + pos.tiles * g.nrb) break;
      p += pos.tiles * g.nrb;
    }
    sh->b0 = b;
    sh->rb0 = (begin - p) / pos.tiles;
    sh->tile0 = (begin - p) % pos.tiles;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh->tmem, 0);
  const uint32_t ts = tmem + 4 * NQ;                    // S^T of the two buffers

  if (warp >= LD_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == LD_WARPS && count > 0 && elect_one()) {
      // ---------------- products
      const int su = nl + (R ? 1 : 0);
      LdPos p;
      p.at(g, sh->b0);
      p.rb = sh->rb0;
      p.tile = sh->tile0;
      bool opens = true;             // the tile whose P V comes next is the first of its query block
      auto values = [&](int i) {     // O^T += V^T P^T of tile i
        ld_wait(&sh->pfull[i & 1], (i >> 1) & 1, abort);
        tc_fence_after();
        ld_values<NQ>(nblk, tmem, (kb + (i & 1) * LD_KBYTES) >> 4, nl, opens ? 0 : 1);
        umma_commit(&sh->kfree[i & 1]);
      };
      for (int i = 0; i < count; ++i) {
        const bool first = i == 0 || p.tile == 0;
        // a new query block's tiles come only after the block before is finished
        if (i > 0 && first) {
          values(i - 1);
          opens = true;
        }
        ld_wait(&sh->kfull[i & 1], (i >> 1) & 1, abort);
        tc_fence_after();
        ld_scores<NQ>(su, ts + (i & 1) * NQ, (kb + (i & 1) * LD_KBYTES) >> 4, qb >> 4);
        umma_commit(&sh->sfull[i & 1]);
        if (i > 0 && !first) {
          values(i - 1);
          opens = false;
        }
        p.next(g);
      }
      values(count - 1);
      umma_commit(&sh->drain);
      ld_wait(&sh->drain, 0, abort);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    if (count > 0) {
      // ---------------- workers
      // softmax: S^T's row kr is in tensor-memory lane 32 quarter + (kr & 15); the upper 16 lanes of the warp take
      // half of the column group's columns from the lower ones
      const int quarter = warp & 3, grp = warp >> 2, kr = quarter * 16 + (lane & 15);
      const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
      const int col0 = grp * CPT + (lane >> 4) * CPH;
      LdPos cur, ahead;
      cur.at(g, sh->b0);
      cur.rb = sh->rb0;
      cur.tile = sh->tile0;
      ahead = cur;

      // row offsets of the tile at `p` into buffer `buf` (the first 64 workers)
      auto find_rows = [&](const LdPos& p, int buf) {
        if (tid >= LD_TILE) return;
        const int j = p.tile * LD_TILE + tid;
        long long off = -1;
        if (j < p.len) {
          const uint32_t page_at = g.page_mul ? __umulhi((uint32_t)j, g.page_mul) >> g.page_shift : (uint32_t)j >> g.page_shift;
          const long long page = a.block_table[(size_t)p.b * a.max_pages + page_at];
          if (page < 0 || page >= a.pages) set_status(VQ2_ERR_SHAPE);
          else off = (page * a.page_size + (j - (int)page_at * a.page_size)) * g.rb;
        }
        sh->rows[buf][tid] = off;
      };
      // a tile on its way through registers: 16 lanes take a row's latent in pieces of 32 values, 8 lanes its rotary part
      uint4 lat[4], rope[2];
      uint32_t sc[4];
      const int piece = tid & 15, chunk = tid & 7;
      auto load_rows = [&](int buf) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const long long off = sh->rows[buf][(tid >> 4) + 16 * k];
          lat[k] = make_uint4(0, 0, 0, 0);
          sc[k] = 0;
          if (off >= 0 && piece < 2 * nl) {
            const uint8_t* r = (const uint8_t*)a.cache + off;
            lat[k] = __ldg((const uint4*)r + piece);
            sc[k] = __ldg((const uint16_t*)(r + L / 2 + 2 * R) + (piece >> 1));
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const long long off = sh->rows[buf][(tid >> 3) + 32 * k];
          rope[k] = make_uint4(0, 0, 0, 0);
          if (off >= 0 && chunk * 8 < R) rope[k] = __ldg((const uint4*)((const uint8_t*)a.cache + off + L / 2) + chunk);
        }
      };
      // Registers -> tile. A piece's four words become four 16-byte chunks; the chunks of 8 neighbouring lanes (one row,
      // pieces p .. p + 7) would fall on two bank groups, so each lane starts at another of its words: all eight.
      const int turn = (piece >> 1) & 3;
      auto expand = [&](int number) {
        const uint32_t tile = kb + (number & 1) * LD_KBYTES;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (piece >= 2 * nl) break;
          const int row = (tid >> 4) + 16 * k;
          uint32_t s = sc[k];
          if ((s & 0x7C00u) == 0x7C00u) {       // a non-finite scale: the row reads as NaN, see the softmax
            s = 0;
            sh->bad[number & 1][row] = number;
          }
          const __half2 s2 = __half2half2(__ushort_as_half((unsigned short)s)), c2 = __hmul2(s2, __float2half2_rn(-24.f));
          uint32_t w0 = lat[k].x, w1 = lat[k].y, w2 = lat[k].z, w3 = lat[k].w, t;
          if (turn & 1) { t = w0; w0 = w1; w1 = w2; w2 = w3; w3 = t; }
          if (turn & 2) { t = w0; w0 = w2; w2 = t; t = w1; w1 = w3; w3 = t; }
          const uint32_t w[4] = {w0, w1, w2, w3};
          const uint32_t base = tile + (piece >> 1) * LD_UNIT + row * 128;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            // nibble u = n + 8 in the top mantissa bits of 16 + u; (16 + u) s - 24 s = n s, exact in fp16
            const uint32_t h[4] = {(w[q] << 6 & 0x03C003C0u) | 0x4C004C00u, (w[q] << 2 & 0x03C003C0u) | 0x4C004C00u,
                                   (w[q] >> 2 & 0x03C003C0u) | 0x4C004C00u, (w[q] >> 6 & 0x03C003C0u) | 0x4C004C00u};
            uint4 v;
            __half2 x;
            x = __hfma2(*(const __half2*)&h[0], s2, c2); v.x = *(uint32_t*)&x;
            x = __hfma2(*(const __half2*)&h[1], s2, c2); v.y = *(uint32_t*)&x;
            x = __hfma2(*(const __half2*)&h[2], s2, c2); v.z = *(uint32_t*)&x;
            x = __hfma2(*(const __half2*)&h[3], s2, c2); v.w = *(uint32_t*)&x;
            const int c = (piece & 1) * 4 + ((q + turn) & 3);
            sts128_v(base + ((c ^ (row & 7)) << 4), v);
          }
        }
        if (R) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int row = (tid >> 3) + 32 * k;
            sts128_v(tile + nl * LD_UNIT + row * 128 + ((chunk ^ (row & 7)) << 4), rope[k]);
          }
        }
      };
      // Query rows of block (p.b, p.rb): rotated, scaled to fp16's range by a power of two, into Q's tile; a warp a row.
      auto stage_q = [&](const LdPos& p) {
        for (int r = warp; r < NQ; r += LD_WARPS) {
          const int row = p.rb * NQ + r, rows = a.T * a.heads;
          const size_t at = ((size_t)p.b * rows + row) * (L + R);
          float v[3][8];
          float m = 0.f;
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const int u = k < 2 ? lane + 32 * k : lane;          // 8-value unit: of the latent part, of the rotary part
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = 0.f;
            if (row < rows && u * 8 < (k < 2 ? L : R)) load8<DT>(a.q, at + (k < 2 ? 0 : L) + u * 8, v[k]);
            if (k < 2) fwht64_lanes8(v[k]);
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[k][i]));
          }
          const float2 f = f16_range_scale(fminf(warp_max(m), 3.0e38f));
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const int u = k < 2 ? lane + 32 * k : lane;
            const int unit = k < 2 ? u >> 3 : nl, c = u & 7;
            if (k < 2 ? u * 8 < L : R && u < 8)
              sts128_v(qb + unit * (NQ * 128) + r * 128 + ((c ^ (r & 7)) << 4),
                       make_uint4(pack2<VQ2_DT_F16>(v[k][0] * f.x, v[k][1] * f.x), pack2<VQ2_DT_F16>(v[k][2] * f.x, v[k][3] * f.x),
                                  pack2<VQ2_DT_F16>(v[k][4] * f.x, v[k][5] * f.x), pack2<VQ2_DT_F16>(v[k][6] * f.x, v[k][7] * f.x)));
          }
          if (lane == 0) {
            sh->fac[r] = a.scale * 1.4426950408889634f * f.y;
            sh->lim[r] = row < rows ? max(0, min(p.len, p.len - a.T + 1 + row / a.heads)) : 0;
          }
        }
      };
      float l[CPH];
      // The softmax of tile i at p: logits from tensor memory, P into the rotary unit's place.
      auto softmax = [&](int i, const LdPos& p, bool opens) {
        ld_wait(&sh->sfull[i & 1], (i >> 1) & 1, abort);
        tc_fence_after();
        float z[CPH], ref[CPH];
        {
          float full[CPT];
          ld_tmem_load<CPT>(ts + (i & 1) * NQ + lanes + grp * CPT, full);
#pragma unroll
          for (int c = 0; c < CPH; ++c) {
            const float up = __shfl_sync(0xffffffffu, full[CPH + c], lane & 15);
            z[c] = lane < 16 ? full[c] : up;
          }
        }
        const int j = p.tile * LD_TILE + kr;
        const bool edge = (p.tile + 1) * LD_TILE > p.len - a.T + 1;           // some row sees part of the tile only
        const bool gone = sh->rows[i & 3][kr] < 0;
        bool raise = opens;
#pragma unroll
        for (int c = 0; c < CPH; ++c) {
          z[c] *= sh->fac[col0 + c];
          if (gone || (edge && j >= sh->lim[col0 + c])) z[c] = -INFINITY;
          ref[c] = opens ? -INFINITY : sh->ref[col0 + c];
          raise |= z[c] > ref[c] + LD_RAISE;
        }
        if (sh->bad[i & 1][kr] == i) {
          // the latent is key and value: every query row that sees this one is NaN as a whole; its values
          // were expanded to zeros, so that rows that do not see it are untouched
#pragma unroll
          for (int c = 0; c < CPH; ++c) {
            if (z[c] != -INFINITY) l[c] = __int_as_float(0x7FFFFFFF);
            z[c] = -INFINITY;
          }
        }
        if (ld_any_group(grp, raise)) {
          float f[CPH];
#pragma unroll
          for (int c = 0; c < CPH; ++c) {
            float m = z[c];
#pragma unroll
            for (int o = 8; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if ((lane & 15) == 0) sh->red[quarter][col0 + c] = m;
          }
          // O is rescaled below: every product into it so far has to be done (P V of the tile before)
          if (!opens) ld_wait(&sh->kfree[(i - 1) & 1], ((i - 1) >> 1) & 1, abort);
          tc_fence_after();
          ld_sync_group(grp);
#pragma unroll
          for (int c = 0; c < CPH; ++c) {
            const int k = col0 + c;
            const float m = fmaxf(fmaxf(fmaxf(sh->red[0][k], sh->red[1][k]), fmaxf(sh->red[2][k], sh->red[3][k])), ref[c]);
            f[c] = ref[c] == m ? 1.f : ref[c] == -INFINITY ? 0.f : ex2(ref[c] - m);
            ref[c] = m;
            l[c] = l[c] == 0.f ? 0.f : l[c] * f[c];
          }
          if (quarter == 0 && (lane & 15) == 0)
#pragma unroll
            for (int c = 0; c < CPH; ++c) sh->down[col0 + c] = f[c];
          ld_sync_group(grp);                  // everyone has read the old maxima and the partial ones
          if (!opens)
#pragma unroll 1
            for (int k = 0; k < nblk * (CPT / 8); ++k) {
              const int c8 = grp * CPT + k % (CPT / 8) * 8;
              const uint32_t at = tmem + lanes + k / (CPT / 8) * NQ + c8;
              float o[8];
              tmem_ld8(at, o);
#pragma unroll
              for (int c = 0; c < 8; ++c) o[c] *= sh->down[c8 + c];
              tmem_st8(at, (const uint32_t*)o);
              tmem_st_wait();
              keep_live8((const uint32_t*)o);
            }
          if (quarter == 0 && (lane & 15) == 0)
#pragma unroll
            for (int c = 0; c < CPH; ++c) sh->ref[col0 + c] = ref[c];
        }
        uint32_t ph[CPH / 2];
#pragma unroll
        for (int c = 0; c < CPH; c += 2) {
          const float p0 = ex2(z[c] - ((ref[c] == -INFINITY ? 0.f : ref[c]) - LD_BIAS));
          const float p1 = ex2(z[c + 1] - ((ref[c + 1] == -INFINITY ? 0.f : ref[c + 1]) - LD_BIAS));
          l[c] += p0;
          l[c + 1] += p1;
          ph[c / 2] = pack2<VQ2_DT_F16>(p0, p1);
        }
        // rows of 2 NQ bytes, 16-byte chunks swizzled as the descriptor says
        const uint32_t prow = kb + (i & 1) * LD_KBYTES + nl * LD_UNIT + kr * (2 * NQ), at = col0 * 2;
        if (NQ == 64) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
            sts128_v(prow + ((((at >> 4) + k) ^ (kr & 7)) << 4), make_uint4(ph[4 * k % (CPH / 2)], ph[(4 * k + 1) % (CPH / 2)],
                                                                            ph[(4 * k + 2) % (CPH / 2)], ph[(4 * k + 3) % (CPH / 2)]));
        } else if (NQ == 32) {
          sts128_v(prow + (((at >> 4) ^ ((kr >> 1) & 3)) << 4), make_uint4(ph[0], ph[1], ph[2 % (CPH / 2)], ph[3 % (CPH / 2)]));
        } else {
          asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(prow + (((at >> 4) ^ ((kr >> 2) & 1)) << 4) + (at & 15)), "r"(ph[0]), "r"(ph[1])
                       : "memory");
        }
        fence_async_smem();
        tc_fence_before();
        ld_sync_workers();
        if (tid == 0) mbar_arrive(&sh->pfull[i & 1]);
      };
      // O^T, with its maxima and denominators -> the result, or this block's part of it
      auto finish = [&](const LdPos& p, int seg, bool whole) {
#pragma unroll
        for (int c = 0; c < CPH; ++c) {
          float s = l[c];
#pragma unroll
          for (int o = 8; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          if ((lane & 15) == 0) sh->lsum[quarter][col0 + c] = s;
        }
        ld_sync_workers();
        const int dl = quarter * 32 + lane;       // row of O^T within a block of 128
        if (!whole) {
          const size_t slot = 2 * (size_t)blockIdx.x + (seg > 0);
          if (tid < NQ)
            g.ml[slot * NQ + tid] = make_float2(sh->ref[tid], (sh->lsum[0][tid] + sh->lsum[1][tid]) + (sh->lsum[2][tid] + sh->lsum[3][tid]));
          for (int m = 0; m < nblk; ++m) {
            float o[CPT];
            ld_tmem_load<CPT>(tmem + lanes + m * NQ + grp * CPT, o);
            const int d = m * 128 + dl;
            if (d < L)
#pragma unroll
              for (int c = 0; c < CPT; ++c) g.part[(slot * NQ + grp * CPT + c) * L + d] = o[c];
          }
          return;
        }
        // through shared memory (the tiles are free), 128 values a step, to have a row's group of 64 side by side
        float* buf = (float*)smem;
        constexpr int PITCH = 132;
        for (int m = 0; m < nblk; ++m) {
          float o[CPT];
          ld_tmem_load<CPT>(tmem + lanes + m * NQ + grp * CPT, o);
#pragma unroll
          for (int c = 0; c < CPT; ++c) buf[(grp * CPT + c) * PITCH + dl] = o[c];
          ld_sync_workers();
          for (int u = tid; u < NQ * 16; u += LD_WORKERS) {
            const int r = u >> 4, d = (u & 15) * 8, row = p.rb * NQ + r;
            const float den = (sh->lsum[0][r] + sh->lsum[1][r]) + (sh->lsum[2][r] + sh->lsum[3][r]);
            const float inv = den != 0.f ? 1.f / den : 0.f;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = den != 0.f ? buf[r * PITCH + d + i] * inv : 0.f;
            fwht64_lanes8(v);
            if (row < a.T * a.heads && m * 128 + d < L) store8<DT>(a.out, ((size_t)p.b * a.T * a.heads + row) * L + m * 128 + d, v);
          }
          ld_sync_workers();
        }
      };

      find_rows(ahead, 0);
      ld_sync_workers();
      load_rows(0);
      if (count > 1) {
        ahead.next(g);
        find_rows(ahead, 1);
      }
      int seg = 0;
      bool whole = false, opens = true;        // of the tile before: its query block is all here; it is its first tile
      LdPos prev = cur;
      for (int i = 0; i <= count; ++i) {
        const bool first = i < count && (i == 0 || cur.tile == 0);
        if (i > 0 && (first || i == count)) {  // the query block before ends with tile i - 1
          softmax(i - 1, prev, opens);
          ld_wait(&sh->kfree[(i - 1) & 1], ((i - 1) >> 1) & 1, abort);
          tc_fence_after();
          finish(prev, seg, whole);
          tc_fence_before();
          ++seg;
          if (i < count) ld_sync_workers();
        }
        if (i == count) break;
        if (first) {
          stage_q(cur);
          whole = cur.tile == 0 && i + cur.tiles <= count;
#pragma unroll
          for (int c = 0; c < CPH; ++c) l[c] = 0.f;
        }
        if (i > 1) ld_wait(&sh->kfree[i & 1], ((i >> 1) - 1) & 1, abort);
        expand(i);
        fence_async_smem();
        tc_fence_before();
        ld_sync_workers();
        if (tid == 0) mbar_arrive(&sh->kfull[i & 1]);
        // the next tile's loads go out now and land under the products
        if (i + 1 < count) load_rows((i + 1) & 3);
        if (i + 2 < count) {
          ahead.next(g);
          find_rows(ahead, (i + 2) & 3);
        }
        if (i > 0 && !first) softmax(i - 1, prev, opens);
        opens = first;
        prev = cur;
        cur.next(g);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (warp == LD_WARPS) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS));
}

// Joins the parts of query blocks that several blocks worked on, in order; writes zeros for empty sequences. A thread
// takes 8 values of a query row.
template <int DT, int NQ>
__global__ void __launch_bounds__(256) latent_join_kernel(LdArgs g) {
  pdl_wait();
  const vq2_latent_decode_args& a = g.a;
  const int L = a.latent_dim, U = L / 8, rows = a.T * a.heads;
  const long long idx = (long long)blockIdx.x * 256 + threadIdx.x, row = idx / U;
  const int d = (int)(idx - row * U) * 8;
  const bool in = row < (long long)a.B * rows;
  const int b = in ? (int)(row / rows) : 0, r = in ? (int)(row - (long long)b * rows) : 0;
  const int total = g.start[a.B], quota = max(1, (total + g.grid - 1) / g.grid);
  const int s0 = g.start[b], tiles = (g.start[b + 1] - s0) / g.nrb;
  const int begin = s0 + r / NQ * tiles, end = begin + tiles;
  const int c0 = begin / quota, c1 = tiles ? (end - 1) / quota : c0;
  const bool mine = in && (tiles == 0 || c1 > c0);
  if (!__any_sync(0xffffffffu, mine)) return;
  float v[8] = {}, m = -INFINITY, l = 0.f;
  if (mine && tiles) {
    for (int c = c0; c <= c1; ++c) m = fmaxf(m, g.ml[(2 * c + (c == c0 && begin != c * quota)) * NQ + r % NQ].x);
    for (int c = c0; c <= c1; ++c) {
      const size_t at = (size_t)(2 * c + (c == c0 && begin != c * quota)) * NQ + r % NQ;
      const float2 ml = g.ml[at];
      const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : ex2(ml.x - m);
      l += ml.y * f;
      const float4* p = (const float4*)(g.part + at * L + d);
      const float4 x = p[0], y = p[1];
      v[0] = fmaf(f, x.x, v[0]); v[1] = fmaf(f, x.y, v[1]); v[2] = fmaf(f, x.z, v[2]); v[3] = fmaf(f, x.w, v[3]);
      v[4] = fmaf(f, y.x, v[4]); v[5] = fmaf(f, y.y, v[5]); v[6] = fmaf(f, y.z, v[6]); v[7] = fmaf(f, y.w, v[7]);
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = l != 0.f ? v[i] * inv : 0.f;
  fwht64_lanes8(v);
  if (mine) store8<DT>(a.out, (size_t)row * L + d, v);
}

static int ld_nq(int T, int heads) {
  const long long rows = (long long)T * heads;
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

struct LdLayout {
  size_t start, ml, part, total;
};
static LdLayout ld_layout(int B, int nq, int L, int grid) {
  LdLayout w;
  w.start = 0;
  w.ml = ((size_t)(B + 1) * 4 + 255) / 256 * 256;
  w.part = w.ml + ((size_t)2 * grid * nq * 8 + 255) / 256 * 256;
  w.total = w.part + (size_t)2 * grid * nq * L * 4 + 256;
  return w;
}
constexpr int LD_MAX_GRID = 148;        // workspace is sized without a device; a B200 has 148 SMs

template <int DT, int NQ>
static int ld_launch(const LdArgs& g, cudaStream_t st) {
  auto kernel = latent_decode_kernel<DT, NQ>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ld_smem<NQ>()) != cudaSuccess) return VQ2_ERR_CUDA;
  kernel<<<g.grid, LD_THREADS, ld_smem<NQ>(), st>>>(g);
  if (cudaGetLastError() != cudaSuccess) return VQ2_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  const long long threads = (long long)g.a.B * g.a.T * g.a.heads * (g.a.latent_dim / 8);
  cfg.gridDim = dim3((unsigned)((threads + 255) / 256));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, latent_join_kernel<DT, NQ>, g) == cudaSuccess ? VQ2_OK : VQ2_ERR_CUDA;
}

}  // namespace vq2

using namespace vq2;

extern "C" size_t vq2_latent_decode_workspace_size(int B, int T, int heads, int latent_dim, int rope_dim) {
  if (B <= 0 || T <= 0 || heads <= 0 || !latent_dims_ok(latent_dim, rope_dim)) return 0;
  return ld_layout(B, ld_nq(T, heads), latent_dim, LD_MAX_GRID).total;
}

extern "C" int vq2_latent_decode(const vq2_latent_decode_args* a, void* ws, size_t ws_bytes, void* stream) {
  if (!a || !a->q || !a->cache || !a->block_table || !a->kv_len || !a->out) return VQ2_ERR_NULL;
  if (a->B <= 0 || a->T <= 0 || a->heads <= 0 || a->page_size <= 0 || a->max_pages <= 0 || a->pages <= 0 ||
      !latent_dims_ok(a->latent_dim, a->rope_dim) || !(a->scale > 0.f) || (long long)a->T * a->heads > 1 << 20 ||
      (long long)a->B * a->T * a->heads * (a->latent_dim / 8) / 256 >= 0x7FFFFFFFLL)
    return VQ2_ERR_SHAPE;
  if (a->dtype != VQ2_DT_BF16 && a->dtype != VQ2_DT_F16) return VQ2_ERR_DTYPE;
  if (((uintptr_t)a->q | (uintptr_t)a->cache | (uintptr_t)a->out) & 15) return VQ2_ERR_ALIGN;
  if (!ws || ws_bytes < vq2_latent_decode_workspace_size(a->B, a->T, a->heads, a->latent_dim, a->rope_dim))
    return VQ2_ERR_WORKSPACE;
  LdArgs g = {};
  g.a = *a;
  const int nq = ld_nq(a->T, a->heads), sms = device_sm_count();
  if (sms <= 0) return VQ2_ERR_CUDA;
  g.rb = latent_row_bytes(a->latent_dim, a->rope_dim);
  g.nrb = (a->T * a->heads + nq - 1) / nq;
  g.grid = min(sms, LD_MAX_GRID);
  g.capacity = a->pages * a->page_size;
  // j / page_size for 0 <= j < 2^31: a shift, or with s = ceil(log2 page_size) the high half of j * ceil(2^(31+s) / page_size)
  int s = 0;
  while ((1LL << s) < a->page_size) ++s;
  if ((1LL << s) == a->page_size) {
    g.page_mul = 0;
    g.page_shift = s;
  } else {
    g.page_mul = (uint32_t)(((1ULL << (31 + s)) + a->page_size - 1) / a->page_size);
    g.page_shift = s - 1;
  }
  const LdLayout w = ld_layout(a->B, nq, a->latent_dim, g.grid);
  uint8_t* base = (uint8_t*)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
  g.start = (int*)(base + w.start);
  g.ml = (float2*)(base + w.ml);
  g.part = (float*)(base + w.part);
  cudaStream_t st = (cudaStream_t)stream;
  const bool bf = a->dtype == VQ2_DT_BF16;
  if (nq == 16) return bf ? ld_launch<VQ2_DT_BF16, 16>(g, st) : ld_launch<VQ2_DT_F16, 16>(g, st);
  if (nq == 32) return bf ? ld_launch<VQ2_DT_BF16, 32>(g, st) : ld_launch<VQ2_DT_F16, 32>(g, st);
  return bf ? ld_launch<VQ2_DT_BF16, 64>(g, st) : ld_launch<VQ2_DT_F16, 64>(g, st);
}
