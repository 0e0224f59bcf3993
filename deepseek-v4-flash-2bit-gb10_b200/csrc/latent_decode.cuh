// What the two kernels of absorbed latent attention share: a block's share of the work, the preparation of the query rows
// and the joining of the parts.
#pragma once
#include "vq2_common.cuh"

namespace vq2 {

constexpr int LD_TILE = 64;             // cached rows a tile

struct LdArgs {
  vq2_latent_decode_args a;
  int rb;               // bytes of a cached row
  int nrb;              // blocks of NQ query rows a sequence
  int grid;             // blocks that share the tiles
  uint32_t page_mul, page_shift;   // j / page_size = (j * mul) >> 32 >> shift (or j >> shift where mul is 0)
  int* start;           // [B + 1] first position of each sequence
  float2* ml;           // [parts][NQ] maximum and denominator of a part
  float* part;          // [parts][L][NQ]; a block's part of query block n is number n + block
  uint8_t* q;           // [query blocks][units][NQ][128 bytes] rotated query rows, fp16, swizzled (for fp16 then their remainders)
  float2* meta;         // [query blocks][NQ] factor of a row's logits, and its token (as int bits)
};

// Wait that ends early once any thread of the block has given up; it never leaves the caller's loop,
// so every thread keeps to the same sequence of block barriers. The block's last lines report the abort.
__device__ __forceinline__ void ld_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  for (uint32_t i = 1; !mbar_try_wait(bar, parity); ++i)
    if ((i & 63) == 0 && (*abort || i >= VQ2_WAIT_LIMIT)) {
      *abort = 1;
      return;
    }
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
struct LdStart {
  int b, rb, tile;
  __device__ __forceinline__ LdPos position(const LdArgs& g) const {
    LdPos p;
    p.at(g, b);
    p.rb = rb;
    p.tile = tile;
    return p;
  }
};

// A block's share of the tiles: returns their number and leaves in `start` (shared memory, valid after the caller's next block
// barrier) where they begin. Each of the first 32 WARPS threads sums a run of sequences, a scan gives the runs' first
// positions, and the thread whose run holds the block's first tile walks to it. Block 0 writes the sequences' positions for
// the join kernel. Every thread of the block calls it.
template <int WARPS>
__device__ __forceinline__ int ld_share(const LdArgs& g, int* scan, LdStart* start) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int B = g.a.B, run = (B + WARPS * 32 - 1) / (WARPS * 32);
  const int r0 = min(B, tid * run), r1 = warp < WARPS ? min(B, r0 + run) : r0;
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
  if (lane == 31 && warp < WARPS) scan[warp] = inc;
  __syncthreads();
  int before = inc - mine, total = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
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
    start->b = b;
    start->rb = (begin - p) / pos.tiles;
    start->tile = (begin - p) % pos.tiles;
  }
  return count;
}

// The pages of a tile's rows, two rows a lane of a warp, and then the rows' places in the cache.
struct LdRows {
  int j[2], page_at[2], page[2];
  __device__ __forceinline__ void find(const LdArgs& g, const LdPos& p) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      j[k] = p.tile * LD_TILE + (threadIdx.x & 31) + 32 * k;
      page_at[k] = (int)(g.page_mul ? __umulhi((uint32_t)j[k], g.page_mul) >> g.page_shift : (uint32_t)j[k] >> g.page_shift);
      page[k] = j[k] < p.len ? __ldg(g.a.block_table + (size_t)p.b * g.a.max_pages + page_at[k]) : -1;
    }
  }
  // Byte offset of row k of this lane, -1 where there is none; a page outside the cache is reported.
  __device__ __forceinline__ long long offset(const LdArgs& g, const LdPos& p, int k) const {
    const bool in = page[k] >= 0 && page[k] < g.a.pages;
    if (!in && j[k] < p.len) set_status(VQ2_ERR_SHAPE);
    return in ? ((long long)page[k] * g.a.page_size + (j[k] - page_at[k] * g.a.page_size)) * g.rb : -1;
  }
};


// Query rows, one warp a row: latent part rotated, all scaled into fp16's range by a power of two. Written as swizzled units of
// NQ rows x 64 values, or (OPERANDS, 16 rows) as the left operands of m16n8k16 products. Rounding a rotated fp16 row to fp16 would cost
// as much as rounding the output (2e-4 of it each), so its remainders follow as a second term: in fp16, or (OPERANDS) in their upper
// 8 bits, whose 3 significant ones leave 2^-14 of the row. A bf16 output rounds 8 times coarser and needs none, nor does the rotary part
// (only scaled).
constexpr int LQ_WARPS = 4;
template <int DT, int NQ, bool OPERANDS>
__global__ void __launch_bounds__(LQ_WARPS * 32) latent_query_kernel(LdArgs g) {
  pdl_launch_dependents();
  const vq2_latent_decode_args& a = g.a;
  const int lane = threadIdx.x & 31, L = a.latent_dim, R = a.rope_dim, nl = L / 64, units = nl + (R ? 1 : 0), rows = a.T * a.heads;
  const int at = blockIdx.x * LQ_WARPS + (threadIdx.x >> 5), item = at / NQ, r = at % NQ;          // query block, row in it
  const int b = item / g.nrb, row = item % g.nrb * NQ + r;
  const size_t q0 = ((size_t)b * rows + row) * (L + R);
  float v[3][8], m = 0.f;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int u = k < 2 ? lane + 32 * k : lane;          // 8-value unit: of the latent part, of the rotary part
#pragma unroll
    for (int i = 0; i < 8; ++i) v[k][i] = 0.f;
    if (row < rows && u * 8 < (k < 2 ? L : R)) load8<DT>(a.q, q0 + (k < 2 ? 0 : L) + u * 8, v[k]);
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (k < 2) fwht64_lanes8(v[k]);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[k][i]));
  }
  const float2 f = f16_range_scale(fminf(warp_max(m), 3.0e38f));
  constexpr bool TWO = DT == VQ2_DT_F16;
  const size_t bytes = (size_t)units * (NQ * 128);
  uint8_t* dst = g.q + item * bytes * (TWO ? 2 : 1);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int u = k < 2 ? lane + 32 * k : lane, unit = k < 2 ? u >> 3 : nl, c = u & 7;
    if (!(k < 2 ? u * 8 < L : R && u < 8)) continue;
    const uint32_t w[4] = {pack2<VQ2_DT_F16>(v[k][0] * f.x, v[k][1] * f.x), pack2<VQ2_DT_F16>(v[k][2] * f.x, v[k][3] * f.x),
                           pack2<VQ2_DT_F16>(v[k][4] * f.x, v[k][5] * f.x), pack2<VQ2_DT_F16>(v[k][6] * f.x, v[k][7] * f.x)};
    uint32_t rest[4] = {};
    if (TWO && k < 2)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 h = __half22float2(*(const __half2*)&w[j]);
        rest[j] = pack2<VQ2_DT_F16>(v[k][2 * j] * f.x - h.x, v[k][2 * j + 1] * f.x - h.y);
      }
    if (OPERANDS) {
      // piece 2 unit + c / 4, lane 4 (r mod 8) + c mod 4; values 0-1 and 2-3 are registers r / 8 and r / 8 + 2 of its first product
#pragma unroll
      for (int j = 0; j < 4; ++j)
        ((uint32_t*)dst)[(((2 * unit + (c >> 2)) * 2 + (j >> 1)) * 32 + (r & 7) * 4 + (c & 3)) * 4 + (r >> 3) + 2 * (j & 1)] = w[j];
      if (TWO && k < 2)
#pragma unroll
        for (int j = 0; j < 4; ++j)      // rounded to the upper 8 bits of each half
          ((uint16_t*)(dst + bytes))[(((2 * unit + (c >> 2)) * 2 + (j >> 1)) * 32 + (r & 7) * 4 + (c & 3)) * 4 + (r >> 3) + 2 * (j & 1)] =
              (uint16_t)__byte_perm(rest[j] + 0x00800080u, 0, 0x0031);
    } else {
      const size_t to = (size_t)unit * (NQ * 128) + r * 128 + ((c ^ (r & 7)) << 4);
      *(uint4*)(dst + to) = make_uint4(w[0], w[1], w[2], w[3]);
      if (TWO && k < 2) *(uint4*)(dst + bytes + to) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
    }
  }
  // a row that pads the block sees nothing
  if (lane == 0)
    g.meta[at] = make_float2(a.scale * 1.4426950408889634f * f.y, __int_as_float(row < rows ? row / a.heads : -(1 << 30)));
}

// Adds up the parts of a query block, divides and rotates; writes zeros for empty sequences. A block takes 64 values of 8 query
// rows: a warp every WARPS-th part (a lane reads the 8 rows' values side by side, a sector) with a running maximum of its own, then
// the warps' sums are joined in their order. With a pass for the maxima first there is one more round trip to memory, which is
// most of the time where a query block has few parts. WARPS is 16 where it has many, 4 otherwise (64 query blocks of 5 parts: 48 us
// for the whole call, 53 us with 16 warps; 2 query blocks of 148 parts: 45 us, 78 us with 8).
template <int DT, int NQ, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) latent_join_kernel(LdArgs g) {
  __shared__ float buf[WARPS][8][65];
  __shared__ float mx[WARPS][8], den[WARPS][8];
  pdl_wait();
  const vq2_latent_decode_args& a = g.a;
  const int L = a.latent_dim, rows = a.T * a.heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = blockIdx.x % (NQ / 8) * 8, d0 = blockIdx.x / (NQ / 8) % (L / 64) * 64, item = blockIdx.x / (NQ / 8) / (L / 64);
  const int b = item / g.nrb, rb = item % g.nrb;
  if (rb * NQ + r0 >= rows) return;
  // (reads through L2: this kernel may have started while the main one was still writing)
  const int total = __ldcg(g.start + a.B), s0 = __ldcg(g.start + b), s1 = __ldcg(g.start + b + 1);
  const int quota = max(1, (total + g.grid - 1) / g.grid), tiles = (s1 - s0) / g.nrb;
  const int begin = s0 + rb * tiles, c0 = begin / quota, c1 = tiles ? (begin + tiles - 1) / quota : c0 - 1;
  float m[8], l[8], v[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m[i] = -INFINITY;
    l[i] = v[0][i] = v[1][i] = 0.f;
  }
#pragma unroll 2
  for (int c = c0 + warp; c <= c1; c += WARPS) {
    const size_t at = (size_t)(item + c);
    float x[2][8];
    float2 ml[8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float4* p = (const float4*)(g.part + (at * L + d0 + lane + 32 * k) * NQ + r0);
      const float4 y = __ldcg(p), z = __ldcg(p + 1);
      x[k][0] = y.x; x[k][1] = y.y; x[k][2] = y.z; x[k][3] = y.w;
      x[k][4] = z.x; x[k][5] = z.y; x[k][6] = z.z; x[k][7] = z.w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ml[i] = __ldcg(g.ml + at * NQ + r0 + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // a part that saw nothing has maximum -inf and, unless it met a NaN, denominator 0: it changes nothing, a NaN all
      const float n = fmaxf(m[i], ml[i].x);
      const float f = m[i] == n ? 1.f : ex2(m[i] - n), e = ml[i].x == n ? 1.f : ex2(ml[i].x - n);
      m[i] = n;
      l[i] = l[i] * f + ml[i].y * e;
      v[0][i] = v[0][i] * f + x[0][i] * e;
      v[1][i] = v[1][i] * f + x[1][i] * e;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    buf[warp][i][lane] = v[0][i];
    buf[warp][i][lane + 32] = v[1][i];
    if (lane == 0) {
      mx[warp][i] = m[i];
      den[warp][i] = l[i];
    }
  }
  __syncthreads();
  if (tid >= 64) return;
  const int r = tid >> 3, d = (tid & 7) * 8, row = rb * NQ + r0 + r, warps = min(WARPS, max(0, c1 - c0 + 1));
  float q = 0.f, o[8] = {}, n = -INFINITY;
  for (int w = 0; w < warps; ++w) n = fmaxf(n, mx[w][r]);
  for (int w = 0; w < warps; ++w) {
    const float f = mx[w][r] == n ? 1.f : ex2(mx[w][r] - n);
    q = fmaf(den[w][r], f, q);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = fmaf(buf[w][r][d + i], f, o[i]);
  }
  const float inv = q != 0.f ? 1.f / q : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = q != 0.f ? o[i] * inv : 0.f;
  fwht64_lanes8(o);
  if (row < rows) store8<DT>(a.out, ((size_t)b * rows + row) * L + d0 + d, o);
}

}  // namespace vq2
