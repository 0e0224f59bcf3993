// K8 latent attention, absorbed form: attention of T new tokens a sequence over the 4-bit latent
// cache. For the query row (t, h) of sequence b, with cached rows j = 0 .. kv_len[b] - 1,
//   z_j = scale * (q_c . c_j + q_r . r_j),  j <= kv_len[b] - T + t;   out = sum_j softmax(z)_j c_j
// H is symmetric and H H = I, so q_c . c_j = (H q_c) . (n s)_j and out = H sum_j p_j (n s)_j: the
// kernel rotates the query and the result, never a cached row.
//
// Both products run on tcgen05 with the cached rows as the wide operand and NQ = 32 or 64 query
// rows (heads x tokens of one sequence) as the narrow one (up to 16 rows, and calls with few tiles, have a kernel of their own: ld_nq):
//   S^T [64 cached x NQ] = K Q^T       K tile in shared memory, rows = cached rows (K-major)
//   O^T [L x NQ]        += V^T P^T     the same tile read along the other direction (MN-major): the
//                                      latent is key and value, expanded from 4 bits once for both
// A row is held as n s in fp16, which is exact (|n| <= 7, s has 8 significant bits), q in fp16 with a
// power-of-two scale a row (fp16 queries in two such terms, both into the same S: see the query kernel), P in fp16 with its largest values between 2^5 and 2^15, so that values down to
// 2^-29 of the largest still count; sums are fp32 in tensor memory.
//
// Work: the (sequence, block of NQ query rows, tile of 64 cached rows) triples in order, split evenly over one
// block an SM; each block leaves, for every query block it worked on, its unnormalised sum, maximum and denominator.
// Three launches, chained by programmatic dependent launch: `query` rotates and scales the query rows once and lays
// them out as the product wants them (in each block, on 8 warps, that took 13,000 cycles a query block), the main kernel, and
// `join`, which adds up the parts in order and rotates the result.
// Roles: a loader warp brings in the cached rows as they are, one bulk copy a row (loads through
// L1 have too few lines to be in flight beside 220 KB of shared memory); 16 worker warps expand a tile of 64 rows and do its softmax;
// one thread issues the products. Both products are bound by reading the tile from shared memory, so that
// path is kept busy: a tile is handed over in parts of 128 latent values, S starts on the first part, and
// a part is filled again as soon as P V has used it. With 32 query rows in one term (bf16) there is room for two tiles, and the softmax of
// a tile runs under the products of the next. In the steady state no barrier spans the block.
// What bounds it: with 64 query rows, or 32 in two terms (fp16), there is room for one tile, so its expansion, S, softmax and P V follow one another: 5,300
// cycles a tile, where the products take 2,040 (36 of S at 34 cycles, 16 of P V at 51, measured alone) and the matrix units
// need 1,088 of those. 4 sequences of 65,536 rows, 64 query rows: 115 us a call, DRAM 13 % and tensor pipe 30 % busy;
// 32 query rows 88 us.
#include <algorithm>
#include "latent_decode.cuh"

namespace vq2 {

constexpr int LD_WORKERS = 512, LD_WARPS = LD_WORKERS / 32;
constexpr int LD_THREADS = LD_WORKERS + 128;     // 96 registers each at launch: 512 x 104 + 128 x 64 afterwards
constexpr int LD_UNIT = LD_TILE * 128;  // bytes of a unit of the tile: 64 rows of 64 fp16 values
constexpr int LD_UNITS = 9;             // 8 for the latent, 1 for the rotary part (P takes its place once S is done)
constexpr int LD_KBYTES = LD_UNITS * LD_UNIT;
constexpr float LD_BIAS = 5.f, LD_RAISE = 10.f;    // P = 2^(z - m + BIAS); m is raised when z exceeds it by RAISE

constexpr int LD_PARTS = 2;             // of a tile: four units each, the last with the rotary unit
constexpr int LD_RAW = LD_TILE * 400;   // a tile's raw rows (at most 400 bytes each)
// Tiles and raw tiles that fit beside Q (NQ x 1152 bytes) in 227 KB.
// (TWO: fp16 query rows in two terms, 32 of them.)
template <int NQ, bool TWO> constexpr int LD_TILES = NQ == 64 || TWO ? 1 : 2;
template <int NQ, bool TWO> constexpr int LD_RAWS = NQ == 64 || TWO ? 3 : 1;
template <int NQ, bool TWO> constexpr int LD_QBYTES = LD_UNITS * NQ * 128 * (TWO ? 2 : 1);

template <int NQ>
struct LdShared {
  uint64_t kfull[2][LD_PARTS], kfree[2][LD_PARTS], sfull[2], pfull[2], drain;      // by tile buffer
  uint64_t rfull[3], rfree[3];       // by raw tile
  uint64_t qfull, qfree;
  uint32_t there[3][2];              // rows of a raw tile that were found
  uint32_t tmem;
  int abort;
  LdStart start;
  int flag[2][LD_TILE];              // 2 i: the row is not there in tile i; 2 i + 1: it holds a non-finite scale
  float red[4][NQ];
  alignas(16) float2 meta[2][NQ];    // of this query block and the next
  float ref[NQ], down[NQ];           // maximum that P and O are relative to; factor of its last change
  float lsum[4][NQ];
  int scan[LD_WARPS];
};
template <int NQ, bool TWO>
constexpr size_t ld_smem() {
  return (size_t)LD_TILES<NQ, TWO> * LD_KBYTES + (size_t)LD_RAWS<NQ, TWO> * LD_RAW + LD_QBYTES<NQ, TWO> + sizeof(LdShared<NQ>) + 1024;
}
static_assert(ld_smem<64, false>() <= 227 * 1024 && ld_smem<32, false>() <= 227 * 1024 && ld_smem<32, true>() <= 227 * 1024, "latent decode shared memory");

__device__ __forceinline__ void ld_sync_workers() { asm volatile("barrier.cta.sync 1, 512;" ::: "memory"); }
__device__ __forceinline__ void ld_sync_group(int g) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(2 + g) : "memory"); }
__device__ __forceinline__ bool ld_any_group(int g, bool p) {
  uint32_t r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n barrier.cta.red.or.pred q, %1, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
               : "=r"(r) : "r"(2 + g), "r"((uint32_t)p) : "memory");
  return r != 0;
}
template <int N>
__device__ __forceinline__ void ld_tmem_load(uint32_t t, float* v) {
  if (N == 16) tmem_ld16(t, v);
  else tmem_ld8(t, v);
}
// 32 bytes of fp32 in one store (a whole sector).
__device__ __forceinline__ void store32(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}

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
template <int NQ, int U, int KS = 0>
__device__ __forceinline__ void ld_score_unit(uint32_t d, uint32_t k, uint32_t q, uint32_t acc) {
  constexpr uint32_t id = (1u << 4) | ((uint32_t)(NQ >> 3) << 17) | ((uint32_t)(LD_TILE >> 4) << 24);
  umma_at<U * (LD_UNIT >> 4) + 2 * KS, U * (NQ * 8) + 2 * KS, LP_DESC_HI, id>(d, k, q, U + KS > 0 ? 1 : acc);
  if constexpr (KS < 3) ld_score_unit<NQ, U, KS + 1>(d, k, q, acc);
}
// Unit u of S, u known at run time (the rotary unit, or a last single one).
template <int NQ>
__device__ __forceinline__ void ld_score_any(int u, uint32_t d, uint32_t k, uint32_t q) {
  ld_score_unit<NQ, 0>(d, k + u * (LD_UNIT >> 4), q + u * (NQ * 8), u > 0);
}
// O^T block M += V^T P^T: 128 latent values (the second unit of the last block may be P itself, where the latent has an odd
// number of units: its rows of O^T are not read). P lies as rows of 2 NQ bytes in the swizzle of that width.
template <int NQ, int M, int KS = 0>
__device__ __forceinline__ void ld_value_block(uint32_t d, uint32_t v, uint32_t p, uint32_t acc) {
  constexpr uint32_t id = (1u << 4) | (1u << 15) | (1u << 16) | ((uint32_t)(NQ >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t p_hi = (uint32_t)(16 * NQ >> 4) | 1u << 14 | (NQ == 64 ? 2u : 4u) << 29;
  umma_at<M * (2 * LD_UNIT >> 4) + KS * 128, KS * (2 * NQ), p_hi, id>(d + M * NQ, v, p, KS > 0 ? 1 : acc);
  if constexpr (KS + 1 < LD_TILE / 16) ld_value_block<NQ, M, KS + 1>(d, v, p, acc);
}

template <int NQ, bool TWO>
__global__ void __launch_bounds__(LD_THREADS, 1) latent_decode_kernel(LdArgs g) {
  constexpr int TILES = LD_TILES<NQ, TWO>, RAWS = LD_RAWS<NQ, TWO>;
  constexpr int CPT = NQ / 4, CPH = NQ / 8;     // columns of S^T (query rows) a column group has, a softmax thread takes
  constexpr uint32_t COLS = NQ == 64 ? 512 : 256;    // tensor memory: O^T 4 x NQ columns, S^T 2 x NQ
  extern __shared__ __align__(1024) uint8_t ld_smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)ld_smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t kb = smem_u32(smem), qb = kb + TILES * LD_KBYTES, raw = qb + LD_QBYTES<NQ, TWO>;
  LdShared<NQ>* sh = (LdShared<NQ>*)(smem + TILES * LD_KBYTES + LD_QBYTES<NQ, TWO> + RAWS * LD_RAW);
  const vq2_latent_decode_args& a = g.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int L = a.latent_dim, R = a.rope_dim, nl = L / 64, nblk = (nl + 1) / 2, parts = (nl + 3) / 4, units = nl + (R ? 1 : 0);
  volatile int* abort = &sh->abort;
  pdl_launch_dependents();

  if (tid == 0) {
    for (int k = 0; k < 2; ++k) {
      for (int m = 0; m < LD_PARTS; ++m) {
        mbar_init(&sh->kfull[k][m], LD_WARPS);
        mbar_init(&sh->kfree[k][m], 1);
      }
      mbar_init(&sh->sfull[k], 1);
      mbar_init(&sh->pfull[k], LD_WARPS);
    }
    for (int k = 0; k < RAWS; ++k) {
      mbar_init(&sh->rfull[k], 1);
      mbar_init(&sh->rfree[k], LD_WARPS);
    }
    mbar_init(&sh->qfull, 1);
    mbar_init(&sh->qfree, 1);
    mbar_init(&sh->drain, 1);
    sh->abort = 0;
    fence_mbar_init();
  }
  if (warp == LD_WARPS) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem)), "r"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid < 2 * LD_TILE) sh->flag[tid >> 6][tid & 63] = -1;

  const int count = ld_share<LD_WARPS>(g, sh->scan, &sh->start);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh->tmem, 0);
  const uint32_t ts = tmem + 4 * NQ;                    // S^T of the two buffers

  if (warp >= LD_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == LD_WARPS && count > 0 && elect_one()) {
      // ---------------- products
      LdPos p = sh->start.position(g);
      bool opens = true;             // the tile whose P V comes next is the first of its query block
      auto values = [&](int i) {     // O^T += V^T P^T of tile i, a block of 128 values after another
        const int b = i % TILES;
        ld_wait(&sh->pfull[b], (i / TILES) & 1, abort);
        tc_fence_after();
        const uint32_t t = (kb + b * LD_KBYTES) >> 4, v = t | (LD_UNIT >> 4) << 16, pd = (t + nl * (LD_UNIT >> 4)) | 1u << 16;
        const uint32_t acc = opens ? 0 : 1;
        ld_value_block<NQ, 0>(tmem, v, pd, acc);
        if (nblk > 1) ld_value_block<NQ, 1>(tmem, v, pd, acc);
        umma_commit(&sh->kfree[b][0]);
        if (nblk > 2) {
          ld_value_block<NQ, 2>(tmem, v, pd, acc);
          if (nblk > 3) ld_value_block<NQ, 3>(tmem, v, pd, acc);
          umma_commit(&sh->kfree[b][1]);
        }
      };
      auto scores = [&](int i) {     // S^T = K Q^T of tile i, part by part as it arrives
        const int b = i % TILES;
        const uint32_t k = ((kb + b * LD_KBYTES) >> 4) | 1u << 16, q = (qb >> 4) | 1u << 16, d = ts + b * NQ;
        ld_wait(&sh->kfull[b][0], (i / TILES) & 1, abort);
        tc_fence_after();
        ld_score_unit<NQ, 0>(d, k, q, 0);
        if (nl > 1) ld_score_unit<NQ, 1>(d, k, q, 1);
        if (nl > 2) ld_score_unit<NQ, 2>(d, k, q, 1);
        if (nl > 3) ld_score_unit<NQ, 3>(d, k, q, 1);
        const uint32_t q2 = q + units * (NQ * 8);         // the second term follows the first
        if constexpr (TWO) {
          ld_score_unit<NQ, 0>(d, k, q2, 1);
          if (nl > 1) ld_score_unit<NQ, 1>(d, k, q2, 1);
          if (nl > 2) ld_score_unit<NQ, 2>(d, k, q2, 1);
          if (nl > 3) ld_score_unit<NQ, 3>(d, k, q2, 1);
        }
        if (nl > 4) {
          ld_wait(&sh->kfull[b][1], (i / TILES) & 1, abort);
          tc_fence_after();
          ld_score_unit<NQ, 4>(d, k, q, 1);
          if (nl > 5) ld_score_unit<NQ, 5>(d, k, q, 1);
          if (nl > 6) ld_score_unit<NQ, 6>(d, k, q, 1);
          if (nl > 7) ld_score_unit<NQ, 7>(d, k, q, 1);
          if constexpr (TWO) {
            ld_score_unit<NQ, 4>(d, k, q2, 1);
            if (nl > 5) ld_score_unit<NQ, 5>(d, k, q2, 1);
            if (nl > 6) ld_score_unit<NQ, 6>(d, k, q2, 1);
            if (nl > 7) ld_score_unit<NQ, 7>(d, k, q2, 1);
          }
        }
        if (R) ld_score_any<NQ>(nl, d, k, q);
        umma_commit(&sh->sfull[b]);
      };
      int seg = -1;
      for (int i = 0; i < count; ++i) {
        const bool first = i == 0 || p.tile == 0, last = i + 1 == count || p.tile + 1 == p.tiles;
        // a new query block's tiles come only after the block before is finished
        if (TILES == 2 && i > 0 && first) {
          values(i - 1);
          opens = true;
        }
        if (TILES == 1) opens = first;
        if (first) ld_wait(&sh->qfull, ++seg & 1, abort);
        scores(i);
        if (last) umma_commit(&sh->qfree);
        if (TILES == 1) {
          values(i);
        } else if (i > 0 && !first) {
          values(i - 1);
          opens = false;
        }
        p.next(g);
      }
      if (TILES == 2) values(count - 1);
      umma_commit(&sh->drain);
      ld_wait(&sh->drain, 0, abort);
    } else if (warp == LD_WARPS + 1 && count > 0) {
      // ---------------- loader: the whole warp, two rows a lane. Page numbers are read a tile ahead.
      LdPos p = sh->start.position(g);
      LdRows rows;
      rows.find(g, p);
      int seg = -1;
      for (int i = 0; i < count; ++i) {
        const int st = i % RAWS;
        if (i == 0 || p.tile == 0) {
          // a query block's rows, once the products with the block before are done
          const int bytes = units * NQ * 128 * (TWO ? 2 : 1), item = p.b * g.nrb + p.rb;
          if (++seg == 0) pdl_wait();
          else ld_wait(&sh->qfree, (seg - 1) & 1, abort);
          if (lane == 0) {
            mbar_arrive_expect_tx(&sh->qfull, bytes + NQ * 8);
            bulk_g2s(smem + (qb - kb), g.q + (size_t)item * bytes, bytes, &sh->qfull);
            bulk_g2s(sh->meta[seg & 1], g.meta + (size_t)item * NQ, NQ * 8, &sh->qfull);
          }
        }
        const long long off[2] = {rows.offset(g, p, 0), rows.offset(g, p, 1)};
        const uint32_t in0 = __ballot_sync(0xffffffffu, off[0] >= 0), in1 = __ballot_sync(0xffffffffu, off[1] >= 0);
        const long long lead = __shfl_sync(0xffffffffu, off[0], 0);
        const bool run = __all_sync(0xffffffffu, off[0] == lead + (long long)lane * g.rb && off[1] == lead + (long long)(lane + 32) * g.rb);
        p.next(g);
        if (i + 1 < count) rows.find(g, p);
        ld_wait(&sh->rfree[st], ((i / RAWS) & 1) ^ 1, abort);
        if (lane < 2) sh->there[st][lane] = lane ? in1 : in0;
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&sh->rfull[st], (__popc(in0) + __popc(in1)) * g.rb);
        __syncwarp();
        uint8_t* dst = smem + (raw - kb) + st * LD_RAW;
        if (run) {                         // 64 rows side by side: one copy
          if (lane == 0) bulk_g2s(dst, (const uint8_t*)a.cache + lead, LD_TILE * g.rb, &sh->rfull[st]);
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (off[k] >= 0) bulk_g2s(dst + (lane + 32 * k) * g.rb, (const uint8_t*)a.cache + off[k], g.rb, &sh->rfull[st]);
        }
      }
      for (int i = max(0, count - RAWS); i < count; ++i) ld_wait(&sh->rfull[i % RAWS], (i / RAWS) & 1, abort);   // no copy left in flight
      ld_wait(&sh->qfull, seg & 1, abort);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    if (count > 0) {
      // ---------------- workers
      // softmax: S^T's row kr is in tensor-memory lane 32 quarter + (kr & 15); the upper 16 lanes of the warp take
      // half of the column group's columns from the lower ones
      const int quarter = warp & 3, grp = warp >> 2, kr = quarter * 16 + (lane & 15);
      const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
      const int col0 = grp * CPT + (lane >> 4) * CPH;
      // A warp takes 4 rows of a tile, 8 lanes a row: 128 bytes of nibbles (four units) a part, its scales and its rotary part.
      // The raw tile goes into registers as a whole, so that its place is free for the one after.
      uint4 lat[LD_PARTS], rope, sc;
      bool here = false;
      const int row = warp * 4 + (lane >> 3), piece = lane & 7;
      auto read_raw = [&](int i) {
        const int st = i % RAWS;
        ld_wait(&sh->rfull[st], (i / RAWS) & 1, abort);
        here = (sh->there[st][row >> 5] >> (row & 31)) & 1;
        const uint32_t r = raw + st * LD_RAW + row * g.rb;
#pragma unroll
        for (int m = 0; m < LD_PARTS; ++m) {
          lat[m] = make_uint4(0, 0, 0, 0);
          if (here && 8 * m + piece < 2 * nl) lat[m] = lds128_v(r + 128 * m + 16 * piece);
        }
        sc = rope = make_uint4(0, 0, 0, 0);
        if (here) sc = lds128_v(r + L / 2 + 2 * R);
        if (here && piece * 8 < R) rope = lds128_v(r + L / 2 + 16 * piece);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->rfree[st]);
      };
      // Registers -> tile, a part after another. A piece's four words become four 16-byte chunks of a 128-byte row; each of the
      // part's four units takes its words in another order, so that 8 neighbouring lanes fall on all bank groups.
      auto expand = [&](int number) {
        const int b = number % TILES, turn = piece >> 1;
        const uint32_t tile = kb + b * LD_KBYTES + row * 128;
#pragma unroll
        for (int m = 0; m < LD_PARTS; ++m) {
          if (m >= parts) break;
          if (number >= TILES) ld_wait(&sh->kfree[b][m], (number / TILES - 1) & 1, abort);
          // (after the wait: until P V of the buffer's tile before has begun, a slower column group may still read its flags)
          if (m == 0 && !here && piece == 0) sh->flag[b][row] = 2 * number;
          if (8 * m + piece < 2 * nl) {
            const uint32_t two = piece & 4 ? (m ? sc.w : sc.y) : (m ? sc.z : sc.x);
            uint32_t s = piece & 2 ? two >> 16 : two & 0xFFFFu;
            if ((s & 0x7C00u) == 0x7C00u) {       // a non-finite scale: the row reads as NaN, see the softmax
              s = 0;
              sh->flag[b][row] = 2 * number + 1;
            }
            const __half2 s2 = __half2half2(__ushort_as_half((unsigned short)s)), c2 = __hmul2(s2, __float2half2_rn(-24.f));
            uint32_t w0 = lat[m].x, w1 = lat[m].y, w2 = lat[m].z, w3 = lat[m].w, t;
            if (turn & 1) { t = w0; w0 = w1; w1 = t; t = w2; w2 = w3; w3 = t; }
            if (turn & 2) { t = w0; w0 = w2; w2 = t; t = w1; w1 = w3; w3 = t; }
            const uint32_t w[4] = {w0, w1, w2, w3};
#pragma unroll
            for (int q = 0; q < 4; ++q)
              sts128_v(tile + (4 * m + turn) * LD_UNIT + ((((piece & 1) * 4 + (q ^ turn)) ^ (row & 7)) << 4),
                       make_uint4(ln_pair<0>(w[q], s2, c2), ln_pair<1>(w[q], s2, c2), ln_pair<2>(w[q], s2, c2), ln_pair<3>(w[q], s2, c2)));
          }
          if (m == parts - 1 && R) sts128_v(tile + nl * LD_UNIT + ((piece ^ (row & 7)) << 4), rope);
          fence_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->kfull[b][m]);
        }
      };
      float l[CPH], ref[CPH], fac[CPH];      // of this thread's query rows: denominator (its cached rows), maximum, factor
      // The softmax of tile i at p: logits from tensor memory, P into the rotary unit's place.
      auto softmax = [&](int i, const LdPos& p, bool opens, int seg) {
        const int b = i % TILES;
        ld_wait(&sh->sfull[b], (i / TILES) & 1, abort);
        ld_wait(&sh->kfull[b][parts - 1], (i / TILES) & 1, abort);        // long done: orders the other warps' flags before their reads
        tc_fence_after();
        float z[CPH];
        {
          float full[CPT];
          ld_tmem_load<CPT>(ts + b * NQ + lanes + grp * CPT, full);
#pragma unroll
          for (int c = 0; c < CPH; ++c) {
            const float up = __shfl_sync(0xffffffffu, full[CPH + c], lane & 15);
            z[c] = (lane < 16 ? full[c] : up) * fac[c];
          }
        }
        const int flag = sh->flag[b][kr];
        if ((p.tile + 1) * LD_TILE > p.len - a.T + 1) {              // some query row sees part of the tile only
          const int j = p.tile * LD_TILE + kr;
#pragma unroll
          for (int c = 0; c < CPH; ++c)
            if (j > p.len - a.T + __float_as_int(sh->meta[seg & 1][col0 + c].y) || j >= p.len) z[c] = -INFINITY;
        }
        if (flag == 2 * i) {
#pragma unroll
          for (int c = 0; c < CPH; ++c) z[c] = -INFINITY;
        }
        if (flag == 2 * i + 1) {
          // the latent is key and value: every query row that sees this one is NaN as a whole; its values
          // were expanded to zeros, so that rows that do not see it are untouched
#pragma unroll
          for (int c = 0; c < CPH; ++c) {
            if (z[c] != -INFINITY) l[c] = __int_as_float(0x7FFFFFFF);
            z[c] = -INFINITY;
          }
        }
        bool raise = opens;
#pragma unroll
        for (int c = 0; c < CPH; ++c) raise |= z[c] - ref[c] > LD_RAISE;     // (differences first, here and below: exact where a sum is not)
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
          if (!opens) ld_wait(&sh->kfree[(i - 1) % TILES][parts - 1], ((i - 1) / TILES) & 1, abort);
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
        }
        uint32_t ph[CPH / 2];
#pragma unroll
        for (int c = 0; c < CPH; c += 2) {
          const float p0 = ex2((z[c] - (ref[c] == -INFINITY ? 0.f : ref[c])) + LD_BIAS);
          const float p1 = ex2((z[c + 1] - (ref[c + 1] == -INFINITY ? 0.f : ref[c + 1])) + LD_BIAS);
          l[c] += p0;
          l[c + 1] += p1;
          ph[c / 2] = pack2<VQ2_DT_F16>(p0, p1);
        }
        // rows of 2 NQ bytes, 16-byte chunks swizzled as the descriptor says
        const uint32_t prow = kb + b * LD_KBYTES + nl * LD_UNIT + kr * (2 * NQ), at = col0 * 2;
        if (NQ == 64)
          sts128_v(prow + (((at >> 4) ^ (kr & 7)) << 4), make_uint4(ph[0], ph[1], ph[2 % (CPH / 2)], ph[3 % (CPH / 2)]));
        else
          asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(prow + (((at >> 4) ^ ((kr >> 1) & 3)) << 4) + (at & 15)), "r"(ph[0]), "r"(ph[1])
                       : "memory");
        fence_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->pfull[b]);
      };
      // O^T with its maxima and denominators -> this block's part of the query block
      auto finish = [&](const LdPos& p) {
        const size_t slot = (size_t)(p.b * g.nrb + p.rb) + blockIdx.x;
#pragma unroll
        for (int c = 0; c < CPH; ++c) {
          float s = l[c];
#pragma unroll
          for (int o = 8; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          if ((lane & 15) == 0) {
            sh->lsum[quarter][col0 + c] = s;
            if (quarter == 0) sh->ref[col0 + c] = ref[c];
          }
        }
#pragma unroll 1
        for (int m = 0; m < nblk; ++m) {
          float o[CPT];
          ld_tmem_load<CPT>(tmem + lanes + m * NQ + grp * CPT, o);
          const int d = m * 128 + quarter * 32 + lane;
          if (d < L)
#pragma unroll
            for (int c = 0; c < CPT; c += 8) store32(g.part + (slot * L + d) * NQ + grp * CPT + c, o + c);
        }
        ld_sync_workers();
        if (tid < NQ)
          g.ml[slot * NQ + tid] = make_float2(sh->ref[tid], (sh->lsum[0][tid] + sh->lsum[1][tid]) + (sh->lsum[2][tid] + sh->lsum[3][tid]));
        ld_sync_workers();
      };

      // Tiles are expanded up to TILES ahead of the softmax, but not past the end of a query block (pe, ps: the next of each).
      LdPos pe = sh->start.position(g), ps = pe;
      int ie = 0, is = 0, seg = -1;
      read_raw(0);
      while (is < count) {
        const bool first = ie == 0 || pe.tile == 0;
        if (ie < count && ie - is < TILES && (!first || ie == is)) {
          if (first) {
            ld_wait(&sh->qfull, ++seg & 1, abort);
#pragma unroll
            for (int c = 0; c < CPH; ++c) {
              l[c] = 0.f;
              ref[c] = -INFINITY;
              fac[c] = sh->meta[seg & 1][col0 + c].x;
            }
          }
          expand(ie);
          if (++ie < count) read_raw(ie);
          pe.next(g);
          if (ie < count && ie - is < TILES && pe.tile != 0) continue;
        }
        softmax(is, ps, is == 0 || ps.tile == 0, seg);
        if (is + 1 == count || ps.tile + 1 == ps.tiles) {
          ld_wait(&sh->kfree[is % TILES][parts - 1], (is / TILES) & 1, abort);
          tc_fence_after();
          finish(ps);
          tc_fence_before();
        }
        ++is;
        ps.next(g);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (tid == 0 && *abort) set_status(VQ2_ERR_TIMEOUT);
  pdl_wait();        // also where there was nothing to do: the query kernel is done when this one is
  if (warp == LD_WARPS) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS));
}

// Query rows a block, by the rows of a sequence. Up to 16 the narrow kernel; up to 32, or more, the wide one with that many
// (64 sequences, 320,206 cached rows: 16 query rows 81 us narrow, 116 with 32 wide, 144 with 64; 32 rows 120 us with 32 wide, 138 as two
// narrow blocks, 148 with 64 wide; 48 rows 154 us with 64 wide, 195 narrow, 200 with 32). Where the narrow kernel's blocks have at most 5
// tiles each, time is mostly latency, and it has less of it (in graphs, 64 rows of 8 sequences: 2048 cached rows each 32 us, 37 wide;
// 4096 each 44 and 43 us; 64 rows of one sequence, 64 cached: 11 and 17 us). fp16 queries in two terms take the room of 64 rows with
// 32 (4 sequences of 65,536 rows, 64 heads: 168 us, bf16 115; 64 sequences, 16 heads, narrow: 97 and 81). The rule goes by the table's
// width, as the lengths are on the device: a table far wider than they are takes the wide kernel where the narrow one would be faster.
static int ld_nq(int B, int T, int heads, long long most, bool two) {
  const long long rows = (long long)T * heads;
  return rows <= 16 || (double)B * ((most + LD_TILE - 1) / LD_TILE) * ((rows + 15) / 16) <= 5 * 2 * 148 ? 16 : two || rows <= 32 ? 32 : 64;
}

struct LdLayout {
  size_t start, ml, meta, q, part, total;
};
static LdLayout ld_layout(int B, int nq, int nrb, int L, int R, int grid) {
  const size_t items = (size_t)B * nrb, parts = items + grid;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  LdLayout w;
  w.start = take((size_t)(B + 1) * 4);
  w.ml = take(parts * nq * 8);
  w.meta = take(items * nq * 8);
  w.q = take(items * (L / 64 + (R ? 1 : 0)) * nq * 256);       // (a second term of fp16 rows included)
  w.part = take(parts * nq * L * 4);
  w.total = at + 256;
  return w;
}
// Blocks that share the tiles: two an SM for the narrow kernel. The workspace is sized without a device; a B200 has 148 SMs.
static int ld_blocks(int nq, int sms) { return std::min(sms, 148) * (nq == 16 ? 2 : 1); }

// Three launches: query rows, the main kernel (NQ rows a block; NARROW: the one for 16), the join; the later two by programmatic
// dependent launch.
template <int DT, int NQ, bool NARROW>
static int ld_launch(const LdArgs& g, cudaStream_t st) {
  constexpr bool TWO = DT == VQ2_DT_F16;
  void (*kernel)(LdArgs);
  size_t smem;
  if constexpr (NARROW) {
    static void (*const by_groups[8])(LdArgs) = {
        latent_decode_narrow_kernel<1, TWO>, latent_decode_narrow_kernel<2, TWO>, latent_decode_narrow_kernel<3, TWO>,
        latent_decode_narrow_kernel<4, TWO>, latent_decode_narrow_kernel<5, TWO>, latent_decode_narrow_kernel<6, TWO>,
        latent_decode_narrow_kernel<7, TWO>, latent_decode_narrow_kernel<8, TWO>};
    kernel = by_groups[g.a.latent_dim / 64 - 1];
    smem = LN_SMEM;
  } else {
    kernel = latent_decode_kernel<NQ, TWO>;
    smem = ld_smem<NQ, TWO>();
  }
  static bool raised[8][64];
  if (!smem_limit_once(kernel, smem, raised[NARROW ? g.a.latent_dim / 64 - 1 : 0])) return VQ2_ERR_CUDA;
  const int items = g.a.B * g.nrb;
  latent_query_kernel<DT, NQ, NARROW><<<items * NQ / LQ_WARPS, LQ_WARPS * 32, 0, st>>>(g);
  if (cudaGetLastError() != cudaSuccess) return VQ2_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(g.grid);
  cfg.blockDim = dim3(NARROW ? LN_THREADS : LD_THREADS);
  cfg.dynamicSmemBytes = smem;
  if (cudaLaunchKernelEx(&cfg, kernel, g) != cudaSuccess) return VQ2_ERR_CUDA;
  cfg.gridDim = dim3((unsigned)(items * (g.a.latent_dim / 64) * (NQ / 8)));
  cfg.dynamicSmemBytes = 0;
  const bool many = g.grid > 8 * items;          // parts a query block: at most about grid / items
  cfg.blockDim = dim3(many ? 512 : 128);
  return cudaLaunchKernelEx(&cfg, many ? latent_join_kernel<DT, NQ, 16> : latent_join_kernel<DT, NQ, 4>, g) == cudaSuccess ? VQ2_OK : VQ2_ERR_CUDA;
}

}  // namespace vq2

using namespace vq2;

extern "C" size_t vq2_latent_decode_workspace_size(int B, int T, int heads, int latent_dim, int rope_dim) {
  if (B <= 0 || T <= 0 || heads <= 0 || !latent_dims_ok(latent_dim, rope_dim) || (long long)T * heads > 1 << 20 ||
      (long long)B * ((long long)T * heads + 64) >= 1LL << 27)
    return 0;
  // the most that a kernel which may be taken needs
  size_t most = 0;
  for (const int nq : {16, ld_nq(B, T, heads, 1LL << 40, false), ld_nq(B, T, heads, 1LL << 40, true)})
    most = std::max(most, ld_layout(B, nq, (int)(((long long)T * heads + nq - 1) / nq), latent_dim, rope_dim, ld_blocks(nq, 148)).total);
  return most;
}

static bool ld_sizes_ok(int B, int T, int heads, int max_pages, int page_size) {
  if (B <= 0 || T <= 0 || heads <= 0 || page_size <= 0 || max_pages <= 0 || (long long)T * heads > 1 << 20 ||
      (long long)B * ((long long)T * heads + 64) >= 1LL << 27)
    return false;
  // positions (tiles of all query blocks in order) are 32-bit numbers
  return (double)B * (((double)max_pages * page_size + LD_TILE - 1) / LD_TILE) * ((double)T * heads / 16 + 1) < 2147483648.;
}

extern "C" int vq2_latent_decode_query_rows(int B, int T, int heads, int max_pages, int page_size, int dtype) {
  if (!ld_sizes_ok(B, T, heads, max_pages, page_size) || (dtype != VQ2_DT_BF16 && dtype != VQ2_DT_F16)) return 0;
  return ld_nq(B, T, heads, (long long)max_pages * page_size, dtype == VQ2_DT_F16);
}

extern "C" int vq2_latent_decode(const vq2_latent_decode_args* a, void* ws, size_t ws_bytes, void* stream) {
  if (!a || !a->q || !a->cache || !a->block_table || !a->kv_len || !a->out) return VQ2_ERR_NULL;
  if (a->pages <= 0 || !latent_dims_ok(a->latent_dim, a->rope_dim) || !(a->scale > 0.f) ||
      !ld_sizes_ok(a->B, a->T, a->heads, a->max_pages, a->page_size))
    return VQ2_ERR_SHAPE;
  if (a->dtype != VQ2_DT_BF16 && a->dtype != VQ2_DT_F16) return VQ2_ERR_DTYPE;
  if (((uintptr_t)a->q | (uintptr_t)a->cache | (uintptr_t)a->out) & 15) return VQ2_ERR_ALIGN;
  if (!ws || ws_bytes < vq2_latent_decode_workspace_size(a->B, a->T, a->heads, a->latent_dim, a->rope_dim))
    return VQ2_ERR_WORKSPACE;
  LdArgs g = {};
  g.a = *a;
  const int nq = ld_nq(a->B, a->T, a->heads, (long long)a->max_pages * a->page_size, a->dtype == VQ2_DT_F16), sms = device_sm_count();
  if (sms <= 0) return VQ2_ERR_CUDA;
  g.rb = latent_row_bytes(a->latent_dim, a->rope_dim);
  g.nrb = (a->T * a->heads + nq - 1) / nq;
  g.grid = ld_blocks(nq, sms);
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
  const LdLayout w = ld_layout(a->B, nq, g.nrb, a->latent_dim, a->rope_dim, g.grid);
  uint8_t* base = (uint8_t*)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
  g.start = (int*)(base + w.start);
  g.ml = (float2*)(base + w.ml);
  g.part = (float*)(base + w.part);
  g.q = base + w.q;
  g.meta = (float2*)(base + w.meta);
  cudaStream_t st = (cudaStream_t)stream;
  const bool bf = a->dtype == VQ2_DT_BF16;
  if (nq == 16) return bf ? ld_launch<VQ2_DT_BF16, 16, true>(g, st) : ld_launch<VQ2_DT_F16, 16, true>(g, st);
  if (nq == 32) return bf ? ld_launch<VQ2_DT_BF16, 32, false>(g, st) : ld_launch<VQ2_DT_F16, 32, false>(g, st);
  return ld_launch<VQ2_DT_BF16, 64, false>(g, st);
}
