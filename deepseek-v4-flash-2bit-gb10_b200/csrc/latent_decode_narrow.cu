// K8, few query rows: absorbed latent attention over the 4-bit cache for blocks of 16 query rows (heads x tokens of one sequence).
//
// With 16 query rows a cached row costs 17,400 multiply-adds and 400 bytes: the warps' own matrix instructions
// (m16n8k16, 1024 a clock) do them in the time that the row takes from memory (17 cycles), and take their operands from
// registers, so a row is expanded from its nibbles straight into the operand and never written back to shared
// memory. Through tcgen05 the expanded tile is written once and read twice there, by way of several hand-overs.
//
// A block of 8 warps, two on an SM so that one computes while the other waits, keeps three tiles of 64 raw rows coming. Of each tile
//   S    warp w takes cached rows 16 (w & 3) .. + 15 and one half of the values; the halves of two warps are added through
//        shared memory, each keeping 8 rows. The contraction index is permuted so that a thread's two operand registers are
//        neighbours in one word of nibbles.
//   P    each warp writes its rows' probabilities (2 KB for the block), then the one block barrier of a tile
//   O    warp w takes values 64 w .. 64 w + 63 of all 64 rows: word n of a row's eight for column n, its nibble j for product j
// 3 instructions expand 2 values, once for S and once for O. No unit is full (issue slots 46 % busy, tensor pipe 33 %, shared memory
// 37 %): a warp waits for its own last instruction, for the matrix unit and at the barrier of a tile. The maximum is raised only when
// a logit exceeds it by 2^10, as in the wide kernel. 64 sequences, 320,206 cached rows, 16 heads: 81 us a call, of which 10 are latency (a call over
// 64 rows); 197,000 rows more cost 34 us, about 3,000 cycles a tile and SM where the matrix instructions need 1,088.
#include "latent_decode.cuh"

namespace vq2 {

constexpr int LN_ROWS = 16, LN_WARPS = 8, LN_THREADS = LN_WARPS * 32;
constexpr int LN_STAGES = 3, LN_STAGE = LD_TILE * 400;
constexpr float LN_BIAS = 5.f, LN_RAISE = 10.f;                // P = 2^(z - m + BIAS)

struct LnShared {
  uint4 q[18][2][32];                  // query rows as operands: piece of 32 values, product, lane
  uint2 rest[16][2][32];               // of fp16 rows: what q rounded away, in 8 bits a value
  uint4 p[2][LD_TILE / 16][32];        // probabilities as operands: 16 cached rows, lane
  float4 half[LN_WARPS][32];           // sums over half of the values, on their way to the other warp of the pair
  uint64_t rfull[LN_STAGES];
  uint32_t there[LN_STAGES][2];        // rows of a tile that were found
  float red[LN_WARPS][LN_ROWS];
  int abort;
  LdStart start;
  int scan[LN_WARPS];
};
constexpr size_t LN_SMEM = (size_t)LN_STAGES * LN_STAGE + sizeof(LnShared) + 128;
static_assert(2 * (LN_SMEM + 1024) <= 228 * 1024, "two blocks on an SM");

// The left operand's four registers are neighbours as they come from shared memory (moved there they cost as much as the
// product).
__device__ __forceinline__ void mma16816(float* c, const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// Nibbles J of both halves of w, as n s in fp16: nibble u = n + 8 in the top mantissa bits of 16 + u; (16 + u) s - 24 s, exact.
template <int J>
__device__ __forceinline__ uint32_t ln_pair(uint32_t w, __half2 s2, __half2 c2) {
  uint32_t h;                            // (and, or) in one instruction: given two constants the compiler makes it two
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(h) : "r"(J < 2 ? w << (6 - 4 * J) : w >> (4 * J - 6)), "r"(0x03C003C0u), "r"(0x4C004C00u));
  const __half2 x = __hfma2(*(const __half2*)&h, s2, c2);
  return *(const uint32_t*)&x;
}
__device__ __forceinline__ bool ln_any(bool p) {
  uint32_t r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 256, p;\n selp.u32 %0, 1, 0, q;\n}"
               : "=r"(r) : "r"((uint32_t)p) : "memory");
  return r != 0;
}
__device__ __forceinline__ void ln_sync() { asm volatile("barrier.cta.sync 1, 256;" ::: "memory"); }

__device__ __forceinline__ void ln_sync_pair(int k) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(2 + k) : "memory"); }

// Eight 8-bit values (the upper bytes of halves) as an operand.
__device__ __forceinline__ uint4 ln_rest(const uint2& x) {
  return make_uint4(__byte_perm(x.x, 0, 0x1404), __byte_perm(x.x, 0, 0x3424), __byte_perm(x.y, 0, 0x1404), __byte_perm(x.y, 0, 0x3424));
}

// Pieces FROM .. TO - 1 (32 values each) of the latent part of S for 16 cached rows: acc[u] for rows 8 u .. 8 u + 7 of them.
// TWO: with the query rows' second term.
template <int FROM, int TO, bool TWO>
__device__ __forceinline__ void ln_scores(float (*acc)[2][4], const uint4 (*q)[2][32], const uint2 (*rest)[2][32], const uint8_t* row0,
                                          const uint8_t* row1, const uint32_t* sc0, const uint32_t* sc1, int lane) {
#pragma unroll
  for (int n = FROM; n < TO; ++n) {
    const uint4 qa = q[n][0][lane], qb = q[n][1][lane];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t s = __byte_perm((u ? sc1 : sc0)[n >> 2], 0, (n >> 1) & 1 ? 0x3232 : 0x1010);
      const __half2 s2 = *(const __half2*)&s, c2 = __hmul2(s2, __float2half2_rn(-24.f));
      const uint32_t w = *(const uint32_t*)((u ? row1 : row0) + (4 * n + (lane & 3)) * 4);
      const uint32_t k0 = ln_pair<0>(w, s2, c2), k1 = ln_pair<1>(w, s2, c2), k2 = ln_pair<2>(w, s2, c2), k3 = ln_pair<3>(w, s2, c2);
      mma16816(acc[u][0], qa, k0, k1);
      mma16816(acc[u][1], qb, k2, k3);
      if (TWO) {
        mma16816(acc[u][0], ln_rest(rest[n][0][lane]), k0, k1);
        mma16816(acc[u][1], ln_rest(rest[n][1][lane]), k2, k3);
      }
    }
  }
}

// NL: groups of 64 latent values, known at compile time so that a tile's work is three straight runs of instructions.
template <int NL, bool TWO>
__global__ void __launch_bounds__(LN_THREADS, 2) latent_decode_narrow_kernel(LdArgs g) {
  extern __shared__ __align__(128) uint8_t ln_smem[];
  LnShared* sh = (LnShared*)(ln_smem + LN_STAGES * LN_STAGE);
  const vq2_latent_decode_args& a = g.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  constexpr int L = NL * 64, PITCH = ((NL * 32 + 128 + 16) / 16 | 1) * 16;      // raw rows: an odd number of 16-byte units apart
  const int R = a.rope_dim, units = NL + (R ? 1 : 0), tail = L / 2 + 2 * R;     // scales from byte `tail` of a row
  volatile int* abort = &sh->abort;
  pdl_launch_dependents();
  if (tid == 0) {
    for (int s = 0; s < LN_STAGES; ++s) mbar_init(&sh->rfull[s], 1);
    sh->abort = 0;
    fence_mbar_init();
  }
  const int count = ld_share<LN_WARPS>(g, sh->scan, &sh->start);
  __syncthreads();
  if (count > 0) {
    const int gr = lane >> 2, t = lane & 3;       // fragment row (query rows gr, gr + 8; a cached row of S; a column of O) and quarter
    const int quad = warp & 3, half = warp >> 2, mine = 16 * quad + 8 * half;     // this warp's cached rows after the exchange
    LdPos p = sh->start.position(g), pl = p;      // the tile at work; the next tile to be loaded
    LdRows rows;
    // A warp loads tile n (at `pl`, pages found before): a copy a row, or one where the 64 rows lie side by side.
    auto load = [&](int n) {
      const int st = n % LN_STAGES;
      uint8_t* dst = ln_smem + st * LN_STAGE;
      const long long off[2] = {rows.offset(g, pl, 0), rows.offset(g, pl, 1)};
      const uint32_t in0 = __ballot_sync(0xffffffffu, off[0] >= 0), in1 = __ballot_sync(0xffffffffu, off[1] >= 0);
      const long long lead = __shfl_sync(0xffffffffu, off[0], 0);
      const bool run = __all_sync(0xffffffffu, off[0] == lead + (long long)lane * g.rb && off[1] == lead + (long long)(lane + 32) * g.rb);
#pragma unroll
      for (int k = 0; k < 2; ++k)      // a row that is not there: zero scales, so that it adds nothing to O
        if (off[k] < 0) *(uint4*)(dst + (lane + 32 * k) * PITCH + tail) = make_uint4(0, 0, 0, 0);
      if (lane < 2) sh->there[st][lane] = lane ? in1 : in0;
      fence_async_smem();              // the zeros come before a later tile's copy to the same place
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(&sh->rfull[st], (__popc(in0) + __popc(in1)) * g.rb);
      __syncwarp();
      if (run && PITCH == g.rb) {
        if (lane == 0) bulk_g2s(dst, (const uint8_t*)a.cache + lead, LD_TILE * g.rb, &sh->rfull[st]);
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (off[k] >= 0) bulk_g2s(dst + (lane + 32 * k) * PITCH, (const uint8_t*)a.cache + off[k], g.rb, &sh->rfull[st]);
      }
    };
    // the first tiles: a warp each; then warp 0 finds the pages of the tile that it will load in step 0
    for (int n = 0; n < LN_STAGES - 1 && n < count; ++n) {
      if (warp == n) {
        rows.find(g, pl);
        load(n);
      }
      pl.next(g);
    }
    if (warp == 0 && LN_STAGES - 1 < count) rows.find(g, pl);
    float o[8][4], l[2], ref[2], fac[2];
    int tok[2];
    // ---------------- O: values 64 warp .. 64 warp + 63 of all rows of tile i
    auto values = [&](int i) {
      const uint8_t* tile = ln_smem + i % LN_STAGES * LN_STAGE;
      const uint4 (*pb)[32] = sh->p[i & 1];
      if (NL == LN_WARPS || warp < NL) {
        const uint8_t* col = tile + 2 * t * PITCH + (warp * 8 + gr) * 4;
        const uint8_t* srow = tile + 2 * t * PITCH + tail + 2 * warp;
#pragma unroll
        for (int ks = 0; ks < LD_TILE / 16; ++ks) {
          const uint4 pa = pb[ks][lane];
          uint32_t w[4], s[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = (16 * ks + (k & 1) + 8 * (k >> 1)) * PITCH;
            w[k] = *(const uint32_t*)(col + r);
            s[k] = *(const uint16_t*)(srow + r);
          }
          const uint32_t sa = s[0] | s[1] << 16, sb = s[2] | s[3] << 16;
          const __half2 sa2 = *(const __half2*)&sa, sb2 = *(const __half2*)&sb;
          const __half2 ca2 = __hmul2(sa2, __float2half2_rn(-24.f)), cb2 = __hmul2(sb2, __float2half2_rn(-24.f));
          // halves of two rows' words side by side: values 2 j in the low ones, 2 j + 1 in the high ones
          const uint32_t al = __byte_perm(w[0], w[1], 0x5410), ah = __byte_perm(w[0], w[1], 0x7632);
          const uint32_t bl = __byte_perm(w[2], w[3], 0x5410), bh = __byte_perm(w[2], w[3], 0x7632);
          mma16816(o[0], pa, ln_pair<0>(al, sa2, ca2), ln_pair<0>(bl, sb2, cb2));
          mma16816(o[1], pa, ln_pair<0>(ah, sa2, ca2), ln_pair<0>(bh, sb2, cb2));
          mma16816(o[2], pa, ln_pair<1>(al, sa2, ca2), ln_pair<1>(bl, sb2, cb2));
          mma16816(o[3], pa, ln_pair<1>(ah, sa2, ca2), ln_pair<1>(bh, sb2, cb2));
          mma16816(o[4], pa, ln_pair<2>(al, sa2, ca2), ln_pair<2>(bl, sb2, cb2));
          mma16816(o[5], pa, ln_pair<2>(ah, sa2, ca2), ln_pair<2>(bh, sb2, cb2));
          mma16816(o[6], pa, ln_pair<3>(al, sa2, ca2), ln_pair<3>(bl, sb2, cb2));
          mma16816(o[7], pa, ln_pair<3>(ah, sa2, ca2), ln_pair<3>(bh, sb2, cb2));
        }
      }
    };
    auto finish = [&](int item) {
      // ---------------- this block's part of the query block
      const size_t slot = (size_t)item + blockIdx.x;
      if (warp < NL) {
        float* dst = g.part + (slot * L + (warp * 8 + 2 * t) * 8) * LN_ROWS + gr;
#pragma unroll
        for (int v = 0; v < 8; ++v)
#pragma unroll
          for (int k = 0; k < 4; ++k) dst[((k & 1) * 8 + v) * LN_ROWS + 8 * (k >> 1)] = o[v][k];
      }
      ln_sync();                     // the maxima's place is free
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float s = l[k] + __shfl_xor_sync(0xffffffffu, l[k], 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        if (t == 0) sh->red[warp][gr + 8 * k] = s;
      }
      ln_sync();
      if (warp == 0 && t == 0)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float s = 0.f;
#pragma unroll
          for (int w = 0; w < LN_WARPS; ++w) s += sh->red[w][gr + 8 * k];
          g.ml[slot * LN_ROWS + gr + 8 * k] = make_float2(ref[k], s);
        }
      ln_sync();
    };
    // The products of O run a tile behind, beside those of S of the next: two independent chains in one run of instructions.
    int item = 0;
    for (int i = 0;; ++i) {
      const int st = i % LN_STAGES;
      const bool fresh = i == 0 || i == count || p.tile == 0;
      if (i > 0 && fresh) {
        values(i - 1);
        finish(item);
      }
      if (i == count) break;
      if (fresh) {                                // a new query block: its rows to shared memory (the one before is done with)
        item = p.b * g.nrb + p.rb;
        if (i == 0) pdl_wait();
        const uint4* src = (const uint4*)(g.q + (size_t)item * LN_ROWS * units * 128 * (TWO ? 2 : 1));
        for (int u = tid; u < LN_ROWS * units * 8; u += LN_THREADS) ((uint4*)sh->q)[u] = __ldcg(src + u);
        if (TWO)
          for (int u = tid; u < NL * 64; u += LN_THREADS) ((uint4*)sh->rest)[u] = __ldcg(src + LN_ROWS * units * 8 + u);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 m = __ldcg(g.meta + item * LN_ROWS + gr + 8 * k);
          fac[k] = m.x;
          tok[k] = __float_as_int(m.y);
          l[k] = 0.f;
          ref[k] = -INFINITY;
        }
#pragma unroll
        for (int v = 0; v < 8; ++v) o[v][0] = o[v][1] = o[v][2] = o[v][3] = 0.f;
        ln_sync();
      }
      ld_wait(&sh->rfull[st], (i / LN_STAGES) & 1, abort);
      uint8_t* tile = ln_smem + st * LN_STAGE;
      // ---------------- S: 16 cached rows, half of the values
      float z[4];
      {
        uint8_t* row0 = tile + (16 * quad + gr) * PITCH;
        uint8_t* row1 = row0 + 8 * PITCH;
        const uint4 x0 = *(const uint4*)(row0 + tail), x1 = *(const uint4*)(row1 + tail);
        const uint32_t sc0[4] = {x0.x, x0.y, x0.z, x0.w}, sc1[4] = {x1.x, x1.y, x1.z, x1.w};
        float acc[2][2][4] = {};
        auto low = [&]() { ln_scores<0, NL + 1, TWO>(acc, sh->q, sh->rest, row0, row1, sc0, sc1, lane); };
        auto high = [&]() {
          ln_scores<NL + 1, 2 * NL, TWO>(acc, sh->q, sh->rest, row0, row1, sc0, sc1, lane);
          if (R) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint4 qa = sh->q[2 * NL + k][0][lane], qb = sh->q[2 * NL + k][1][lane];
              const int d = k * 32 + 8 * t;
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (d < R) w = *(const uint4*)((u ? row1 : row0) + L / 2 + 2 * d);
                mma16816(acc[u][0], qa, w.x, w.y);
                mma16816(acc[u][1], qb, w.z, w.w);
              }
            }
          }
        };
        if (fresh) {
          if (half == 0) low();
          else high();
        } else if (half == 0) {
          low();
          values(i - 1);
        } else {
          high();
          values(i - 1);
        }
        const int away = half ^ 1;                // the rows that the other warp of the pair keeps
        float give[4], keep[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float v0 = acc[0][0][k] + acc[0][1][k], v1 = acc[1][0][k] + acc[1][1][k];
          give[k] = away ? v1 : v0;
          keep[k] = away ? v0 : v1;
        }
        sh->half[warp][lane] = make_float4(give[0], give[1], give[2], give[3]);
        ln_sync_pair(quad);
        const float4 got = sh->half[warp ^ 4][lane];
        z[0] = (keep[0] + got.x) * fac[0];
        z[1] = (keep[1] + got.y) * fac[0];
        z[2] = (keep[2] + got.z) * fac[1];
        z[3] = (keep[3] + got.w) * fac[1];
        // A non-finite scale has made the logits NaN for those who see the row; its values must not reach the others.
        // (An exponent of all ones carries into the top bit when one is added to it. Both warps of the pair have read it.)
        uint32_t bad = 0;
#pragma unroll
        for (int k = 0; k < (NL + 1) / 2; ++k)
          bad |= (((sc0[k] & 0x7C007C00u) + 0x04000400u) | ((sc1[k] & 0x7C007C00u) + 0x04000400u)) & 0x80008000u;
        if (bad) {
          for (int k = 0; k < 16; ++k) {
            uint16_t* h = (uint16_t*)((k < 8 ? row0 : row1) + tail) + (k & 7);
            if ((*h & 0x7C00u) == 0x7C00u) *h = 0;
          }
          fence_async_smem();          // before a later tile's copy to the same place
        }
      }
      // ---------------- softmax: query row gr (z[0], z[1]) and gr + 8 (z[2], z[3]), cached rows mine + 2 t and + 1
      const uint32_t there = sh->there[st][mine >> 5] >> ((mine & 31) + 2 * t);
      bool raise = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = p.tile * LD_TILE + mine + 2 * t + (k & 1);
        if (!((there >> (k & 1)) & 1) || j > p.len - a.T + tok[k >> 1]) z[k] = -INFINITY;
        raise |= z[k] - ref[k >> 1] > LN_RAISE;      // (differences first, here and below: exact where a sum with a large logit is not)
      }
      uint4 (*pb)[32] = sh->p[i & 1];
      float pr[4];
      auto probabilities = [&]() {
#pragma unroll
        for (int k = 0; k < 4; ++k) pr[k] = ex2((z[k] - (ref[k >> 1] == -INFINITY ? 0.f : ref[k >> 1])) + LN_BIAS);
        // registers 0, 1 (rows gr, gr + 8) of the operand of 16 cached rows for the first 8 of them, 2, 3 for the others
        *((uint2*)&pb[quad][lane] + half) = make_uint2(pack2<VQ2_DT_F16>(pr[0], pr[1]), pack2<VQ2_DT_F16>(pr[2], pr[3]));
      };
      probabilities();
      if (ln_any(raise)) {
        // the block's maxima, then everything relative to them
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float m = fmaxf(z[2 * k], z[2 * k + 1]);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          if (t == 0) sh->red[warp][gr + 8 * k] = m;
        }
        ln_sync();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float m = ref[k];
#pragma unroll
          for (int w = 0; w < LN_WARPS; ++w) m = fmaxf(m, sh->red[w][gr + 8 * k]);
          const float f = ref[k] == m ? 1.f : ref[k] == -INFINITY ? 0.f : ex2(ref[k] - m);
          ref[k] = m;
          l[k] = l[k] == 0.f ? 0.f : l[k] * f;
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            o[v][2 * k] *= f;
            o[v][2 * k + 1] *= f;
          }
        }
        probabilities();
        ln_sync();
      }
      // Every warp is past its work on the tile before: the next tile to come takes its place. The warps take turns, and
      // the one whose turn is next reads its tile's page numbers now.
      if (i + LN_STAGES - 1 < count) {
        if (warp == (i & 7)) load(i + LN_STAGES - 1);
        pl.next(g);
        if (warp == ((i + 1) & 7) && i + LN_STAGES < count) rows.find(g, pl);
      }
      l[0] += pr[0] + pr[1];
      l[1] += pr[2] + pr[3];
      p.next(g);
    }
  }
  __syncthreads();
  if (tid == 0 && *abort) set_status(VQ2_ERR_TIMEOUT);
  pdl_wait();        // also where there was nothing to do: the query kernel is done when this one is
}

}  // namespace vq2
