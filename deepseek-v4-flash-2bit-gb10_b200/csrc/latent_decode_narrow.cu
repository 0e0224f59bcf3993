// K8, few query rows: absorbed latent attention over the 4-bit cache for blocks of 16 query rows (heads x tokens of one sequence).
//
// With 16 query rows a cached row costs 17,400 multiply-adds and 400 bytes: the warps' own matrix instructions
// (m16n8k16, 1024 a clock) do them in the time that the row takes from memory (17 cycles), and take their operands from
// registers, so a row is expanded from its nibbles straight into the operand and never written back to shared
// memory. Through tcgen05 the expanded tile would be written once and read twice there, and that path, not memory, was the
// bound (16 query rows: 5,100 cycles a tile of 64 rows; here ~1,500).
//
// A loader warp keeps raw rows coming through a ring. Of each tile, warp w of eight
//   S    takes cached rows 8 w .. 8 w + 7 against all 16 query rows, whose operand it keeps in registers (144 of them). The
//        contraction index is permuted so that a thread's two operand registers are neighbours in one word of nibbles.
//   P    writes its probabilities (2 KB for the block), the one block barrier a tile
//   O    takes values 64 w .. 64 w + 63 of all 64 rows: word n of a row's eight for column n, its nibble j for product j
// The softmax is as in the wide kernel: a maximum is raised only when a logit exceeds it by 2^10.
#include "latent_decode.cuh"

namespace vq2 {

constexpr int LN_ROWS = 16, LN_WARPS = 8, LN_THREADS = 384;    // 168 registers each at launch: 256 x 232 + 128 x 40 afterwards
constexpr int LN_STAGES = 6, LN_STAGE = LD_TILE * 400;
constexpr float LN_BIAS = 5.f, LN_RAISE = 10.f;                // P = 2^(z - m + BIAS)
constexpr int LN_PPITCH = 144;                                 // bytes of a row of P: 64 fp16 values, rows on different banks

struct LnShared {
  uint64_t rfull[LN_STAGES], rfree[LN_STAGES];
  uint32_t there[LN_STAGES][2];        // rows of a tile that were found
  alignas(16) uint8_t p[2][LN_ROWS * LN_PPITCH];
  float red[LN_WARPS][LN_ROWS];
  int abort;
  LdStart start;
  int scan[LN_WARPS];
};
constexpr size_t LN_SMEM = (size_t)LN_STAGES * LN_STAGE + sizeof(LnShared) + 128;

// Bytes between raw rows in shared memory: an odd number of 16-byte units, so that eight rows' words, and two apart
// the words of four row pairs, fall on different banks.
__host__ __device__ __forceinline__ int ln_pitch(int rb) { return (rb / 16 | 1) * 16; }

__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Nibbles J of both halves of w, as n s in fp16: nibble u = n + 8 in the top mantissa bits of 16 + u; (16 + u) s - 24 s, exact.
template <int J>
__device__ __forceinline__ uint32_t ln_pair(uint32_t w, __half2 s2, __half2 c2) {
  const uint32_t h = ((J < 2 ? w << (6 - 4 * J) : w >> (4 * J - 6)) & 0x03C003C0u) | 0x4C004C00u;
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

// NL: groups of 64 latent values, known at compile time so that a tile's work is three straight runs of instructions.
template <int NL>
__global__ void __launch_bounds__(LN_THREADS, 1) latent_decode_narrow_kernel(LdArgs g) {
  extern __shared__ __align__(128) uint8_t ln_smem[];
  LnShared* sh = (LnShared*)(ln_smem + LN_STAGES * LN_STAGE);
  const vq2_latent_decode_args& a = g.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  constexpr int L = NL * 64;
  const int R = a.rope_dim, pitch = ln_pitch(g.rb), units = NL + (R ? 1 : 0);
  volatile int* abort = &sh->abort;
  pdl_launch_dependents();
  if (tid == 0) {
    for (int s = 0; s < LN_STAGES; ++s) {
      mbar_init(&sh->rfull[s], 1);
      mbar_init(&sh->rfree[s], LN_WARPS);
    }
    sh->abort = 0;
    fence_mbar_init();
  }
  const int count = ld_share<LN_WARPS>(g, sh->scan, &sh->start);
  __syncthreads();

  if (warp >= LN_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == LN_WARPS && count > 0) {
      // ---------------- loader
      LdPos p = sh->start.position(g);
      LdRows rows;
      rows.find(g, p);
      for (int i = 0; i < count; ++i) {
        const int st = i % LN_STAGES;
        uint8_t* dst = ln_smem + st * LN_STAGE;
        const long long off[2] = {rows.offset(g, p, 0), rows.offset(g, p, 1)};
        const uint32_t in0 = __ballot_sync(0xffffffffu, off[0] >= 0), in1 = __ballot_sync(0xffffffffu, off[1] >= 0);
        const long long first = __shfl_sync(0xffffffffu, off[0], 0);
        const bool run = __all_sync(0xffffffffu, off[0] == first + (long long)lane * g.rb && off[1] == first + (long long)(lane + 32) * g.rb);
        p.next(g);
        if (i + 1 < count) rows.find(g, p);
        ld_wait(&sh->rfree[st], ((i / LN_STAGES) & 1) ^ 1, abort);
#pragma unroll
        for (int k = 0; k < 2; ++k)      // a row that is not there: zero scales, so that it adds nothing to O
          if (off[k] < 0) *(uint4*)(dst + (lane + 32 * k) * pitch + L / 2 + 2 * R) = make_uint4(0, 0, 0, 0);
        if (lane < 2) sh->there[st][lane] = lane ? in1 : in0;
        fence_async_smem();              // the zeros come before a later tile's copy to the same place
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&sh->rfull[st], (__popc(in0) + __popc(in1)) * g.rb);
        __syncwarp();
        if (run && pitch == g.rb) {      // 64 rows side by side: one copy
          if (lane == 0) bulk_g2s(dst, (const uint8_t*)a.cache + first, LD_TILE * g.rb, &sh->rfull[st]);
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (off[k] >= 0) bulk_g2s(dst + (lane + 32 * k) * pitch, (const uint8_t*)a.cache + off[k], g.rb, &sh->rfull[st]);
        }
      }
      for (int i = max(0, count - LN_STAGES); i < count; ++i) ld_wait(&sh->rfull[i % LN_STAGES], (i / LN_STAGES) & 1, abort);   // none left in flight
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    if (count > 0) {
      const int gr = lane >> 2, t = lane & 3;       // fragment row (query rows gr, gr + 8; S's cached row; O's column) and quarter
      LdPos p = sh->start.position(g);
      uint4 q[2 * NL + 2][2];                       // query rows gr and gr + 8: pieces of 32 latent values, then 2 of rotary ones
      float o[8][4], l[2], ref[2], fac[2];
      int tok[2];
      bool fresh = true;                            // the query kernel's results not yet waited for
      for (int i = 0; i < count; ++i) {
        const int st = i % LN_STAGES, item = p.b * g.nrb + p.rb;
        if (i == 0 || p.tile == 0) {                // a new query block
          if (fresh) pdl_wait();
          fresh = false;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int row = item * LN_ROWS + gr + 8 * k;
            const uint4* src = (const uint4*)(g.q + (size_t)row * units * 128) + t;
#pragma unroll
            for (int n = 0; n < 2 * NL + 2; ++n) q[n][k] = n < 2 * NL || (n - 2 * NL) * 32 < R ? src[n * 4] : make_uint4(0, 0, 0, 0);
            const float2 m = g.meta[row];
            fac[k] = m.x;
            tok[k] = __float_as_int(m.y);
            l[k] = 0.f;
            ref[k] = -INFINITY;
          }
#pragma unroll
          for (int v = 0; v < 8; ++v) o[v][0] = o[v][1] = o[v][2] = o[v][3] = 0.f;
        }
        ld_wait(&sh->rfull[st], (i / LN_STAGES) & 1, abort);
        uint8_t* tile = ln_smem + st * LN_STAGE;
        // ---------------- S: cached row 8 warp + gr against the 16 query rows
        float z[4];
        {
          uint8_t* row = tile + (warp * 8 + gr) * pitch;
          uint4* scales = (uint4*)(row + L / 2 + 2 * R);
          const uint4 sc = *scales;
          const uint32_t scale[4] = {sc.x, sc.y, sc.z, sc.w};
          float acc[4][4] = {};
#pragma unroll
          for (int n = 0; n < 2 * NL; ++n) {
            const uint32_t s = __byte_perm(scale[n >> 2], 0, (n >> 1) & 1 ? 0x3232 : 0x1010);
            const __half2 s2 = *(const __half2*)&s, c2 = __hmul2(s2, __float2half2_rn(-24.f));
            const uint32_t w = *(const uint32_t*)(row + (4 * n + t) * 4);
            mma16816(acc[2 * (n & 1)], q[n][0].x, q[n][1].x, q[n][0].y, q[n][1].y, ln_pair<0>(w, s2, c2), ln_pair<1>(w, s2, c2));
            mma16816(acc[2 * (n & 1) + 1], q[n][0].z, q[n][1].z, q[n][0].w, q[n][1].w, ln_pair<2>(w, s2, c2), ln_pair<3>(w, s2, c2));
          }
          if (R) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int d = k * 32 + 8 * t, n = 2 * NL + k;
              uint4 w = make_uint4(0, 0, 0, 0);
              if (d < R) w = *(const uint4*)(row + L / 2 + 2 * d);
              mma16816(acc[2 * k], q[n][0].x, q[n][1].x, q[n][0].y, q[n][1].y, w.x, w.y);
              mma16816(acc[2 * k + 1], q[n][0].z, q[n][1].z, q[n][0].w, q[n][1].w, w.z, w.w);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) z[k] = ((acc[0][k] + acc[1][k]) + (acc[2][k] + acc[3][k])) * fac[k >> 1];
          // A non-finite scale has made the logits NaN for those who see the row; its values must not reach the others.
          // (An exponent of all ones carries into the top bit when one is added to it.)
          uint32_t bad = 0;
#pragma unroll
          for (int k = 0; k < (NL + 1) / 2; ++k) bad |= ((scale[k] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
          if (__any_sync(0xffffffffu, bad)) {      // (the vote: a row's four lanes have all read its scales)
            uint16_t* h = (uint16_t*)scales;
            for (int k = 0; k < 8; ++k)
              if ((h[k] & 0x7C00u) == 0x7C00u) h[k] = 0;
            fence_async_smem();          // before a later tile's copy to the same place
          }
        }
        // ---------------- softmax: query row gr (z[0], z[1]) and gr + 8 (z[2], z[3]), cached rows 8 warp + 2 t and + 1
        const uint32_t there = sh->there[st][warp >> 2] >> ((warp & 3) * 8 + 2 * t);
        bool raise = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = p.tile * LD_TILE + warp * 8 + 2 * t + (k & 1);
          if (!((there >> (k & 1)) & 1) || j > p.len - a.T + tok[k >> 1]) z[k] = -INFINITY;
          raise |= z[k] > ref[k >> 1] + LN_RAISE;
        }
        uint8_t* pb = sh->p[i & 1];
        float pr[4];
        auto probabilities = [&]() {
#pragma unroll
          for (int k = 0; k < 4; ++k) pr[k] = ex2(z[k] - ((ref[k >> 1] == -INFINITY ? 0.f : ref[k >> 1]) - LN_BIAS));
#pragma unroll
          for (int k = 0; k < 2; ++k)
            *(uint32_t*)(pb + (gr + 8 * k) * LN_PPITCH + (warp * 8 + 2 * t) * 2) = pack2<VQ2_DT_F16>(pr[2 * k], pr[2 * k + 1]);
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
        l[0] += pr[0] + pr[1];
        l[1] += pr[2] + pr[3];
        // ---------------- O: values 64 warp .. 64 warp + 63 of all the tile's rows
        if (warp < NL) {
          const uint8_t* col = tile + 2 * t * pitch + (warp * 8 + gr) * 4;
          const uint8_t* srow = tile + 2 * t * pitch + L / 2 + 2 * R + 2 * warp;
#pragma unroll
          for (int ks = 0; ks < LD_TILE / 16; ++ks) {
            const uint8_t* pa = pb + gr * LN_PPITCH + (16 * ks + 2 * t) * 2;
            const uint32_t a0 = *(const uint32_t*)pa, a1 = *(const uint32_t*)(pa + 8 * LN_PPITCH), a2 = *(const uint32_t*)(pa + 16),
                           a3 = *(const uint32_t*)(pa + 8 * LN_PPITCH + 16);
            uint32_t w[4], s[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = (16 * ks + (k & 1) + 8 * (k >> 1)) * pitch;
              w[k] = *(const uint32_t*)(col + r);
              s[k] = *(const uint16_t*)(srow + r);
            }
            const uint32_t sa = s[0] | s[1] << 16, sb = s[2] | s[3] << 16;
            const __half2 sa2 = *(const __half2*)&sa, sb2 = *(const __half2*)&sb;
            const __half2 ca2 = __hmul2(sa2, __float2half2_rn(-24.f)), cb2 = __hmul2(sb2, __float2half2_rn(-24.f));
            // halves of two rows' words side by side: values 2 j in the low ones, 2 j + 1 in the high ones
            const uint32_t al = __byte_perm(w[0], w[1], 0x5410), ah = __byte_perm(w[0], w[1], 0x7632);
            const uint32_t bl = __byte_perm(w[2], w[3], 0x5410), bh = __byte_perm(w[2], w[3], 0x7632);
            mma16816(o[0], a0, a1, a2, a3, ln_pair<0>(al, sa2, ca2), ln_pair<0>(bl, sb2, cb2));
            mma16816(o[1], a0, a1, a2, a3, ln_pair<0>(ah, sa2, ca2), ln_pair<0>(bh, sb2, cb2));
            mma16816(o[2], a0, a1, a2, a3, ln_pair<1>(al, sa2, ca2), ln_pair<1>(bl, sb2, cb2));
            mma16816(o[3], a0, a1, a2, a3, ln_pair<1>(ah, sa2, ca2), ln_pair<1>(bh, sb2, cb2));
            mma16816(o[4], a0, a1, a2, a3, ln_pair<2>(al, sa2, ca2), ln_pair<2>(bl, sb2, cb2));
            mma16816(o[5], a0, a1, a2, a3, ln_pair<2>(ah, sa2, ca2), ln_pair<2>(bh, sb2, cb2));
            mma16816(o[6], a0, a1, a2, a3, ln_pair<3>(al, sa2, ca2), ln_pair<3>(bl, sb2, cb2));
            mma16816(o[7], a0, a1, a2, a3, ln_pair<3>(ah, sa2, ca2), ln_pair<3>(bh, sb2, cb2));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->rfree[st]);
        if (i + 1 == count || p.tile + 1 == p.tiles) {
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
        }
        p.next(g);
      }
    }
  }
  __syncthreads();
  if (tid == 0 && *abort) set_status(VQ2_ERR_TIMEOUT);
  pdl_wait();        // also where there was nothing to do: the query kernel is done when this one is
}

}  // namespace vq2
