// K9 latent attention, expanded form: causal attention of a ragged batch of prompt chunks. Sequence
// b has query rows cu_q[b] .. cu_q[b+1] - 1 and key rows cu_k[b] .. cu_k[b+1] - 1; its last query sees
// all its keys (a cached prefix comes before them). Keys of head h are [k_nope[:, h], k_rope] with the
// rotary part shared by all heads:
//   z_ij = scale * (q_i . k_j),  j <= i + keys - queries;   out_i = sum_j softmax(z_i)_j v_j
//
// One CTA takes 256 queries of a head as two tiles of 128 and walks the keys 128 at a time, with a
// running maximum and sum per row. Tensor memory holds, per tile, the scores S (128 columns; the
// probabilities P overwrite them as packed 16-bit values) and the output O (128 columns): 512 in all.
//   warp 0       TMA: 16 KB units of 128 rows x 64 values (128-byte swizzle), the keys of a step before the values of the
//                step before it, through two rings; values past a dimension's end arrive as zeros
//   warp 1       tcgen05.mma: S = Q K^T (both from shared memory), O += P V (P from tensor memory, V as it
//                lies, rows = keys, so no transpose); the two tiles alternate, so one tile's products
//                run under the other tile's softmax
//   warps 4-11   softmax, one thread a query row (4 warps a tile): the row's 128 scores in registers
// A row's maximum is refreshed only when it rose by more than 2^8 in the exponent, so that O is rarely rescaled: P is at most 2^8
// times what it is at the maximum. In bf16, with the range of fp32, that is 1 and every P rounds by 2^-9 of itself. In fp16 it is 2^7,
// so that P ends at 2^15, a key of 2^-21 of the largest still rounds by 2^-12 of itself and one of 2^-32 is the last to count (held
// at 1, keys 2^-14 below a dominant one lost bits and those 2^-25 below it were gone, all of the output where that key's value is 0).
// P goes over in halves of 64 keys, so that O's products start under the second half's exponentials.
// Where there are fewer blocks of queries than SMs, a block's keys are split into parts, one CTA each, and a second kernel joins
// them (below: lp_split).
// What bounds it: the products of a step (two tiles, 128 keys) take 2560 cycles, the step about 3400: 1700 for a
// tile's softmax (1024 of them its exponentials) and the hand-overs before and after it, under which only the other tile's
// products run. 8192 tokens, 32 heads, 128 + 64 and 128 values: 0.61 ms, 1125 TFLOP/s, at the power limit (fp16 draws more there:
// 0.62 where bf16 takes 0.59); the library's plain bf16 product of 8192^3 sustains 1395.
// A key that a row does not see has probability 0; a NaN or an infinity in its value reaches the row all the same (0 times
// NaN) if both are in one step of 128 keys of one sequence, but never another sequence's rows.
#include <algorithm>
#include <type_traits>
#include "vq2_common.cuh"

namespace vq2 {

constexpr int LP_MAX_D = 128;      // values a head: of the positionless key part, and of v
constexpr int LP_TILE = 128;       // query rows a tile, key rows a step
constexpr int LP_UNIT = LP_TILE * 128;         // bytes of a unit: 128 rows of 64 16-bit values
// Steps in flight: 96 KB for keys (2 steps of 192 values, so a step's keys load under the step before),
// 32 KB for values (1 step of 128, loaded between its last product and the next step's first).
constexpr int LP_KUNITS = 6, LP_VUNITS = 2, LP_KMAX = 3;
constexpr int LP_THREADS = 384;
constexpr float LP_RAISE = 8.f;    // log2 by which a row's maximum may grow before O is rescaled
constexpr float LP_BIAS_F16 = 7.f; // log2 of P at its row's maximum, in fp16
constexpr float LP_FAR = 65536.f;  // log2 units from 0 beyond which scores are taken relative to the maximum before they are scaled

struct LpShared {
  uint64_t kfull[LP_KMAX], kempty[LP_KMAX], vfull[2], vempty[2];
  uint64_t qfull[2], sfull[2], pfull[2][2], ofull[2], vtail, cleared, drain;
  uint32_t tmem;
  int abort;
};
constexpr size_t LP_SMEM = (size_t)(6 + LP_KUNITS + LP_VUNITS) * LP_UNIT + sizeof(LpShared) + 1024;
static_assert(LP_SMEM <= 227 * 1024, "latent prefill shared memory");

// Shared-memory descriptors as two words: the low one holds the address (in 16-byte units, so a step
// along the contraction is one 32-bit add) and the leading offset, the high one is a constant: 8-row
// groups 1024 bytes apart, 128-byte swizzle. K-major operands (rows of S's operands) have no leading
// offset; in V, whose rows run along the contraction, it is the distance between units of 64 columns.
constexpr uint32_t LP_DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %5, 0;\n mov.b64 x, {%1, %3};\n mov.b64 y, {%2, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p;\n}"
               ::"r"(d), "r"(a), "r"(b), "r"(LP_DESC_HI), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n .reg .pred p;\n .reg .b64 y;\n setp.ne.b32 p, %5, 0;\n mov.b64 y, {%2, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n}"
               ::"r"(d), "r"(a), "r"(b), "r"(LP_DESC_HI), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
// One lane of a converged warp. The compiler knows that a branch on it has a single thread, so addresses
// and descriptors stay in uniform registers there (a branch on a lane number moves them there one by one).
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 64 columns of this thread's lane; a tcgen05.wait::ld has to follow before the values are used.
__device__ __forceinline__ void tmem_ld64(uint32_t t, float* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
               "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,"
               "%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
                 "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
                 "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
                 "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
                 "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
                 "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
                 "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
                 "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
               : "r"(t));
}
__device__ __forceinline__ void tmem_st32(uint32_t t, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
               "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
               ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                 "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
                 "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
                 "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
               : "memory");
}

// A row's 128 scores as registers.
__device__ __forceinline__ void tmem_ld128(uint32_t t, float* v) {
  tmem_ld64(t, v);
  tmem_ld64(t + 64, v + 64);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 128; ++i) asm volatile("" : "+f"(v[i]));     // no use of a value moves before the wait
}

// A position in a ring of N stages: the stage and the parity of the phase it is in.
template <int N>
struct Ring {
  int stage = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next() {
    if (++stage == N) {
      stage = 0;
      parity ^= 1;
    }
  }
};

// A block of queries: blocks are numbered (query block, sequence, head), the last query block of every head and sequence first,
// as it has most keys. Offsets are clamped to the tensors, so wrong ones give wrong rows and no access out of range.
struct LpBlock {
  int h, b, q0, nq, k0, nk, row0, past, ntile, n0, n1, nsteps;
  __device__ __forceinline__ bool at(const vq2_latent_prefill_args& a, int nqb, int block) {
    const int per = a.heads * a.B;
    h = block % per % a.heads;
    b = block % per / a.heads;
    q0 = min(max(a.cu_q[b], 0), a.total_q);
    nq = min(max(a.cu_q[b + 1], q0), a.total_q) - q0;
    k0 = min(max(a.cu_k[b], 0), a.total_k);
    nk = min(max(a.cu_k[b + 1], k0), a.total_k) - k0;
    row0 = (nqb - 1 - block / per) * 2 * LP_TILE;
    if (row0 >= nq) return false;
    past = nk - nq;                               // key i + past is the newest that query i sees
    ntile = nq - row0 > LP_TILE ? 2 : 1;
    // key steps of each tile, by its last row
    n0 = (max(0, min(nk, min(nq, row0 + LP_TILE) + past)) + LP_TILE - 1) / LP_TILE;
    n1 = ntile > 1 ? (max(0, min(nk, min(nq, row0 + 2 * LP_TILE) + past)) + LP_TILE - 1) / LP_TILE : 0;
    nsteps = max(n0, n1);
    return true;
  }
};

// The key steps of a block in parts of `steps` steps (more where that would be over `most` parts), one CTA each. Of a block with
// several parts each leaves its unnormalised rows and their maxima (in log2 units) and sums; slot = block * most + part, 256 rows.
struct LpParts {
  int most, steps;
  float* o;
  float2* ml;
  __device__ __forceinline__ int length(int nsteps) const { return max(steps, (nsteps + most - 1) / most); }
};

// KU, VU: units of 64 values in a key row (positionless part, then rotary part) and in a value row.
template <int DT, int KU, int VU>
__global__ void __launch_bounds__(LP_THREADS, 1)
latent_prefill_kernel(vq2_latent_prefill_args a, int nqb, LpParts parts, const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tr, const __grid_constant__ CUtensorMap tv) {
  extern __shared__ __align__(1024) uint8_t lp_smem_raw[];
  LpBlock w;
  if (!w.at(a, nqb, blockIdx.x)) return;
  const int per_part = parts.length(w.nsteps), first = blockIdx.y * per_part;      // this CTA's first key step
  if (first && first >= w.nsteps) return;
  const bool whole = w.nsteps <= per_part;
  // from here on keys and steps count from the part's first
  const int h = w.h, q0 = w.q0, nq = w.nq, row0 = w.row0, ntile = w.ntile;
  const int k0 = w.k0 + first * LP_TILE, nk = w.nk - first * LP_TILE, past = w.past - first * LP_TILE;
  const int n0 = min(max(w.n0 - first, 0), per_part), n1 = min(max(w.n1 - first, 0), per_part);
  const int nsteps = max(n0, n1);
  const bool tail = nsteps * LP_TILE > nk;        // the last step's values end inside their units
  auto n_of = [&](int t) { return t ? n1 : n0; };
  const int kn = (a.nope_dim + 63) / 64;          // units of the positionless part
  constexpr int KS = KU == 1 ? LP_KMAX : LP_KUNITS / KU, VS = LP_VUNITS / VU;      // stages

  uint8_t* smem = (uint8_t*)(((uintptr_t)lp_smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t qbase = smem_u32(smem), kring = qbase + 6 * LP_UNIT, vring = kring + LP_KUNITS * LP_UNIT;
  LpShared* sh = (LpShared*)(smem + (6 + LP_KUNITS + LP_VUNITS) * LP_UNIT);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 32) {
    // the first copy through a tensor map would wait for the map itself
    asm volatile("prefetch.tensormap [%0];\n prefetch.tensormap [%1];\n prefetch.tensormap [%2];\n prefetch.tensormap [%3];"
                 ::"l"(&tq), "l"(&tk), "l"(&tr), "l"(&tv) : "memory");
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < LP_KMAX; ++s) { mbar_init(&sh->kfull[s], 1); mbar_init(&sh->kempty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&sh->vfull[s], 1); mbar_init(&sh->vempty[s], 1); }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh->qfull[t], 1);
      mbar_init(&sh->sfull[t], 1);
      mbar_init(&sh->pfull[t][0], 4);
      mbar_init(&sh->pfull[t][1], 4);
      mbar_init(&sh->ofull[t], 1);
    }
    mbar_init(&sh->vtail, 1);
    mbar_init(&sh->cleared, 1);
    mbar_init(&sh->drain, 1);
    sh->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh->tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh->tmem, 0);
  volatile int* abort = &sh->abort;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 && nsteps > 0 && elect_one()) {
      // ---------------- loader
      auto queries = [&](int t) {
        mbar_arrive_expect_tx(&sh->qfull[t], KU * LP_UNIT);
#pragma unroll
        for (int s = 0; s < KU; ++s)
          tma_load_3d(qbase + (t * 3 + s) * LP_UNIT, &tq, s < kn ? s * 64 : a.nope_dim, h, q0 + row0 + t * LP_TILE, &sh->qfull[t]);
      };
      queries(0);
      // keys of step j go out before the values of step j - 1: the scores of a step are computed first
      Ring<KS> rk;
      Ring<VS> rv;
      bool ok = true;
      int nkeys = 0, nvals = 0;                      // steps loaded
      for (int j = 0; j <= nsteps; ++j) {
        if (j < nsteps) {
          if (!(ok = mbar_wait(&sh->kempty[rk.stage], rk.parity ^ 1))) break;       // passes at once in the first round
          mbar_arrive_expect_tx(&sh->kfull[rk.stage], KU * LP_UNIT);
#pragma unroll
          for (int s = 0; s < KU; ++s)
            tma_load_3d(kring + (rk.stage * KU + s) * LP_UNIT, s < kn ? &tk : &tr, s < kn ? s * 64 : 0, s < kn ? h : 0, k0 + j * LP_TILE,
                        &sh->kfull[rk.stage]);
          rk.next();
          ++nkeys;
          if (j == 0 && ntile > 1) queries(1);       // after the first keys: tile 0 starts on them
        }
        if (j > 0) {
          if (!(ok = mbar_wait(&sh->vempty[rv.stage], rv.parity ^ 1))) break;
          uint64_t* bar = tail && j == nsteps ? &sh->vtail : &sh->vfull[rv.stage];
          mbar_arrive_expect_tx(bar, VU * LP_UNIT);
#pragma unroll
          for (int s = 0; s < VU; ++s)
            tma_load_3d(vring + (rv.stage * VU + s) * LP_UNIT, &tv, s * 64, h, k0 + (j - 1) * LP_TILE, bar);
          rv.next();
          ++nvals;
        }
      }
      if (!ok) *abort = 1;
      // no copy is in flight when the block ends, also where a wait gave up
      for (int t = 0; t < ntile; ++t) mbar_wait(&sh->qfull[t], 0);
      for (int q = max(0, nkeys - KS); q < nkeys; ++q) mbar_wait(&sh->kfull[q % KS], (q / KS) & 1);
      for (int q = max(0, nvals - VS); q < nvals; ++q)
        tail && q == nsteps - 1 ? mbar_wait(&sh->vtail, 0) : mbar_wait(&sh->vfull[q % VS], (q / VS) & 1);
    } else if (warp == 1 && nsteps > 0 && elect_one()) {
      // ---------------- products: one thread issues them all
      constexpr uint32_t fmt = DT == VQ2_DT_BF16 ? (1u << 7) | (1u << 10) : 0u;
      constexpr uint32_t id_s = (1u << 4) | fmt | ((LP_TILE >> 3) << 17) | ((LP_TILE >> 4) << 24);
      // whole units of values: columns past v_dim are zeros in V (a descriptor known at compile time is what lets a product be
      // issued in 15 cycles)
      constexpr uint32_t id_o = (1u << 4) | fmt | (1u << 16) | ((uint32_t)(VU * 64 >> 3) << 17) | ((LP_TILE >> 4) << 24);
      constexpr uint32_t U = LP_UNIT >> 4;
      const uint32_t qlo = (qbase >> 4) | 1u << 16, klo = (kring >> 4) | 1u << 16, vlo = (vring >> 4) | U << 16;
      const int lastt = ntile - 1;                  // it has the most steps
      Ring<KS> rk;
      Ring<VS> rv;
      bool ok = true;
      auto scores = [&](int t) {                    // S_t = Q_t K^T: columns past a part's end are zeros in K
        const uint32_t qa = qlo + t * 3 * U, kb = klo + rk.stage * (KU * U);
#pragma unroll
        for (int s = 0; s < KU; ++s)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) umma_ss(tmem + t * 128, qa + s * U + 2 * ks, kb + s * U + 2 * ks, id_s, (s | ks) != 0);
        umma_commit(&sh->sfull[t]);
        if (t == lastt) {                           // the stage is free once the products issued so far are done
          umma_commit(&sh->kempty[rk.stage]);
          rk.next();
        }
      };
      ok = mbar_wait(&sh->kfull[0], 0);
      for (int t = 0; t < ntile && ok; ++t) {
        ok = mbar_wait(&sh->qfull[t], 0);
        tc_fence_after();
        if (ok && (n_of(t) > 0 || t == lastt)) scores(t);
      }
      for (int j = 0; j < nsteps && ok; ++j) {
        const uint32_t vb = vlo + rv.stage * (VU * U);
        ok = tail && j == nsteps - 1 ? mbar_wait(&sh->cleared, 0) : mbar_wait(&sh->vfull[rv.stage], rv.parity);
        bool loaded = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (t > lastt || j >= n_of(t) || !ok) continue;
          // O_t += P_t V, the first 64 keys as soon as their probabilities are there
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (!(ok = mbar_wait(&sh->pfull[t][half], j & 1))) break;
            tc_fence_after();
#pragma unroll
            for (int ks = half * 4; ks < half * 4 + 4; ++ks)
              umma_ts(tmem + 256 + t * 128, tmem + t * 128 + ks * 8, vb + ks * 128, id_o, ks > 0 ? 1 : j != 0);
          }
          if (!ok) break;
          if (t == lastt) umma_commit(&sh->vempty[rv.stage]);
          if (j + 1 < n_of(t)) {
            if (!loaded) ok = loaded = mbar_wait(&sh->kfull[rk.stage], rk.parity);
            if (!ok) break;
            tc_fence_after();
            scores(t);
          } else {
            umma_commit(&sh->ofull[t]);
          }
        }
        rv.next();
      }
      if (!ok) *abort = 1;
      umma_commit(&sh->drain);
      mbar_wait(&sh->drain, 0);
    } else if (warp == 2 && nsteps > 0 && tail) {
      // ---------------- the last step's value rows past the last key belong to another sequence: their
      // probabilities are 0, but 0 times a NaN there would reach this one's output, so they are cleared
      const int sv = (nsteps - 1) % VS * VU, live = nk - (nsteps - 1) * LP_TILE;
      if (!__all_sync(0xffffffffu, mbar_wait(&sh->vtail, 0))) *abort = 1;
      else
        for (int s = 0; s < VU; ++s)
          for (int i = live * 8 + lane; i < LP_TILE * 8; i += 32)
            sts128_v(vring + (sv + s) * LP_UNIT + i * 16, make_uint4(0, 0, 0, 0));
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->cleared);
    }
  } else {
    // ---------------- softmax: thread = query row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int t = (warp - 4) >> 2, r = (warp & 3) * 32 + lane, i = row0 + t * LP_TILE + r;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + t * 128, to = tmem + lanes + 256 + t * 128;
    const float sl = a.scale * 1.4426950408889634f;
    const int seen = max(0, min(nk, i + 1 + past));           // keys 0 .. seen - 1
    const int n = n_of(t);
    float m = -INFINITY;                                      // the maximum that P and O are relative to
    float2 l2 = make_float2(0.f, 0.f);
    bool ok = true, far = false;
    for (int j = 0; j < n; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(&sh->sfull[t], j & 1))) { ok = false; break; }
      tc_fence_after();
      float s[128];
      tmem_ld128(ts, s);
      const int lim = seen - j * LP_TILE;
      if (__any_sync(0xffffffffu, lim < LP_TILE)) {
#pragma unroll
        for (int c = 0; c < 128; ++c) s[c] = c < lim ? s[c] : -INFINITY;
      }
      float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c < 128; c += 8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) m4[k] = c + 4 + k < 128 ? fmaxf(m4[k], fmaxf(s[c + k], s[c + 4 + k])) : fmaxf(m4[k], s[c + k]);
      }
      const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
      // the first step sets the maximum; later ones raise it when it grew by more than LP_RAISE
      const bool raise = m == -INFINITY ? mx > m : (mx - m) * sl > LP_RAISE;
      if (__any_sync(0xffffffffu, raise) ) {
        const float mn = raise ? mx : m, f = raise ? ex2((m - mn) * sl) : 1.f;
        m = mn;
        far = __any_sync(0xffffffffu, m != -INFINITY && fabsf(m) * sl > LP_FAR);
        l2.x *= f;
        l2.y *= f;
        if (j > 0) {              // every product into O issued before this step's scores is done
#pragma unroll 1
          for (int c = 0; c < a.v_dim; c += 16) {
            float o[16];
            tmem_ld16(to + c, o);
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] *= f;
            tmem_st16(to + c, (const uint32_t*)o);
            tmem_st_wait();
            keep_live16((const uint32_t*)o);
          }
        }
      }
      constexpr float bias = DT == VQ2_DT_F16 ? LP_BIAS_F16 : 0.f;      // denominators carry the factor too, and so do all parts of a row
      float2 sum = make_float2(0.f, 0.f), sumb = sum;
      if (__builtin_expect(far, 0)) {
        // scale (s - m) as one fused multiply-add rounds -m scale first: by 2^-9 at LP_FAR, by whole powers of 2 beyond 2^24, where P would
        // leave its type's range. Here the difference, exact near m, comes first. (From tensor memory again, 16 scores at a
        // time, so that the other path keeps its registers; P's columns lie below the scores still to be read.)
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 1
        for (int c = 0; c < 128; c += 16) {
          float x[16];
          uint32_t p[8];
          tmem_ld16(ts + c, x);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            x[k] = c + k < lim ? ex2(fmaf(x[k] - base, sl, bias)) : 0.f;
            sum.x += x[k];
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) p[k] = pack2<DT>(x[2 * k], x[2 * k + 1]);
          tmem_st8(ts + (c >> 1), p);
          tmem_st_wait();
          keep_live8(p);
          if ((c & 63) == 48) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->pfull[t][c >> 6]);
          }
        }
      } else {
        const float mb = (m == -INFINITY ? 0.f : -m * sl) + bias;
        const float2 s2 = make_float2(sl, sl), b2 = make_float2(mb, mb);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t p[32];
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            float2 x = ffma2(make_float2(s[half * 64 + c], s[half * 64 + c + 1]), s2, b2);
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            if (c & 2) sumb = fadd2(sumb, x);
            else sum = fadd2(sum, x);
            p[c >> 1] = pack2<DT>(x.x, x.y);
          }
          tmem_st32(ts + half * 32, p);
          tmem_st_wait();
          keep_live16(p);
          keep_live16(p + 16);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->pfull[t][half]);
        }
      }
      l2 = fadd2(l2, fadd2(sum, sumb));
    }
    if (ok && n > 0 && !__all_sync(0xffffffffu, mbar_wait(&sh->ofull[t], 0))) ok = false;
    if (!ok) *abort = 1;
    tc_fence_after();
    if (t < ntile) {
      const float l = l2.x + l2.y;
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
      const long long at = ((long long)(q0 + i) * a.heads + h) * a.v_dim;
      const bool sectors = a.v_dim % 16 == 0 && ((uintptr_t)a.out & 31) == 0;      // a thread's run as whole 32-byte sectors
      const size_t slot = ((size_t)blockIdx.x * parts.most + blockIdx.y) * (2 * LP_TILE) + t * LP_TILE + r;
      if (!whole && i < nq) parts.ml[slot] = make_float2(m * sl, l);
#pragma unroll
      for (int u = 0; u < VU; ++u) {
        float o[64];
        if (n > 0) {
          tmem_ld64(to + u * 64, o);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int k = 0; k < 64; ++k) asm volatile("" : "+f"(o[k]));
        }
        if (i < nq && !whole) {
#pragma unroll
          for (int k = 0; k < 64; ++k) o[k] = n > 0 ? o[k] : 0.f;
#pragma unroll
          for (int c = 0; c < 64; c += 8) store_sector(parts.o + slot * (VU * 64) + u * 64 + c, (const uint32_t*)(o + c));
        } else if (i < nq) {
#pragma unroll
          for (int k = 0; k < 64; ++k) o[k] = n > 0 && l != 0.f ? o[k] * inv : 0.f;
#pragma unroll
          for (int c = 0; c < 64; c += 16) {
            if (u * 64 + c >= a.v_dim) break;
            if (sectors) {
              uint32_t w[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) w[k] = pack2<DT>(o[c + 2 * k], o[c + 2 * k + 1]);
              store_sector((uint16_t*)a.out + at + u * 64 + c, w);
            } else {
              store8<DT>(a.out, at + u * 64 + c, o + c);
              if (u * 64 + c + 8 < a.v_dim) store8<DT>(a.out, at + u * 64 + c + 8, o + c + 8);
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// Adds up the parts of the blocks that have several, in order, and divides. 16 threads a row, 8 values each.
constexpr int LPJ_ROWS = 16;
template <int DT, int VU>
__global__ void __launch_bounds__(LPJ_ROWS * 16) latent_prefill_join_kernel(vq2_latent_prefill_args a, int nqb, LpParts parts) {
  pdl_wait();
  constexpr int per = 2 * LP_TILE / LPJ_ROWS;
  const int block = blockIdx.x / per, r = blockIdx.x % per * LPJ_ROWS + threadIdx.x / 16, d = threadIdx.x % 16 * 8;
  LpBlock w;
  if (!w.at(a, nqb, block) || w.row0 + r >= w.nq || d >= a.v_dim) return;
  const int len = parts.length(w.nsteps);
  if (w.nsteps <= len) return;
  const int count = (w.nsteps + len - 1) / len;
  float n = -INFINITY, l = 0.f, v[8] = {};
#pragma unroll 4
  for (int s = 0; s < count; ++s) {
    // (the main kernel is done: it never signals early, so this launch is only prepared while it runs; each value is read once)
    const size_t slot = ((size_t)block * parts.most + s) * (2 * LP_TILE) + r;
    const float2 ml = __ldcg(parts.ml + slot);
    const float4* p = (const float4*)(parts.o + slot * (VU * 64) + d);
    const float4 x = __ldcg(p), y = __ldcg(p + 1);
    if (ml.y == 0.f) continue;                    // the row saw no key of this part
    const float mx = fmaxf(n, ml.x), f = n == mx ? 1.f : ex2(n - mx), e = ml.x == mx ? 1.f : ex2(ml.x - mx);
    n = mx;
    l = l * f + ml.y * e;
    const float z[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = v[k] * f + z[k] * e;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = l != 0.f ? v[k] * inv : 0.f;
  store8<DT>(a.out, ((long long)(w.q0 + w.row0 + r) * a.heads + w.h) * a.v_dim + d, v);
}

// How the keys are split: not at all where there is a block of queries for every SM; else in the parts that the sizes (sequences taken
// as alike) say are soonest done. A part takes LP_FIXED steps beside its keys, the join LP_JOIN; a schedule ends no later than full
// rounds of parts over the SMs, nor than an even share of all steps and one part more. Whole and split, us on the device, 128 + 64 and
// 128 values: 256 queries after 512, 8 heads 18 and 15; after 4,000, 32 heads 74 and 36; 1,024 after 15,000, 20 heads 241 and 195;
// 1,024 alone, 16 heads 21 and 20; 8,192 alone, 1 head 111 and 34, 4 heads 115 and 97. Where the rule leaves them whole: 512 alone, 8
// heads 14.1; 2,048 alone, 16 heads 35. At most 3 parts an SM: the workspace stays under 60 MB.
constexpr int LP_FIXED = 3, LP_JOIN = 3;          // in key steps (1.8 us)
static LpParts lp_split(const vq2_latent_prefill_args& a, int nqb, int sms) {
  LpParts s = {1, 1 << 30, nullptr, nullptr};
  const long long per = (long long)a.heads * a.B, blocks = nqb * per;
  if (blocks >= sms) return s;
  const int keys = a.total_k / a.B, prefix = std::max(0, (a.total_k - a.total_q) / a.B);
  auto steps_of = [&](int qb) { return (int)((std::min<long long>(keys, prefix + (qb + 1LL) * 2 * LP_TILE) + LP_TILE - 1) / LP_TILE); };
  const int longest = steps_of(nqb - 1);
  long long best = longest + LP_FIXED;
  for (int most = 2; most <= longest && most * blocks <= 3 * sms; ++most) {
    const int len = (longest + most - 1) / most;
    long long all = 0, work = 0;
    for (int qb = 0; qb < nqb; ++qb) {
      all += std::max(1, (steps_of(qb) + len - 1) / len) * per;
      work += steps_of(qb) * per;
    }
    const long long rounds = (all + sms - 1) / sms * (len + LP_FIXED), even = (work + all * LP_FIXED) / sms + len + LP_FIXED;
    const long long cost = std::min(rounds, even) + LP_JOIN;
    if (cost < best) {
      best = cost;
      s.most = most;
      s.steps = len;
    }
  }
  return s;
}
static size_t lp_part_rows(const vq2_latent_prefill_args& a, int nqb, const LpParts& s) {
  return s.most > 1 ? (size_t)nqb * a.heads * a.B * s.most * 2 * LP_TILE : 0;
}

// Tensor map of [rows][heads][dim] 16-bit values with element strides: boxes of 64 values x 1 head x 128 rows.
static int lp_encode(CUtensorMap* m, const void* base, int dim, int heads, int rows, long long stride_h, long long stride_t) {
  if (const int rc = tensor_map_ready()) return rc;
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
  // a dimension of one entry is never stepped over: any legal stride serves
  const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? stride_h : (dim + 7) / 8 * 8) * 2, (cuuint64_t)(rows > 1 ? stride_t : 64 * 1024) * 2};
  const cuuint32_t box[3] = {64, 1, LP_TILE}, one[3] = {1, 1, 1};
  const CUresult r = g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dims, strides, box, one,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? VQ2_OK : VQ2_ERR_CUDA;
}

}  // namespace vq2

using namespace vq2;

static int lp_nqb(int max_q) { return (int)((max_q + 2LL * LP_TILE - 1) / (2 * LP_TILE)); }

extern "C" size_t vq2_latent_prefill_workspace_size(int B, int heads, int v_dim, int max_q, int total_q, int total_k) {
  if (B <= 0 || heads <= 0 || v_dim <= 0 || v_dim > LP_MAX_D || max_q <= 0 || total_q < 0 || total_k < 0) return 0;
  vq2_latent_prefill_args a = {};
  a.B = B;
  a.heads = heads;
  a.total_q = total_q;
  a.total_k = total_k;
  const int nqb = lp_nqb(max_q);
  const size_t rows = lp_part_rows(a, nqb, lp_split(a, nqb, 148));
  return rows ? rows * ((v_dim + 63) / 64 * 64 * 4 + 8) + 256 : 0;
}

extern "C" int vq2_latent_prefill(const vq2_latent_prefill_args* a, void* stream) {
  if (!a) return VQ2_ERR_NULL;
  if (a->B <= 0 || a->heads <= 0 || a->max_q < 0 || a->total_q < 0 || a->total_k < 0 || a->nope_dim <= 0 || a->nope_dim > LP_MAX_D ||
      a->nope_dim % 8 || a->v_dim <= 0 || a->v_dim > LP_MAX_D || a->v_dim % 8 || a->rope_dim < 0 || a->rope_dim > 64 ||
      a->rope_dim % 8 || !(a->scale > 0.f))
    return VQ2_ERR_SHAPE;
  if ((a->q_stride_t | a->q_stride_h | a->k_stride_t | a->k_stride_h | a->v_stride_t | a->v_stride_h | a->r_stride_t) & 7)
    return VQ2_ERR_SHAPE;
  if (a->dtype != VQ2_DT_BF16 && a->dtype != VQ2_DT_F16) return VQ2_ERR_DTYPE;
  if (a->max_q == 0 || a->total_q == 0) return VQ2_OK;
  if (!a->q || !a->cu_q || !a->cu_k || !a->out) return VQ2_ERR_NULL;
  if (a->total_k && (!a->k_nope || !a->v || (a->rope_dim && !a->k_rope))) return VQ2_ERR_NULL;
  if (((uintptr_t)a->q | (uintptr_t)a->k_nope | (uintptr_t)a->v | (uintptr_t)a->k_rope | (uintptr_t)a->out) & 15) return VQ2_ERR_ALIGN;
  const int nqb = lp_nqb(a->max_q);
  const long long blocks = (long long)nqb * a->heads * a->B;
  if (blocks > 0x7FFFFFFFLL) return VQ2_ERR_SHAPE;
  CUtensorMap tq, tk, tr, tv;
  // without keys nothing is loaded; the maps then describe q, so that they are valid
  const bool any = a->total_k > 0;
  int rc = lp_encode(&tq, a->q, a->nope_dim + a->rope_dim, a->heads, a->total_q, a->q_stride_h, a->q_stride_t);
  tk = tr = tv = tq;
  if (!rc && any) rc = lp_encode(&tk, a->k_nope, a->nope_dim, a->heads, a->total_k, a->k_stride_h, a->k_stride_t);
  if (!rc && any) rc = lp_encode(&tv, a->v, a->v_dim, a->heads, a->total_k, a->v_stride_h, a->v_stride_t);
  if (!rc && any && a->rope_dim) rc = lp_encode(&tr, a->k_rope, a->rope_dim, 1, a->total_k, 0, a->r_stride_t);
  if (rc) return rc;
  const int ku = (a->nope_dim + 63) / 64 + (a->rope_dim ? 1 : 0), vu = (a->v_dim + 63) / 64;
  LpParts parts = lp_split(*a, nqb, 148);
  const size_t rows = lp_part_rows(*a, nqb, parts), need = rows * (vu * 64 * 4 + 8) + 256;
  if (rows && a->workspace && a->ws_bytes >= need) {
    parts.o = (float*)(((uintptr_t)a->workspace + 255) & ~(uintptr_t)255);
    parts.ml = (float2*)(parts.o + rows * vu * 64);
  } else {
    parts = {1, 1 << 30, nullptr, nullptr};
  }
  auto join = [&] {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)(blocks * (2 * LP_TILE / LPJ_ROWS)));
    cfg.blockDim = dim3(LPJ_ROWS * 16);
    auto kernel = a->dtype == VQ2_DT_BF16 ? (vu == 1 ? latent_prefill_join_kernel<VQ2_DT_BF16, 1> : latent_prefill_join_kernel<VQ2_DT_BF16, 2>)
                                          : (vu == 1 ? latent_prefill_join_kernel<VQ2_DT_F16, 1> : latent_prefill_join_kernel<VQ2_DT_F16, 2>);
    return cudaLaunchKernelEx(&cfg, kernel, *a, nqb, parts) == cudaSuccess ? VQ2_OK : VQ2_ERR_CUDA;
  };
  auto launch = [&](auto kernel, bool* raised) {
    if (!smem_limit_once(kernel, LP_SMEM, raised)) return VQ2_ERR_CUDA;
    kernel<<<dim3((unsigned)blocks, parts.most), LP_THREADS, LP_SMEM, (cudaStream_t)stream>>>(*a, nqb, parts, tq, tk, tr, tv);
    if (cudaGetLastError() != cudaSuccess) return VQ2_ERR_CUDA;
    return parts.most > 1 ? join() : VQ2_OK;
  };
  auto pick = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    static bool raised[6][64];
    return ku == 1 ? (vu == 1 ? launch(latent_prefill_kernel<DT, 1, 1>, raised[0]) : launch(latent_prefill_kernel<DT, 1, 2>, raised[1]))
         : ku == 2 ? (vu == 1 ? launch(latent_prefill_kernel<DT, 2, 1>, raised[2]) : launch(latent_prefill_kernel<DT, 2, 2>, raised[3]))
                   : (vu == 1 ? launch(latent_prefill_kernel<DT, 3, 1>, raised[4]) : launch(latent_prefill_kernel<DT, 3, 2>, raised[5]));
  };
  return a->dtype == VQ2_DT_BF16 ? pick(std::integral_constant<int, VQ2_DT_BF16>()) : pick(std::integral_constant<int, VQ2_DT_F16>());
}
