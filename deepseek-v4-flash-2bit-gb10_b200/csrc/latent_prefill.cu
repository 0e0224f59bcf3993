// K9 latent attention, expanded form: causal attention of a ragged batch of prompt chunks. Sequence
// b has query rows cu_q[b] .. cu_q[b+1] - 1 and key rows cu_k[b] .. cu_k[b+1] - 1; its last query sees
// all its keys (a cached prefix comes before them). Keys of head h are [k_nope[:, h], k_rope] with the
// rotary part shared by all heads:
//   z_ij = scale * (q_i . k_j),  j <= i + keys - queries;   out_i = sum_j softmax(z_i)_j v_j
//
// One warp per (query row, head): the lanes hold the row's values, keys come one after another.
#include "vq2_common.cuh"

namespace vq2 {

constexpr int LP_MAX_D = 128;      // values a head: of the positionless key part, and of v

template <int DT>
__global__ void __launch_bounds__(256) latent_prefill_rows_kernel(vq2_latent_prefill_args a) {
  const int lane = threadIdx.x & 31, dn = a.nope_dim, R = a.rope_dim, dv = a.v_dim;
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z;
  // offsets are clamped to the tensors, so wrong ones give wrong rows and no access out of range
  const int q0 = min(max(a.cu_q[b], 0), a.total_q), nq = min(max(a.cu_q[b + 1], q0), a.total_q) - q0;
  const int k0 = min(max(a.cu_k[b], 0), a.total_k), nk = min(max(a.cu_k[b + 1], k0), a.total_k) - k0;
  if (i >= min(nq, a.max_q)) return;
  const long long qi = (long long)(q0 + i) * a.q_stride_t + (long long)h * a.q_stride_h;
  float q[6] = {}, o[4] = {}, m = -INFINITY, l = 0.f;
  for (int p = 0; p < 6; ++p)
    if (lane + 32 * p < dn + R) q[p] = load_act(a.q, DT, qi + lane + 32 * p);
  const int end = min(nk, i + 1 + nk - nq);
  for (int j = 0; j < end; ++j) {
    const long long kj = (long long)(k0 + j) * a.k_stride_t + (long long)h * a.k_stride_h;
    const long long vj = (long long)(k0 + j) * a.v_stride_t + (long long)h * a.v_stride_h;
    float z = 0.f;
    for (int p = 0; p < 6; ++p) {
      const int d = lane + 32 * p;
      if (d < dn) z = fmaf(q[p], load_act(a.k_nope, DT, kj + d), z);
      else if (d < dn + R) z = fmaf(q[p], load_act(a.k_rope, DT, (long long)(k0 + j) * a.r_stride_t + d - dn), z);
    }
    z = warp_sum(z) * a.scale;
    const float mn = fmaxf(m, z), f = expf(m - mn), e = expf(z - mn);
    l = l * f + e;
    for (int p = 0; p < 4; ++p)
      if (lane + 32 * p < dv) o[p] = o[p] * f + e * load_act(a.v, DT, vj + lane + 32 * p);
    m = mn;
  }
  for (int p = 0; p < 4; ++p) {
    const int d = lane + 32 * p;
    if (d >= dv) continue;
    const long long at = ((long long)(q0 + i) * a.heads + h) * dv + d;
    const float v = l > 0.f || l != l ? o[p] / l : 0.f;
    if (DT == VQ2_DT_BF16) ((__nv_bfloat16*)a.out)[at] = __float2bfloat16_rn(v);
    else ((__half*)a.out)[at] = __float2half_rn(v);
  }
}

}  // namespace vq2

using namespace vq2;

extern "C" int vq2_latent_prefill(const vq2_latent_prefill_args* a, void* stream) {
  if (!a) return VQ2_ERR_NULL;
  if (a->B <= 0 || a->heads <= 0 || a->max_q < 0 || a->total_q < 0 || a->total_k < 0 || a->nope_dim <= 0 || a->nope_dim > LP_MAX_D ||
      a->nope_dim % 8 || a->v_dim <= 0 || a->v_dim > LP_MAX_D || a->v_dim % 8 || a->rope_dim < 0 || a->rope_dim > 64 ||
      a->rope_dim % 8 || a->B > 65535 || a->heads > 65535)
    return VQ2_ERR_SHAPE;
  if ((a->q_stride_t | a->q_stride_h | a->k_stride_t | a->k_stride_h | a->v_stride_t | a->v_stride_h | a->r_stride_t) & 7)
    return VQ2_ERR_SHAPE;
  if (a->dtype != VQ2_DT_BF16 && a->dtype != VQ2_DT_F16) return VQ2_ERR_DTYPE;
  if (a->max_q == 0 || a->total_q == 0) return VQ2_OK;
  if (!a->q || !a->cu_q || !a->cu_k || !a->out) return VQ2_ERR_NULL;
  if (a->total_k && (!a->k_nope || !a->v || (a->rope_dim && !a->k_rope))) return VQ2_ERR_NULL;
  if (((uintptr_t)a->q | (uintptr_t)a->k_nope | (uintptr_t)a->v | (uintptr_t)a->k_rope | (uintptr_t)a->out) & 15) return VQ2_ERR_ALIGN;
  auto kernel = a->dtype == VQ2_DT_BF16 ? latent_prefill_rows_kernel<VQ2_DT_BF16> : latent_prefill_rows_kernel<VQ2_DT_F16>;
  kernel<<<dim3((a->max_q + 7) / 8, a->heads, a->B), 256, 0, (cudaStream_t)stream>>>(*a);
  return cudaGetLastError() == cudaSuccess ? VQ2_OK : VQ2_ERR_CUDA;
}
