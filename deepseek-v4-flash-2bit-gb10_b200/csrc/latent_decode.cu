// K8 latent attention, absorbed form: attention of T new tokens a sequence over the 4-bit latent
// cache. For the query row (t, h) of sequence b, with cached rows j = 0 .. kv_len[b] - 1,
//   z_j = scale * (q_c . c_j + q_r . r_j),  j <= kv_len[b] - T + t;   out = sum_j softmax(z)_j c_j
// H is symmetric and H H = I, so q_c . c_j = (H q_c) . (n s)_j and out = H sum_j p_j (n s)_j: the
// kernel rotates the query and the result, never a cached row.
//
// One CTA per query row; a warp streams every eighth cached row, expands it once into registers and
// uses it for both products; running maximum and sum per warp, joined at the end.
#include "vq2_common.cuh"

namespace vq2 {

constexpr int LD_WARPS = 8;

template <int DT>
__global__ void __launch_bounds__(LD_WARPS * 32) latent_decode_rows_kernel(vq2_latent_decode_args a, int rb, long long capacity) {
  __shared__ float qs[LC_MAX_L + LC_MAX_R];
  __shared__ float os[LD_WARPS][LC_MAX_L];
  __shared__ float ms[LD_WARPS], ls[LD_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, L = a.latent_dim, R = a.rope_dim, D = L + R;
  const long long row = blockIdx.x;                       // (b, t, h) flat
  const int b = (int)(row / ((long long)a.T * a.heads)), t = (int)(row / a.heads % a.T);
  for (int u = threadIdx.x; u < (L / 8 + 31) / 32 * 32; u += LD_WARPS * 32) {
    float v[8] = {};
    if (u * 8 < L) load8<DT>(a.q, row * D + u * 8, v);
    fwht64_lanes8(v);
    if (u * 8 < L)
      for (int i = 0; i < 8; ++i) qs[u * 8 + i] = v[i];
  }
  for (int i = threadIdx.x; i < R; i += LD_WARPS * 32) qs[L + i] = load_act(a.q, DT, row * D + L + i);
  __syncthreads();
  const int len = min(max(a.kv_len[b], 0), (int)min((long long)a.max_pages * a.page_size, 0x7FFFFFFFLL));
  const int end = min(len, len - a.T + 1 + t);
  float m = -INFINITY, l = 0.f, o[2][8] = {};
  for (int j = warp; j < end; j += LD_WARPS) {
    const long long page = a.block_table[(size_t)b * a.max_pages + j / a.page_size];
    if (page < 0 || page * a.page_size >= capacity) {
      set_status(VQ2_ERR_SHAPE);
      continue;
    }
    const uint8_t* r = (const uint8_t*)a.cache + (page * a.page_size + j % a.page_size) * rb;
    float k[2][8], z = 0.f;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int w = lane + 32 * p;
      if (w * 8 < L) {
        const uint32_t x = ((const uint32_t*)r)[w];
        const float s = __half2float(__ushort_as_half(((const uint16_t*)(r + L / 2 + 2 * R))[w >> 3]));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          k[p][i] = (float)((int)((x >> (4 * (i >> 1) + 16 * (i & 1))) & 15u) - 8) * s;
          z = fmaf(k[p][i], qs[w * 8 + i], z);
        }
      }
    }
    for (int i = lane; i < R; i += 32) z = fmaf(__half2float(((const __half*)(r + L / 2))[i]), qs[L + i], z);
    z = warp_sum(z) * a.scale;
    const float mn = fmaxf(m, z), f = expf(m - mn), e = expf(z - mn);
    l = l * f + e;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) o[p][i] = (lane + 32 * p) * 8 < L ? o[p][i] * f + e * k[p][i] : 0.f;
    m = mn;
  }
  if (lane == 0) { ms[warp] = m; ls[warp] = l; }
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((lane + 32 * p) * 8 < L) os[warp][(lane + 32 * p) * 8 + i] = o[p][i];
  __syncthreads();
  float mx = -INFINITY, sum = 0.f, f[LD_WARPS];
  for (int w = 0; w < LD_WARPS; ++w) mx = fmaxf(mx, ms[w]);
  for (int w = 0; w < LD_WARPS; ++w) {
    f[w] = ms[w] == -INFINITY ? 0.f : expf(ms[w] - mx);
    sum += f[w] * ls[w];
  }
  for (int u = threadIdx.x; u < (L / 8 + 31) / 32 * 32; u += LD_WARPS * 32) {
    float v[8] = {};
    if (u * 8 < L && sum != 0.f)
      for (int w = 0; w < LD_WARPS; ++w)
        for (int i = 0; i < 8; ++i) v[i] += f[w] * os[w][u * 8 + i];
    for (int i = 0; i < 8; ++i) v[i] = sum != 0.f ? v[i] / sum : 0.f;
    fwht64_lanes8(v);
    if (u * 8 < L) store8<DT>(a.out, row * L + u * 8, v);
  }
}

}  // namespace vq2

using namespace vq2;

extern "C" size_t vq2_latent_decode_workspace_size(int B, int T, int heads, int latent_dim, int rope_dim) {
  if (B <= 0 || T <= 0 || heads <= 0 || !latent_dims_ok(latent_dim, rope_dim)) return 0;
  return 256;
}

extern "C" int vq2_latent_decode(const vq2_latent_decode_args* a, void* ws, size_t ws_bytes, void* stream) {
  if (!a || !a->q || !a->cache || !a->block_table || !a->kv_len || !a->out) return VQ2_ERR_NULL;
  if (a->B <= 0 || a->T <= 0 || a->heads <= 0 || a->page_size <= 0 || a->max_pages <= 0 || a->pages <= 0 ||
      !latent_dims_ok(a->latent_dim, a->rope_dim) || !(a->scale > 0.f) || (long long)a->B * a->T * a->heads > 0x7FFFFFFFLL)
    return VQ2_ERR_SHAPE;
  if (a->dtype != VQ2_DT_BF16 && a->dtype != VQ2_DT_F16) return VQ2_ERR_DTYPE;
  if (((uintptr_t)a->q | (uintptr_t)a->cache | (uintptr_t)a->out) & 15) return VQ2_ERR_ALIGN;
  if (!ws || ws_bytes < vq2_latent_decode_workspace_size(a->B, a->T, a->heads, a->latent_dim, a->rope_dim))
    return VQ2_ERR_WORKSPACE;
  auto kernel = a->dtype == VQ2_DT_BF16 ? latent_decode_rows_kernel<VQ2_DT_BF16> : latent_decode_rows_kernel<VQ2_DT_F16>;
  kernel<<<(unsigned)(a->B * a->T * a->heads), LD_WARPS * 32, 0, (cudaStream_t)stream>>>(
      *a, latent_row_bytes(a->latent_dim, a->rope_dim), a->pages * a->page_size);
  return cudaGetLastError() == cudaSuccess ? VQ2_OK : VQ2_ERR_CUDA;
}
