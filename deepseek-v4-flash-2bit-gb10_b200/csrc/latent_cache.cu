// K7 latent cache: a token's attention latent (L values, L a multiple of 64) held in 4 bits and its
// rotary key (R values) in fp16, one row per token in a paged cache [pages][page_size][row_bytes].
//
// Every 64 values of the latent are rotated by the normalised Sylvester Hadamard matrix H (symmetric,
// H H = I: the same incoherence rotation the expert weights carry), so a channel that stands out is
// spread over its group and 4 bits serve all 64 values:
//   y = H c,   s = clamp(bf16(max|y| * (1/7)), 2^-14, 2048),   n = clamp(rint(y / s), -7, 7)
// The row stands for c' = H (n s). s has 8 significant bits and |n| <= 7, so n s is exact in fp16
// (and no smaller than 2^-14: normal), which the attention kernel relies on. Values beyond 7 * 2048
// (rotary: 65504) saturate; a NaN makes its group read as NaN, so a fault upstream stays visible.
//
// Row: L/2 bytes of nibbles n + 8 (word w holds values 8w .. 8w+7, value j in bits
// 4 (j >> 1) + 16 (j & 1): one mask leaves a pair of neighbours in the halves of a word), 2 R bytes
// of rotary key, 2 L/64 bytes of fp16 scales, zeros up to a multiple of 16.
#include "vq2_common.cuh"

namespace vq2 {

constexpr int LC_MAX_L = 512, LC_MAX_R = 64;
constexpr float LC_S_MIN = 6.103515625e-05f, LC_S_MAX = 2048.f;   // 2^-14, 2^11
constexpr int LC_THREADS = 256;

__host__ __device__ __forceinline__ int latent_row_bytes(int L, int R) {
  return (L / 2 + 2 * R + 2 * (L / 64) + 15) / 16 * 16;
}
__host__ __device__ __forceinline__ bool latent_dims_ok(int L, int R) {
  return L > 0 && L <= LC_MAX_L && L % 64 == 0 && R >= 0 && R <= LC_MAX_R && R % 8 == 0;
}

// Eight 16-bit values to fp32.
template <int DT>
__device__ __forceinline__ void unpack8(const uint4& r, float* v) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float2 f;
    if (DT == VQ2_DT_BF16) {
      f.x = __uint_as_float(w[k] << 16);
      f.y = __uint_as_float(w[k] & 0xFFFF0000u);
    } else {
      f = __half22float2(*(const __half2*)&w[k]);
    }
    v[2 * k] = f.x;
    v[2 * k + 1] = f.y;
  }
}

// Eight consecutive activations (16-byte aligned for the 2-byte types, 32 for fp32).
template <int DT>
__device__ __forceinline__ void load8(const void* p, size_t i, float* v) {
  if (DT == VQ2_DT_F32) {
    const float4* f = (const float4*)((const float*)p + i);
    const float4 a = __ldg(f), b = __ldg(f + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
  unpack8<DT>(__ldg((const uint4*)((const uint16_t*)p + i)), v);
}

// Two fp32 values rounded to a 16-bit type and packed.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t r;
  if (DT == VQ2_DT_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    r = *(const uint32_t*)&h;
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    r = *(const uint32_t*)&h;
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void store8(void* p, size_t i, const float* v) {
  if (DT == VQ2_DT_F32) {
    float4* f = (float4*)((float*)p + i);
    f[0] = make_float4(v[0], v[1], v[2], v[3]);
    f[1] = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
  *(uint4*)((uint16_t*)p + i) = make_uint4(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]),
                                           pack2<DT>(v[6], v[7]));
}

// H x for a 64-group spread over 8 consecutive lanes (values 8 l .. 8 l + 7 in lane l of the eight):
// butterflies over strides 1, 2, 4 in registers and 8, 16, 32 over lanes, in that order, then 1/8.
__device__ __forceinline__ void fwht64_lanes8(float* v) {
#pragma unroll
  for (int len = 1; len < 8; len <<= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(i & len)) {
        const float a = v[i], b = v[i + len];
        v[i] = a + b;
        v[i + len] = a - b;
      }
#pragma unroll
  for (int len = 1; len < 8; len <<= 1) {
    const bool high = threadIdx.x & len;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = __shfl_xor_sync(0xffffffffu, v[i], len);
      v[i] = high ? o - v[i] : v[i] + o;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= 0.125f;
}

// A thread takes 8 values of a token: U = L/8 threads for the latent and 8 for the rotary part (of
// which R/8 work), so the eight lanes of a group are always neighbours in one warp.
template <int DT>
__global__ void __launch_bounds__(LC_THREADS) latent_write_kernel(const void* __restrict__ c, const void* __restrict__ kr,
                                                                  long long c_stride, long long kr_stride,
                                                                  const void* __restrict__ slots, int slot_dtype, int n,
                                                                  int L, int R, long long capacity, uint8_t* __restrict__ cache) {
  const int U = L / 8 + (R ? 8 : 0), rb = latent_row_bytes(L, R);
  const long long idx = (long long)blockIdx.x * LC_THREADS + threadIdx.x;
  const long long tok = idx / U;
  const int u = (int)(idx - tok * U);
  const bool in = tok < n;
  long long slot = -1;
  if (in) slot = slot_dtype == VQ2_ID_I64 ? ((const long long*)slots)[tok] : ((const int*)slots)[tok];
  if (slot >= capacity) {
    set_status(VQ2_ERR_SHAPE);
    slot = -1;
  }
  uint8_t* row = cache + (slot < 0 ? 0 : slot) * rb;
  float v[8] = {};
  const bool rope = u >= L / 8;
  const int part = rope ? u - L / 8 : u;
  if (slot >= 0 && !rope) load8<DT>(c, (size_t)tok * c_stride + part * 8, v);
  if (slot >= 0 && rope && part * 8 < R) load8<DT>(kr, (size_t)tok * kr_stride + part * 8, v);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = v[i];
  fwht64_lanes8(y);                      // every lane of the warp takes part in the shuffles
  float m = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m = fmaxf(m, fabsf(y[i]));
    nan |= y[i] != y[i];
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    nan |= __shfl_xor_sync(0xffffffffu, (int)nan, o) != 0;
  }
  if (slot < 0) return;
  if (!rope) {
    const float s = fminf(fmaxf(__bfloat162float(__float2bfloat16_rn(m * (1.0f / 7.0f))), LC_S_MIN), LC_S_MAX);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int q = nan ? 0 : (int)fminf(fmaxf(rintf(__fdiv_rn(y[i], s)), -7.f), 7.f);
      w |= (uint32_t)(q + 8) << (4 * (i >> 1) + 16 * (i & 1));
    }
    ((uint32_t*)row)[part] = w;
    if ((part & 7) == 0)
      ((uint16_t*)(row + L / 2 + 2 * R))[part >> 3] = nan ? (uint16_t)0x7FFF : __half_as_ushort(__float2half_rn(s));
    const int pad = rb - (L / 2 + 2 * R + L / 32);     // 0 .. 14 bytes after the scales, an even number
    if (part < pad / 2) ((uint16_t*)(row + rb - pad))[part] = 0;
  } else if (part * 8 < R) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] != v[i] ? v[i] : fminf(fmaxf(v[i], -65504.f), 65504.f);
    store8<VQ2_DT_F16>(row + L / 2, part * 8, v);
  }
}

// H x for a 64-group over two neighbouring lanes, 32 values a lane as 16 packed pairs (2 i, 2 i + 1): butterflies over strides
// 1, 2, 4, 8, 16 in registers and 32 over the lanes, without the 1/8: the same sums, bit for bit, as fwht64_lanes8 makes.
__device__ __forceinline__ void fwht64_lanes2(float2* p) {
#pragma unroll
  for (int i = 0; i < 16; ++i) p[i] = make_float2(p[i].x + p[i].y, p[i].x - p[i].y);
  const float2 minus = make_float2(-1.f, -1.f);
#pragma unroll
  for (int len = 1; len < 16; len <<= 1)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (!(i & len)) {
        const float2 a = p[i], b = p[i + len];
        p[i] = fadd2(a, b);
        p[i + len] = ffma2(b, minus, a);
      }
  const float sign = threadIdx.x & 1 ? -1.f : 1.f;           // the high lane: other - own
  const float2 s2 = make_float2(sign, sign);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 o = make_float2(__shfl_xor_sync(0xffffffffu, p[i].x, 1), __shfl_xor_sync(0xffffffffu, p[i].y, 1));
    p[i] = ffma2(p[i], s2, o);
  }
}

// 32 bytes: eight fp32 values, or sixteen of a 16-bit type (whole sectors, so that a thread may write its run alone).
__device__ __forceinline__ void store_sector(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

// The inverse. A thread expands half a group (16 bytes of nibbles) and rotates it with its neighbour's half: one shuffle a value
// (with a group over 8 lanes it is three, half the instructions), and few enough registers for 1280 threads an SM to cover the
// two dependent reads. All rows' groups come first, then all rows' rotary parts, so that a warp has one kind of work.
// Bound by memory latency: 65,536 rows of 512 + 64 values 32 us in calls back to back (49 with 8 lanes a group, 37 with a thread a
// group), 27 us with other work between, 3.8 TB/s.
template <int DT>
__global__ void __launch_bounds__(LC_THREADS, 5) latent_read_kernel(const uint8_t* __restrict__ cache, const void* __restrict__ slots,
                                                                    int slot_dtype, uint32_t n, int L, int R, long long capacity,
                                                                    void* __restrict__ c, void* __restrict__ kr) {
  const int rb = latent_row_bytes(L, R);
  const uint32_t halves = L / 32, pieces = R / 8, groups = (n * halves + 31) / 32 * 32;     // whole warps
  uint32_t idx = blockIdx.x * LC_THREADS + threadIdx.x;
  const bool rotary = idx >= groups;
  if (rotary) idx -= groups;
  const uint32_t per = rotary ? pieces : halves;
  if (rotary && idx >= n * pieces) return;
  const uint32_t tok = idx / per, u = idx - tok * per;
  long long slot = -1;
  if (tok < n) slot = slot_dtype == VQ2_ID_I64 ? __ldg((const long long*)slots + tok) : __ldg((const int*)slots + tok);
  if (slot >= capacity) {
    set_status(VQ2_ERR_SHAPE);
    slot = -1;
  }
  const uint8_t* row = cache + (slot < 0 ? 0 : slot) * rb;
  if (rotary) {
    float v[8] = {};
    if (slot >= 0) load8<VQ2_DT_F16>(row + L / 2, u * 8, v);
    store8<DT>(kr, (size_t)tok * R + u * 8, v);
    return;
  }
  uint4 q = make_uint4(0, 0, 0, 0);
  float s = 0.f;
  if (slot >= 0) {
    q = __ldg((const uint4*)row + u);
    s = __half2float(__ushort_as_half(__ldg((const uint16_t*)(row + L / 2 + 2 * R) + (u >> 1)))) * 0.125f;
  }
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  const float2 s2 = make_float2(s, s), c2 = make_float2(-24.f * s, -24.f * s);
  float2 p[16];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // nibble u = n + 8 in the top mantissa bits of 16 + u; (16 + u) s/8 - 24 s/8 = n s/8, exact
      const uint32_t lo = w[i] << (19 - 4 * j) & 0x00780000u, hi = (j ? w[i] >> (4 * j - 3) : w[i] << 3) & 0x00780000u;
      p[i * 4 + j] = ffma2(make_float2(__uint_as_float(lo | 0x41800000u), __uint_as_float(hi | 0x41800000u)), s2, c2);
    }
  fwht64_lanes2(p);
  if (tok >= n) return;
  const size_t at = (size_t)tok * L + u * 32;
  if (DT == VQ2_DT_F32) {
#pragma unroll
    for (int k = 0; k < 4; ++k) store_sector((float*)c + at + k * 8, (const uint32_t*)(p + 4 * k));
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = pack2<DT>(p[8 * k + i].x, p[8 * k + i].y);
      store_sector((uint16_t*)c + at + k * 16, v);
    }
  }
}

static int latent_check(const vq2_latent_cache* k) {
  if (!k || !k->data) return VQ2_ERR_NULL;
  if (!latent_dims_ok(k->latent_dim, k->rope_dim) || k->pages <= 0 || k->page_size <= 0) return VQ2_ERR_SHAPE;
  if ((uintptr_t)k->data & 15) return VQ2_ERR_ALIGN;
  return VQ2_OK;
}

}  // namespace vq2

using namespace vq2;

extern "C" size_t vq2_latent_row_bytes(int latent_dim, int rope_dim) {
  return latent_dims_ok(latent_dim, rope_dim) ? (size_t)latent_row_bytes(latent_dim, rope_dim) : 0;
}

extern "C" int vq2_latent_cache_write(const vq2_latent_cache* k, const void* c, const void* k_rope, int dtype,
                                      long long c_stride, long long rope_stride, const void* slots, int slot_dtype, int n,
                                      void* stream) {
  if (const int rc = latent_check(k)) return rc;
  if (n < 0) return VQ2_ERR_SHAPE;
  if (dtype < 0 || dtype > 2 || slot_dtype < 0 || slot_dtype > 1) return VQ2_ERR_DTYPE;
  if (n == 0) return VQ2_OK;
  const int L = k->latent_dim, R = k->rope_dim;
  if (!c || !slots || (R && !k_rope)) return VQ2_ERR_NULL;
  if (c_stride < L || c_stride % 8 || (R && (rope_stride < R || rope_stride % 8))) return VQ2_ERR_SHAPE;
  if (((uintptr_t)c | (uintptr_t)(R ? k_rope : nullptr)) & 15) return VQ2_ERR_ALIGN;
  const long long cap = k->pages * k->page_size, threads = (long long)n * (L / 8 + (R ? 8 : 0));
  const long long blocks = (threads + LC_THREADS - 1) / LC_THREADS;
  if (blocks > 0x7FFFFFFFLL) return VQ2_ERR_SHAPE;
  auto kernel = dtype == VQ2_DT_BF16 ? latent_write_kernel<VQ2_DT_BF16>
              : dtype == VQ2_DT_F16 ? latent_write_kernel<VQ2_DT_F16> : latent_write_kernel<VQ2_DT_F32>;
  kernel<<<(unsigned)blocks, LC_THREADS, 0, (cudaStream_t)stream>>>(c, k_rope, c_stride, rope_stride, slots, slot_dtype, n, L, R,
                                                                    cap, (uint8_t*)k->data);
  return cudaGetLastError() == cudaSuccess ? VQ2_OK : VQ2_ERR_CUDA;
}

extern "C" int vq2_latent_cache_read(const vq2_latent_cache* k, const void* slots, int slot_dtype, int n, void* c, void* k_rope,
                                     int dtype, void* stream) {
  if (const int rc = latent_check(k)) return rc;
  if (n < 0 || n >= 1 << 27) return VQ2_ERR_SHAPE;
  if (dtype < 0 || dtype > 2 || slot_dtype < 0 || slot_dtype > 1) return VQ2_ERR_DTYPE;
  if (n == 0) return VQ2_OK;
  const int L = k->latent_dim, R = k->rope_dim;
  if (!c || !slots || (R && !k_rope)) return VQ2_ERR_NULL;
  if (((uintptr_t)c & 31) | ((uintptr_t)(R ? k_rope : nullptr) & 15)) return VQ2_ERR_ALIGN;
  const long long cap = k->pages * k->page_size;
  const unsigned blocks = ((unsigned)n * (L / 32) + 31 + (unsigned)n * (R / 8) + LC_THREADS - 1) / LC_THREADS;
  auto kernel = dtype == VQ2_DT_BF16 ? latent_read_kernel<VQ2_DT_BF16>
              : dtype == VQ2_DT_F16 ? latent_read_kernel<VQ2_DT_F16> : latent_read_kernel<VQ2_DT_F32>;
  kernel<<<blocks, LC_THREADS, 0, (cudaStream_t)stream>>>((const uint8_t*)k->data, slots, slot_dtype, (uint32_t)n, L, R, cap, c,
                                                                    k_rope);
  return cudaGetLastError() == cudaSuccess ? VQ2_OK : VQ2_ERR_CUDA;
}
