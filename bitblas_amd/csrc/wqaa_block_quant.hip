// wqaa_block_quant.hip - the elementwise side of the block-scaled 8-bit path: the quantiser (rows, tiles, silu(gate) * up in front)
// and the norm / residual / gate / norm launch that can quantise what it writes.  All but the gated form is bound by HBM: every value is
// read once into registers, and what a block or a row has to know of itself is reduced across lanes while it sits there.
//
// Lane map of both: a lane owns 8 consecutive k, so 16 lanes (one DPP row) own a block of 128 and its maximum is four row rotations.
#include "wqaa_block.h"

namespace wqaa {

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// max over the 16 lanes of a DPP row / sum over them; every lane gets it
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_row(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, dpp_row<0x128>(v));
  v = max(v, dpp_row<0x124>(v));
  v = max(v, dpp_row<0x122>(v));
  return max(v, dpp_row<0x121>(v));
}
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, dpp_row<CTRL>(__builtin_bit_cast(uint32_t, v)));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = dpp_add<0x121>(dpp_add<0x122>(dpp_add<0x124>(dpp_add<0x128>(v))));
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

template <int DT>
__device__ __forceinline__ float load1(const void* p, long i) {
  if constexpr (DT == WQAA_F32) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (DT == WQAA_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
  else return __builtin_bit_cast(float, (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
}

// 8 elements from element i on; `n` of them exist (the others are 0).  VEC: every piece is whole (n is 0 or 8) and on a 16-byte boundary.
// Otherwise a whole piece still moves as one: the global memory instructions take any address (rows of 2995 elements, 1056 of them with a
// gate and a float32 stream, take 13 us instead of 30, 4096 x 8191 quantise in 36 instead of 57), and only a row's last lane goes element by element.
template <class V>
__device__ __forceinline__ V piece(const void* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void* p, long i, int n, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  if (n <= 0) return;
  if (!VEC && n < 8) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) v[e] = load1<DT>(p, i + e);
  } else if constexpr (DT == WQAA_F32) {
    const f32x4_t a = piece<f32x4_t>(reinterpret_cast<const float*>(p) + i);
    const f32x4_t b = piece<f32x4_t>(reinterpret_cast<const float*>(p) + i + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
  } else if constexpr (DT == WQAA_F16) {
    const f16x8_t a = piece<f16x8_t>(reinterpret_cast<const _Float16*>(p) + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
  } else {
    const u32x4_t a = piece<u32x4_t>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __builtin_bit_cast(float, (e & 1) ? a[e >> 1] & 0xFFFF0000u : a[e >> 1] << 16);
  }
}

__device__ __forceinline__ uint16_t bf16_bits(float f) {      // to nearest even; a NaN stays one
  const uint32_t u = __builtin_bit_cast(uint32_t, f);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

template <int DT, bool VEC>
__device__ __forceinline__ void store8(void* p, long i, int n, const float (&v)[8]) {
  if (n <= 0) return;
  if constexpr (DT == WQAA_F32) {
    float* o = reinterpret_cast<float*>(p) + i;
    if (VEC || n == 8) {
      const f32x4_t a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
      __builtin_memcpy(o, &a, 16);
      __builtin_memcpy(o + 4, &b, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < n) o[e] = v[e];
    }
  } else {
    uint16_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = DT == WQAA_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[e]) : bf16_bits(v[e]);
    uint16_t* o = reinterpret_cast<uint16_t*>(p) + i;
    if (VEC || n == 8) {
      const u32x4_t w = {b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16, b[4] | (uint32_t)b[5] << 16, b[6] | (uint32_t)b[7] << 16};
      __builtin_memcpy(o, &w, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < n) o[e] = b[e];
    }
  }
}

// |x| as ordered bits: the integer maximum lets a NaN through (fmaxf would drop it)
__device__ __forceinline__ uint32_t abs_max8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __builtin_bit_cast(uint32_t, v[e]) & 0x7FFFFFFFu);
  return m;
}

constexpr uint32_t kFloorBits = 0x2B800000u;   // 2^-40: a scale is never so small that its reciprocal leaves float32's normal range

__device__ __forceinline__ float block_scale(uint32_t amax_bits, int q_dtype) {
  return __builtin_bit_cast(float, max(amax_bits, kFloorBits)) / (q_dtype == WQAA_E4M3 ? 448.f : 57344.f);
}

// x / s for 8 values of a block, rounded to 8 bits.  r = 1 / s correctly rounded once per block; x r is within an ulp of the
// quotient, its remainder x - (x r) s is exact in one fma, and adding remainder * r gives the correctly rounded quotient
// (P. Markstein, IBM J. Res. Dev. 34, 1990): 3 operations a value instead of a division.  s is infinite or NaN: the remainder is NaN.
// The remainder is taken negated, n = (x r) s - x: where it vanishes n is +0, and -n r = -0 leaves x r as it is, a -0 of x's included.
// LO: the value is v + lo, lo what v's own rounding lost; it joins the remainder.
template <bool LO = false>
__device__ __forceinline__ u32x2_t quantise8(const float (&v)[8], float s, int q_dtype, const float* lo = nullptr) {
  const float r = 1.f / s;
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = v[e] * r;
    float n = __builtin_fmaf(t, s, -v[e]);
    if constexpr (LO) n -= lo[e];
    q[e] = __builtin_fmaf(-n, r, t);
  }
  int w[2] = {0, 0};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (q_dtype == WQAA_E4M3) {
      w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h], q[4 * h + 1], w[h], false);
      w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h + 2], q[4 * h + 3], w[h], true);
    } else {
      w[h] = __builtin_amdgcn_cvt_pk_bf8_f32(q[4 * h], q[4 * h + 1], w[h], false);
      w[h] = __builtin_amdgcn_cvt_pk_bf8_f32(q[4 * h + 2], q[4 * h + 3], w[h], true);
    }
  }
  return u32x2_t{(uint32_t)w[0], (uint32_t)w[1]};
}

template <bool VEC>
__device__ __forceinline__ void store_q(unsigned char* q, int n, u32x2_t w) {
  if (n <= 0) return;
  if (VEC || n == 8) {
    __builtin_memcpy(q, &w, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) q[e] = (unsigned char)(w[e >> 2] >> (8 * (e & 3)));
  }
}

// silu(g) * u = u g / (1 + 2^(-g log2 e)), off by 2 + 3 sigmoid(-g) roundings at most down to g = -83: the exponent's argument in two
// parts, the reciprocal with one Newton step, and in `lo` what the two products round off.  (A value next to a border between two 8-bit
// values is decided by that: with a plain exponential and reciprocal some ten times as many values fell on the other side.)  Below -83
// exp(-g) is within 2^8 of leaving float32: the reciprocal is the plain one of 1 + exp(-g), and 0 from 2^126 on.
__device__ __forceinline__ float gated(float g, float u, float& lo) {
  constexpr float kL = 1.44269502f, kLLo = 1.92596299e-8f;               // log2 e = kL + kLLo
  const float t = -g * kL;
  const float t_lo = __builtin_fmaf(-g, kL, -t) - g * kLLo;
  const float e2 = __builtin_amdgcn_exp2f(t);
  const float y = 1.f + __builtin_fmaf(e2 * t_lo, 0.693147182f, e2);
  const float r0 = __builtin_amdgcn_rcpf(y);
  // |t| of 120 and more: 2^t is or nears infinity, r 0; or it is 0, r 1, where t_lo may have overflowed (0 t_lo a NaN)
  const float r = __builtin_fabsf(t) < 120.f ? __builtin_fmaf(__builtin_fmaf(-y, r0, 1.f), r0, r0) : __builtin_amdgcn_rcpf(1.f + e2);
  const float c = g * r;
  const float p = c * u;
  lo = __builtin_fmaf(c, u, -p) + __builtin_fmaf(g, r, -c) * u;
  return p;
}

struct QuantArgs {
  const void* x;
  const void* gate;
  unsigned char* q;
  float* s;
  long rows, K, x_ld, gate_ld, s_ld;
  int kb, q_dtype, chunks;          // chunks: workgroups along K
};

// rows: a workgroup takes 16 rows x 4 blocks, so a block's 16 scales leave as one 64-byte piece.  4096 x 8192 bfloat16 21 us, 4.8 TB/s.  With a
// gate the vector unit sets the time (1250 instructions for a lane's 32 values, busy 0.86 of the cycles): 4096 x 28672 143 us, 4.1 TB/s; 16 x 28672 5.9 us,
// 56 workgroups, each lane's four rows one after another.
template <int DT, bool GATED, bool VEC>
__global__ void __launch_bounds__(256) wq_block_quant_rows_kernel(const QuantArgs a) {
  const long wg = blockIdx.x;
  const long r0 = wg / a.chunks * 16;
  const int b0 = (int)(wg % a.chunks) * 4;
  const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int b = b0 + (g & 3);
  const long col = (long)b * kBlock + l * 8;
  const int n = b < a.kb ? (int)min(8L, a.K - col) : 0;
  float x[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long row = r0 + i * 4 + (g >> 2);
    load8<DT, VEC>(a.x, row * a.x_ld + col, row < a.rows ? n : 0, x[i]);
  }
  float lo[4][8];
  if constexpr (GATED) {
    float gt[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long row = r0 + i * 4 + (g >> 2);
      load8<DT, VEC>(a.gate, row * a.gate_ld + col, row < a.rows ? n : 0, gt[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = gated(gt[i][e], x[i][e], lo[i][e]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long row = r0 + i * 4 + (g >> 2);
    const float s = block_scale(row_max(abs_max8(x[i])), a.q_dtype);
    const u32x2_t w = quantise8<GATED>(x[i], s, a.q_dtype, lo[i]);
    if (row < a.rows) {
      store_q<VEC>(a.q + row * a.K + col, n, w);
      if (l == 0 && b < a.kb) a.s[(long)b * a.s_ld + row] = s;
    }
  }
}

// tiles: a workgroup takes one 128 x 128 tile, 8 rows of it in each lane's registers
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) wq_block_quant_tile_kernel(const QuantArgs a) {
  __shared__ uint32_t wmax[4];
  const long wg = blockIdx.x;
  const long r0 = wg / a.kb * kBlock;
  const int b = (int)(wg % a.kb);
  const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
  const long col = (long)b * kBlock + l * 8;
  const int n = (int)min(8L, a.K - col);
  float x[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = r0 + i * 16 + g;
    load8<DT, VEC>(a.x, row * a.x_ld + col, row < a.rows ? n : 0, x[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, abs_max8(x[i]));
  m = row_max(m);
  m = max(m, (uint32_t)__shfl_xor((int)m, 16));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32));
  if ((threadIdx.x & 63) == 0) wmax[threadIdx.x >> 6] = m;
  __syncthreads();
  m = max(max(wmax[0], wmax[1]), max(wmax[2], wmax[3]));
  const float s = block_scale(m, a.q_dtype);
  if (threadIdx.x == 0) a.s[wg] = s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = r0 + i * 16 + g;
    const u32x2_t w = quantise8(x[i], s, a.q_dtype);
    if (row < a.rows) store_q<VEC>(a.q + row * a.K + col, n, w);
  }
}

struct NormArgs {
  wqaa_residual_norm_args p;
};

// One workgroup per row, the row in registers (NV vectors of 8 a lane): read once, two reductions, written once.
template <int DT, bool SF32, int NV, bool VEC>
__global__ void __launch_bounds__(1024) wq_residual_norm_kernel(const NormArgs na) {
  constexpr int ST = SF32 ? WQAA_F32 : DT;
  const wqaa_residual_norm_args& a = na.p;
  __shared__ float part[2][16];
  const long row = blockIdx.x;
  const int T = blockDim.x, waves = T >> 6, wave = threadIdx.x >> 6;
  long col[NV];
  int n[NV];
  float h[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    col[v] = ((long)v * T + threadIdx.x) * 8;
    n[v] = (int)max(0L, min(8L, (long)a.D - col[v]));
    load8<DT, VEC>(a.x, row * a.x_ld + col[v], n[v], h[v]);
  }
  float res[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) load8<ST, VEC>(a.residual, row * a.residual_ld + col[v], a.residual ? n[v] : 0, res[v]);
  const float inv_d = 1.f / (float)a.D;
  // mean of squares; every square is divided by D before it is added, so the sum overflows only where the mean does
  auto row_mean = [&](int which) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) s = __builtin_fmaf(h[v][e] * inv_d, h[v][e], s);
    s = wave_sum(s);
    if (waves == 1) return s;
    if ((threadIdx.x & 63) == 0) part[which][wave] = s;
    __syncthreads();
    float t = 0.f;
    for (int w = 0; w < waves; ++w) t += part[which][w];
    return t;
  };
  auto load_weight = [&](const void* w, int v, float (&wt)[8]) {
    if (a.weight_dtype == WQAA_F32) load8<WQAA_F32, VEC>(w, col[v], n[v], wt);
    else load8<DT, VEC>(w, col[v], n[v], wt);
  };
  if (a.post_weight) {
    const float r = 1.f / sqrtf(row_mean(0) + a.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float wt[8];
      load_weight(a.post_weight, v, wt);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[v][e] = h[v][e] * r * wt[e];
    }
  }
  if (a.gate) {
    const long grow = row / a.gate_rows * a.gate_ld;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float g[8];
      load8<DT, VEC>(a.gate, grow + col[v], n[v], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[v][e] *= g[e];
    }
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[v][e] *= a.scale;
      if (a.residual) h[v][e] = __builtin_fmaf(a.residual_scale, res[v][e], h[v][e]);
    }
    if (a.stream) store8<ST, VEC>(a.stream, row * a.D + col[v], n[v], h[v]);
  }
  if (!a.Y) return;
  const float r = 1.f / sqrtf(row_mean(1) + a.eps);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float y[8], lo[8];
    load_weight(a.weight, v, y);
    // h r w in two products; what they round off (lo) matters only next to a border between two 8-bit values, where it decides
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = r * y[e];
      const float p = h[v][e] * c;
      lo[e] = __builtin_fmaf(h[v][e], c, -p) + h[v][e] * __builtin_fmaf(r, y[e], -c);
      y[e] = p;
    }
    if (a.q_dtype < 0) {
      store8<DT, VEC>(a.Y, row * a.D + col[v], n[v], y);
    } else {
      const float s = block_scale(row_max(abs_max8(y)), a.q_dtype);
      store_q<VEC>(reinterpret_cast<unsigned char*>(a.Y) + row * a.D + col[v], n[v], quantise8<true>(y, s, a.q_dtype, lo));
      if ((threadIdx.x & 15) == 0 && n[v] > 0) a.S[col[v] / kBlock * a.s_ld + row] = s;
    }
  }
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
int esize(int dt) { return dt == WQAA_F32 ? 4 : 2; }

template <typename K, typename A>
int launch(K kernel, long grid, int threads, const A& args, hipStream_t stream, const char* what) {
  kernel<<<dim3((unsigned)grid), dim3(threads), 0, stream>>>(args);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error(WQAA_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
    return WQAA_ERR_LAUNCH;
  }
  return WQAA_OK;
}

int too_many(double grid, int threads, const char* what) {               // (double: the product of two 64-bit numbers)
  if (grid * threads <= 4294967295.0) return WQAA_OK;
  set_error(WQAA_ERR_UNSUPPORTED, "%s: too many rows for one launch", what);
  return WQAA_ERR_UNSUPPORTED;
}
int norm_vectors(int64_t D) { return (int)((D + 7) / 8) <= 1024 ? 1 : (int)((D + 7) / 8) <= 2048 ? 2 : 4; }     // 8-element pieces of a lane
int norm_threads(int64_t D) { return (int)(((D + 7) / 8 + norm_vectors(D) - 1) / norm_vectors(D) + 63) / 64 * 64; }

}  // namespace

int block_quantize_check(const wqaa_block_quant& q) {
  const bool f16 = q.x_dtype == WQAA_F16, bf16 = q.x_dtype == WQAA_BF16, f32 = q.x_dtype == WQAA_F32;
  if ((!f16 && !bf16 && !f32) || (q.q_dtype != WQAA_E4M3 && q.q_dtype != WQAA_E5M2) || (q.tile && q.gate) || q.K > (1l << 30)) {
    set_error(WQAA_ERR_UNSUPPORTED, "block_quantize: float16 / bfloat16 / float32 to e4m3 / e5m2; a gate goes with rows only");
    return WQAA_ERR_UNSUPPORTED;
  }
  if (q.rows > (1l << 40)) return too_many((double)q.rows, 256, "block_quantize");      // (below, rounding up leaves no 64 bits)
  const double blocks = (double)((q.K + kBlock - 1) / kBlock);
  return too_many(q.tile ? (double)((q.rows + kBlock - 1) / kBlock) * blocks : (double)((q.rows + 15) / 16) * (double)(((long)blocks + 3) / 4), 256, "block_quantize");
}

int block_quantize_launch(const wqaa_block_quant& q, hipStream_t stream) {
  const bool f16 = q.x_dtype == WQAA_F16, bf16 = q.x_dtype == WQAA_BF16;
  QuantArgs a;
  a.x = q.X, a.gate = q.gate, a.q = reinterpret_cast<unsigned char*>(q.Q), a.s = q.S;
  a.rows = q.rows, a.K = q.K, a.x_ld = q.x_ld, a.gate_ld = q.gate_ld, a.s_ld = q.s_ld;
  a.kb = (int)((q.K + kBlock - 1) / kBlock), a.q_dtype = q.q_dtype, a.chunks = (a.kb + 3) / 4;
  // vector form: whole 8-element pieces, every row of every operand on a 16-byte boundary (8 for the bytes)
  const bool vec = q.K % 8 == 0 && aligned(q.X, 16) && q.x_ld * esize(q.x_dtype) % 16 == 0 && aligned(q.Q, 8) &&
                   (!q.gate || (aligned(q.gate, 16) && q.gate_ld * esize(q.x_dtype) % 16 == 0));
  if (q.tile) {
    const long grid = (q.rows + kBlock - 1) / kBlock * a.kb;
#define WQ_GO(DT) return vec ? launch(wq_block_quant_tile_kernel<DT, true>, grid, 256, a, stream, "block_quantize") : launch(wq_block_quant_tile_kernel<DT, false>, grid, 256, a, stream, "block_quantize")
    if (f16) WQ_GO(WQAA_F16);
    if (bf16) WQ_GO(WQAA_BF16);
    WQ_GO(WQAA_F32);
#undef WQ_GO
  }
  const long grid = (q.rows + 15) / 16 * a.chunks;
#define WQ_GO(DT, G) return vec ? launch(wq_block_quant_rows_kernel<DT, G, true>, grid, 256, a, stream, "block_quantize") : launch(wq_block_quant_rows_kernel<DT, G, false>, grid, 256, a, stream, "block_quantize")
  if (q.gate) {
    if (f16) WQ_GO(WQAA_F16, true);
    if (bf16) WQ_GO(WQAA_BF16, true);
    WQ_GO(WQAA_F32, true);
  }
  if (f16) WQ_GO(WQAA_F16, false);
  if (bf16) WQ_GO(WQAA_BF16, false);
  WQ_GO(WQAA_F32, false);
#undef WQ_GO
}

template <int DT, bool SF32>
static int norm_go(const NormArgs& a, int nv, int threads, bool vec, hipStream_t stream) {
#define WQ_GO(NV) return vec ? launch(wq_residual_norm_kernel<DT, SF32, NV, true>, a.p.rows, threads, a, stream, "residual_norm") : launch(wq_residual_norm_kernel<DT, SF32, NV, false>, a.p.rows, threads, a, stream, "residual_norm")
  if (nv == 1) WQ_GO(1);
  if (nv == 2) WQ_GO(2);
  WQ_GO(4);
#undef WQ_GO
}

int residual_norm_check(const wqaa_residual_norm_args& n) {
  const bool f16 = n.x_dtype == WQAA_F16, bf16 = n.x_dtype == WQAA_BF16;
  auto same_or_f32 = [&](int t) { return t == n.x_dtype || t == WQAA_F32; };
  if ((!f16 && !bf16) || !same_or_f32(n.stream_dtype) || !same_or_f32(n.weight_dtype) || n.D > 32768 ||
      (n.q_dtype >= 0 && n.q_dtype != WQAA_E4M3 && n.q_dtype != WQAA_E5M2)) {
    set_error(WQAA_ERR_UNSUPPORTED, "residual_norm: float16 / bfloat16 rows of up to 32768, stream and weights of that type or float32");
    return WQAA_ERR_UNSUPPORTED;
  }
  return too_many((double)n.rows, norm_threads(n.D), "residual_norm");
}

int residual_norm_launch(const wqaa_residual_norm_args& n, hipStream_t stream) {
  const bool f16 = n.x_dtype == WQAA_F16;
  NormArgs a;
  a.p = n;
  const int xs = 2, ss = esize(n.stream_dtype);
  const bool vec = n.D % 8 == 0 && aligned(n.x, 16) && n.x_ld * xs % 16 == 0 && (!n.residual || (aligned(n.residual, 16) && n.residual_ld * ss % 16 == 0)) &&
                   (!n.gate || (aligned(n.gate, 16) && n.gate_ld * xs % 16 == 0)) && aligned(n.post_weight, 16) && aligned(n.weight, 16) &&
                   aligned(n.stream, 16) && aligned(n.Y, 16);
  const int nv = norm_vectors(n.D), threads = norm_threads(n.D);
  if (f16) return n.stream_dtype == WQAA_F32 ? norm_go<WQAA_F16, true>(a, nv, threads, vec, stream) : norm_go<WQAA_F16, false>(a, nv, threads, vec, stream);
  return n.stream_dtype == WQAA_F32 ? norm_go<WQAA_BF16, true>(a, nv, threads, vec, stream) : norm_go<WQAA_BF16, false>(a, nv, threads, vec, stream);
}

}  // namespace wqaa
