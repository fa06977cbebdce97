// wqaa_block_gemm_kernel.h - the block-scaled 8-bit product:
//     C[m, n] = sum_b sa[m, b] sw[n / 128, b] sum_{k in block b} a[m, k] w[n, k]
// A block of 128 k is exactly one v_mfma_f32_16x16x128_f8f6f4, so the inner sum is one matrix instruction onto zero and the outer one
// is four float32 fmas a lane with the block's scale.  The weights are the instruction's first operand: a lane then holds four
// consecutive n of ONE row m (n = 4 (lane / 16) + i, m = lane % 16), its scale is one register for the whole fragment column, and
// sw is the same for every n of a wave's weight rows (they lie inside one 128-row tile): sa sw is one product per fragment column.
// Precision: the instruction adds the 8 products of consecutive k with each cut off (towards zero) at 2^-13 of the power of two of the
// largest one, and everything above that level in float32 (measured: a product 2^-13 below the largest of its group of 8 counts, one
// 2^-14 below does not; across groups it counts down to 2^-23).  A result of ordinary data is good to 2^-14.8 in the 2-norm, a
// rounding to float16 costs 2^-12: hence float16 and bfloat16 outputs, and none in float32.
// Operand map of the instruction: lane (r = lane % 16, q = lane / 16) feeds row r and 32 of the 128 k; which 32 is free as long as
// both operands agree - here the 16-byte pieces q and 4 + q of the row's 128 bytes.
#pragma once
#include "wqaa_block.h"

namespace wqaa {

typedef float bf32x4 __attribute__((ext_vector_type(4)));
typedef int bi32x4 __attribute__((ext_vector_type(4)));
typedef int bi32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t bu32x2 __attribute__((ext_vector_type(2)));

// FMT: 0 e4m3, 1 e5m2 (the instruction's format fields); first operand W, second A
template <int WF, int AF>
__device__ __forceinline__ bf32x4 block_mfma(const bi32x4 (&w)[2], const bi32x4 (&a)[2]) {
  const bi32x8 wv = {w[0][0], w[0][1], w[0][2], w[0][3], w[1][0], w[1][1], w[1][2], w[1][3]};
  const bi32x8 av = {a[0][0], a[0][1], a[0][2], a[0][3], a[1][0], a[1][1], a[1][2], a[1][3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, av, bf32x4{0.f, 0.f, 0.f, 0.f}, WF, AF, 0, 0, 0, 0);   // (scales of 0: the form without scales)
}

__device__ __forceinline__ uint16_t block_bf16(float f) {
  const uint32_t u = __builtin_bit_cast(uint32_t, f);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ float block_bias(const void* bias, int dt, int n) {
  if (dt == WQAA_F16) return (float)reinterpret_cast<const _Float16*>(bias)[n];
  return __builtin_bit_cast(float, (uint32_t)reinterpret_cast<const uint16_t*>(bias)[n] << 16);
}
__device__ __forceinline__ void block_store1(void* C, int dt, long i, float v) {
  if (dt == WQAA_F16) reinterpret_cast<_Float16*>(C)[i] = (_Float16)v;
  else reinterpret_cast<uint16_t*>(C)[i] = block_bf16(v);
}
// `n` <= 4 neighbouring elements; four leave as one store, on whatever boundary an odd N puts them (2248 x 22741 x 2560: 228 us with
// a store per element, 176 so)
__device__ __forceinline__ void block_store4(void* C, int dt, long i, int n, const float (&v)[4]) {
  if (n == 4) {
    uint16_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = dt == WQAA_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[e]) : block_bf16(v[e]);
    const bu32x2 w = {b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16};
    __builtin_memcpy(reinterpret_cast<uint16_t*>(C) + i, &w, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < n) block_store1(C, dt, i + e, v[e]);
  }
}

// ---- few rows: the weights stream through registers ------------------------------------------------------------------------------
// One read of W is nearly all there is to do, so nothing is staged: a wave takes NF fragments of 16 weight rows and every WAVES-th
// k-block of them straight into the matrix operand's registers (two 16-byte loads a lane and fragment), the MF fragments of activation rows -
// from L2 - the same way; the waves' partial tiles meet in LDS in a fixed order.  Rows beyond m and n repeat the last one and are
// not stored.  Workgroups along y take 16 MF rows each.  U blocks are asked for at once; PF: the next U before the matrix
// instructions of these.  NF > 1 divides the reads of the activations, which at 16 rows are as many as those of the weights (choose() in
// wqaa_block_gemm.hip has the measured rule).  With more weights in turn than
// the last-level cache holds, 2 GB of them: one row, 28672 x 8192, 38.5 us, 6.1 TB/s; 16 rows, 8192 x 28672, 46 us, 5.1 TB/s (one and the same operands
// again and again: 37.3 and 39.6).
template <int WF, int AF, int WAVES, int U, int NF, int MF, bool PF>
__global__ void __launch_bounds__(WAVES * 64) wq_block_stream_kernel(const BlockGemmArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ __attribute__((aligned(16))) float part[WAVES][NF * 256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int m0 = blockIdx.y * 16 * MF, rows = min(16 * MF, a.M - m0);
  const int n0 = blockIdx.x * 16 * NF;           // (16 NF divides 128: the rows of a workgroup share a weight tile's scales)
  const unsigned char* wp[NF];
#pragma unroll
  for (int g = 0; g < NF; ++g) wp[g] = a.W + (long)min(n0 + g * 16 + r, a.N - 1) * a.K + q * 16;
  const unsigned char* ap[MF];
  const float* sap[MF];
#pragma unroll
  for (int f = 0; f < MF; ++f) {
    const int m = m0 + min(f * 16 + r, rows - 1);
    ap[f] = a.A + (long)m * a.K + q * 16;
    sap[f] = a.sa + m;
  }
  const auto* swp = (const __attribute__((address_space(4))) float*)(a.sw + (long)(n0 / kBlock) * a.KB);
  bf32x4 acc[MF][NF];
#pragma unroll
  for (int f = 0; f < MF; ++f)
#pragma unroll
    for (int g = 0; g < NF; ++g) acc[f][g] = bf32x4{0.f, 0.f, 0.f, 0.f};
  struct Batch {
    bi32x4 w[U][NF][2], x[U][MF][2];
    float sa[U][MF], sw[U];
  };
  auto piece = [](const unsigned char* p) { return *reinterpret_cast<const bi32x4*>(p); };
  auto fetch = [&](Batch& B, int u, int b) {     // block b, whole
    const long k = (long)b * kBlock;
#pragma unroll
    for (int g = 0; g < NF; ++g) B.w[u][g][0] = piece(wp[g] + k), B.w[u][g][1] = piece(wp[g] + k + 64);
#pragma unroll
    for (int f = 0; f < MF; ++f) {
      B.x[u][f][0] = piece(ap[f] + k), B.x[u][f][1] = piece(ap[f] + k + 64);
      B.sa[u][f] = sap[f][(long)b * a.sa_ld];
    }
    B.sw[u] = swp[b];
  };
  auto multiply = [&](const Batch& B) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < MF; ++f) {
        const float s = B.sa[u][f] * B.sw[u];
#pragma unroll
        for (int g = 0; g < NF; ++g) {
          const bf32x4 d = block_mfma<WF, AF>(B.w[u][g], B.x[u][f]);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[f][g][i] = __builtin_fmaf(d[i], s, acc[f][g][i]);
        }
      }
  };
  const int full = a.K / kBlock;                 // blocks that are whole
  const int cnt = full > wave ? (full - wave + WAVES - 1) / WAVES : 0;
  const int nb = cnt / U;
  auto batch = [&](Batch& B, int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(B, u, wave + (i * U + u) * WAVES);
  };
  if constexpr (PF) {
    Batch even, odd;
    if (nb > 0) batch(even, 0);
    int i = 0;
    for (; i + 2 < nb; i += 2) {
      batch(odd, i + 1);
      __builtin_amdgcn_sched_barrier(0);
      multiply(even);
      __builtin_amdgcn_sched_barrier(0);
      batch(even, i + 2);
      __builtin_amdgcn_sched_barrier(0);
      multiply(odd);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (i + 1 < nb) {
      batch(odd, i + 1);
      __builtin_amdgcn_sched_barrier(0);
      multiply(even);
      multiply(odd);
    } else if (nb > 0) {
      multiply(even);
    }
  } else {
    for (int i = 0; i < nb; ++i) {
      Batch B;
      batch(B, i);
      __builtin_amdgcn_sched_barrier(0);
      multiply(B);
    }
  }
  if (nb * U < cnt) {                            // fewer than U blocks left: the others are zero
    Batch B = {};
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (nb * U + u < cnt) fetch(B, u, wave + (nb * U + u) * WAVES);
    multiply(B);
  }
  if (full < a.KB && full % WAVES == wave) {     // the last block holds fewer than 128 k: pieces beyond K are zero in both operands
    const long k = (long)full * kBlock;
    const int left = a.K - full * kBlock - q * 16;
    Batch B = {};
#pragma unroll
    for (int g = 0; g < NF; ++g) {
      if (left > 0) B.w[0][g][0] = piece(wp[g] + k);
      if (left > 64) B.w[0][g][1] = piece(wp[g] + k + 64);
    }
#pragma unroll
    for (int f = 0; f < MF; ++f) {
      if (left > 0) B.x[0][f][0] = piece(ap[f] + k);
      if (left > 64) B.x[0][f][1] = piece(ap[f] + k + 64);
      B.sa[0][f] = sap[f][(long)full * a.sa_ld];
    }
    B.sw[0] = swp[full];
    multiply(B);
  }
#pragma unroll
  for (int f = 0; f < MF; ++f) {                 // one fragment row of the partial tiles at a time
    if (f) __syncthreads();
#pragma unroll
    for (int g = 0; g < NF; ++g) *reinterpret_cast<bf32x4*>(&part[wave][r * (16 * NF) + g * 16 + q * 4]) = acc[f][g];
    __syncthreads();
    for (int t = threadIdx.x; t < 256 * NF; t += WAVES * 64) {
      const int m = f * 16 + t / (16 * NF), n = n0 + t % (16 * NF);
      if (m >= rows || n >= a.N) continue;
      float v = 0.f;
#pragma unroll
      for (int wv = 0; wv < WAVES; ++wv) v += part[wv][t];
      if (a.bias) v += block_bias(a.bias, a.out_dtype, n);
      block_store1(a.C, a.out_dtype, (long)(m0 + m) * a.N + n, v);
    }
  }
#endif
}

// ---- more rows: tiles of BM x 128 through LDS ------------------------------------------------------------------------------------------
// Four waves, S stages of one k-block each, every byte by LDS-DMA.  A stage holds BM activation rows and 128 weight rows of 128 bytes,
// 16-byte piece g of row r at slot g ^ ((r >> 1) & 7) (the lanes of an operand read then hit every bank twice, which is the rate),
// and per wave the scales of its own activation rows (64 of them; rows beyond M read as zero).
// A wave alone on its SIMD spends as long on issuing copies and operand reads as in the matrix unit (neither deeper rings nor operands
// read a block ahead changed that), so a SIMD gets two:
//   G = 1  half a CU's LDS at most, and two workgroups share a CU: for grids that give every CU two tiles or more;
//   G = 2  two such groups of four waves in ONE workgroup, each with its half of the k-blocks and its own ring, one barrier apart: while
//          one reads operands and issues copies (load phase), the other multiplies.  Their sums meet in LDS at the end.  For grids
//          of up to a tile per CU.
// split > 1: the tiles behind the first `whole` have that many workgroups, each with a K slice, which leave float32 partial tiles for the
// reduce launch behind this one: all tiles of a grid that would not fill the chip, or what is left over from its whole rounds.
// TAIL: K is no multiple of 128 (pieces of the last block beyond K are fetched from outside the buffer, which reads as zero)
template <int WF_, int AF_, int BM_, int S_, int G_, bool TAIL_>
struct BlockTile {
  static constexpr bool TAIL = TAIL_;
  static constexpr int WF = WF_, AF = AF_, BM = BM_, BN = 128, S = S_, G = G_, THREADS = 256 * G_;
  static constexpr int WM = 2, WN = 2;                                   // wave grid
  static constexpr int MF = BM / WM / 16, NF = BN / WN / 16;             // fragments of a wave
  static constexpr int A_BYTES = BM * 128, W_BYTES = BN * 128, SC_BYTES = 4 * 256;
  static constexpr int STAGE = A_BYTES + W_BYTES + SC_BYTES;
  static constexpr int AP = BM / 32, WP = BN / 32;                       // DMA pieces (8 rows) of a wave per stage
  static constexpr int PIECES = AP + WP + 1;
  static constexpr int LDS = G * S * STAGE;
  static_assert(LDS <= (G == 1 ? 80 : 160) * 1024 && MF * 16 <= 64, "two groups a CU; one DMA piece holds a wave's row scales");
  static_assert(G == 1 || BM * BN * 4 <= LDS, "the groups' sums meet in LDS");
};

template <int N>
__device__ __forceinline__ void block_wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

#define WQ_BLOCK_BARRIER()                  \
  do {                                      \
    asm volatile("" ::: "memory");          \
    __builtin_amdgcn_sched_barrier(0);      \
    __builtin_amdgcn_s_barrier();           \
    __builtin_amdgcn_sched_barrier(0);      \
    asm volatile("" ::: "memory");          \
  } while (0)

// tile `t` in the order of the walk: group_m M-tiles for each N-tile
__device__ __forceinline__ void block_tile_at(const BlockGemmArgs& a, int blk, int& tile_m, int& tile_n) {
  const int per_group = a.group_m * a.tiles_n;
  const int group = blk / per_group;
  const int first_m = group * a.group_m;
  const int gsz = min(a.group_m, a.tiles_m - first_m);
  const int rem = blk - group * per_group;
  tile_m = first_m + rem % gsz;
  tile_n = rem / gsz;
}
// what this workgroup takes: a tile, and which k-blocks of it.  An XCD's workgroups (index modulo 8) walk neighbouring tiles.
struct BlockShare {
  int tile_m, tile_n, first, end;            // k-blocks first ... end - 1
  long part;                                 // the partial tile that it leaves, or -1: the tile is its own
};
__device__ __forceinline__ BlockShare block_share(const BlockGemmArgs& a) {
  auto walk = [](int i, int n) { return (n & 7) == 0 ? (i & 7) * (n >> 3) + (i >> 3) : i; };
  BlockShare w;
  const int blk = blockIdx.x;
  if (blk < a.whole) {
    block_tile_at(a, walk(blk, a.whole), w.tile_m, w.tile_n);
    w.first = 0, w.end = a.KB, w.part = -1;
  } else {
    const int i = blk - a.whole, t = i / a.split, z = i - t * a.split;
    block_tile_at(a, a.whole + walk(t, a.tiles_m * a.tiles_n - a.whole), w.tile_m, w.tile_n);
    w.first = z * a.split_len, w.end = min(a.KB, w.first + a.split_len), w.part = i;
  }
  return w;
}

template <class P>
__global__ void __launch_bounds__(P::THREADS, 2 / P::G) wq_block_tile_kernel(const BlockGemmArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __attribute__((address_space(3))) void* lds_t;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = wave8 >> 2, wave = wave8 & 3;
  const int r = lane & 15, q = lane >> 4;
  const int wm = wave / P::WN, wn = wave % P::WN;

  const BlockShare share = block_share(a);
  const int tile_m = share.tile_m, tile_n = share.tile_n, s_first = share.first, s_end = share.end;
  // this group's k-blocks: b_first ... b_first + mine - 1; both groups take nt steps
  const int nt = (s_end - s_first + P::G - 1) / P::G;
  const int b_first = s_first + grp * nt, mine = min(nt, s_end - b_first);
  unsigned char* const ring = smem + grp * (P::S * P::STAGE);
  const int m0 = tile_m * P::BM, n0 = tile_n * P::BN;

  // tile-relative buffers: the range ends with the matrix, so rows beyond it read as zero
  const long a_bytes = (long)min(P::BM, a.M - m0) * a.K, w_bytes = (long)min(P::BN, a.N - n0) * a.K;
  const auto a_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(a.A + (long)m0 * a.K), 0, (int)a_bytes, 0x00020000);
  const auto w_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(a.W + (long)n0 * a.K), 0, (int)w_bytes, 0x00020000);
  const int pr = lane >> 3;                                              // row of a piece
  const int g0 = (lane & 7) ^ ((lane >> 4) & 7), g1 = g0 ^ 4;            // source granule of even / odd pieces
  constexpr uint32_t OUT = 0xC0000000u;                                  // beyond every buffer: reads as zero
  const uint32_t va = (uint32_t)(wave * (P::BM / 4) + pr) * (uint32_t)a.K, vw = (uint32_t)(wave * (P::BN / 4) + pr) * (uint32_t)a.K;
  const int sm = m0 + wm * (P::MF * 16) + lane;                          // the row whose scale this lane fetches
  const uint32_t vs = lane < P::MF * 16 && sm < a.M ? (uint32_t)sm * 4u : OUT;
  const int last = a.KB - 1;
  const int tail = a.K - last * kBlock;                                  // k in the last block

  auto stage = [&](int t, int slot) {
    const int b = min(b_first + t, s_end - 1);                           // (beyond the slice: its last block again, never used)
    unsigned char* base = ring + slot * P::STAGE;
    const bool cut = P::TAIL && b == last;
    const bool out0 = cut && g0 * 16 >= tail, out1 = cut && g1 * 16 >= tail;
    const uint32_t k0 = g0 * 16, k1 = g1 * 16;
#pragma unroll
    for (int j = 0; j < P::AP; ++j) {
      const int row = wave * (P::BM / 4) + j * 8;
      const uint32_t v = va + (uint32_t)(j * 8) * (uint32_t)a.K + ((j & 1) ? k1 : k0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(a_rsrc, (lds_t)(base + row * 128), 16, ((j & 1) ? out1 : out0) ? OUT : v, b * kBlock, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < P::WP; ++j) {
      const int row = wave * (P::BN / 4) + j * 8;
      const uint32_t v = vw + (uint32_t)(j * 8) * (uint32_t)a.K + ((j & 1) ? k1 : k0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(w_rsrc, (lds_t)(base + P::A_BYTES + row * 128), 16, ((j & 1) ? out1 : out0) ? OUT : v, b * kBlock, 0, 0);
    }
    // this wave's row scales of the block, 4 bytes a lane
    const auto s_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.sa + (long)b * a.sa_ld), 0, a.M * 4, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(s_rsrc, (lds_t)(base + P::A_BYTES + P::W_BYTES + wave * 256), 4, vs, 0, 0, 0);
  };

  bf32x4 acc[P::MF][P::NF];
#pragma unroll
  for (int f = 0; f < P::MF; ++f)
#pragma unroll
    for (int g = 0; g < P::NF; ++g) acc[f][g] = bf32x4{0.f, 0.f, 0.f, 0.f};
  const int swl = (r >> 1) & 7;
  const int rd0 = r * 128 + ((q ^ swl) * 16), rd1 = r * 128 + (((4 + q) ^ swl) * 16);
  const auto* swp = (const __attribute__((address_space(4))) float*)(a.sw + (long)tile_n * a.KB);

  bi32x4 w[P::NF][2], x[P::MF][2];
  float s[P::MF];
  auto read = [&](int slot) {
    const unsigned char* base = ring + slot * P::STAGE;
#pragma unroll
    for (int g = 0; g < P::NF; ++g) {
      const unsigned char* p = base + P::A_BYTES + (wn * P::NF + g) * 2048;
      w[g][0] = *reinterpret_cast<const bi32x4*>(p + rd0);
      w[g][1] = *reinterpret_cast<const bi32x4*>(p + rd1);
    }
#pragma unroll
    for (int f = 0; f < P::MF; ++f) {
      const unsigned char* p = base + (wm * P::MF + f) * 2048;
      x[f][0] = *reinterpret_cast<const bi32x4*>(p + rd0);
      x[f][1] = *reinterpret_cast<const bi32x4*>(p + rd1);
      s[f] = reinterpret_cast<const float*>(base + P::A_BYTES + P::W_BYTES + wave * 256)[f * 16 + r];
    }
  };
  auto multiply = [&](float sw) {
#pragma unroll
    for (int f = 0; f < P::MF; ++f) s[f] *= sw;
    bf32x4 d[3];
#pragma unroll
    for (int i = 0; i < P::MF * P::NF + 2; ++i) {  // result i's fmas two matrix instructions behind it
      if (i < P::MF * P::NF) d[i % 3] = block_mfma<P::WF, P::AF>(w[i % P::NF], x[i / P::NF]);
      __builtin_amdgcn_sched_barrier(0);
      if (i >= 2) {
        const int j = i - 2;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j / P::NF][j % P::NF][e] = __builtin_fmaf(d[j % 3][e], s[j / P::NF], acc[j / P::NF][j % P::NF][e]);
      }
    }
  };

#pragma unroll
  for (int t = 0; t < P::S - 1; ++t) stage(t, t);
  int slot = 0, fill = P::S - 1;
  if constexpr (P::G == 1) {
    for (int t = 0; t < nt; ++t) {
      const float sw = swp[b_first + t];
      block_wait_vm<(P::S - 2) * P::PIECES>();    // this wave's pieces of block t have landed (one kind of load in flight: in order)
      WQ_BLOCK_BARRIER();                         // everyone's have, and everyone is done with block t - 1, whose slot is filled next
      read(slot);
      __builtin_amdgcn_sched_barrier(0);
      stage(t + P::S - 1, fill);                  // behind the operand reads: its address work runs in their shadow
      __builtin_amdgcn_sched_barrier(0);
      multiply(sw);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (every operand read has long been used: nothing to wait for)
      slot = slot + 1 == P::S ? 0 : slot + 1;
      fill = fill + 1 == P::S ? 0 : fill + 1;
    }
    block_wait_vm<0>();                           // no DMA into LDS outlives the workgroup
  } else {
    block_wait_vm<(P::S - 2) * P::PIECES>();      // block 0
    WQ_BLOCK_BARRIER();
    if (grp == 1) WQ_BLOCK_BARRIER();
    for (int t = 0; t < nt; ++t) {
      // load phase: block t has landed (the wait and the barrier behind the multiply phase before); the slot that is filled held
      // block t - 1, which the whole group had read before the barrier of that load phase
      const float sw = swp[min(b_first + t, s_end - 1)];
      read(slot);
      __builtin_amdgcn_sched_barrier(0);
      stage(t + P::S - 1, fill);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      WQ_BLOCK_BARRIER();
      if (t < mine) multiply(sw);
      block_wait_vm<(P::S - 2) * P::PIECES>();    // block t + 1
      WQ_BLOCK_BARRIER();
      slot = slot + 1 == P::S ? 0 : slot + 1;
      fill = fill + 1 == P::S ? 0 : fill + 1;
    }
    if (grp == 0) WQ_BLOCK_BARRIER();
    block_wait_vm<0>();                           // no copy may land in what follows
    WQ_BLOCK_BARRIER();
    // the second group's sums through LDS, each lane's own fragments (1 KiB a wave and fragment)
    unsigned char* const mine_at = smem + wave * (P::MF * P::NF * 1024) + lane * 16;
    if (grp == 1) {
#pragma unroll
      for (int f = 0; f < P::MF; ++f)
#pragma unroll
        for (int g = 0; g < P::NF; ++g) *reinterpret_cast<bf32x4*>(mine_at + (f * P::NF + g) * 1024) = acc[f][g];
    }
    __syncthreads();
    if (grp == 1) return;
#pragma unroll
    for (int f = 0; f < P::MF; ++f)
#pragma unroll
      for (int g = 0; g < P::NF; ++g) acc[f][g] += *reinterpret_cast<const bf32x4*>(mine_at + (f * P::NF + g) * 1024);
  }

#pragma unroll
  for (int f = 0; f < P::MF; ++f) {
    const int ml = (wm * P::MF + f) * 16 + r, m = m0 + ml;
#pragma unroll
    for (int g = 0; g < P::NF; ++g) {
      const int nl = (wn * P::NF + g) * 16 + q * 4, n = n0 + nl;
      if (share.part >= 0) {                      // a slice: the whole tile, rows and columns beyond the matrix included
        *reinterpret_cast<bf32x4*>(a.ws + (share.part * P::BM + ml) * P::BN + nl) = acc[f][g];
        continue;
      }
      if (m >= a.M || n >= a.N) continue;
      const int cnt = min(4, a.N - n);
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = acc[f][g][i] + (a.bias && i < cnt ? block_bias(a.bias, a.out_dtype, n + i) : 0.f);
      block_store4(a.C, a.out_dtype, (long)m * a.N + n, cnt, v);
    }
  }
#endif
}

// partial tiles of the K slices, in slice order: a workgroup takes 256 x 4 elements of a tile
template <int BN>
__global__ void __launch_bounds__(256) wq_block_reduce_kernel(const BlockGemmArgs a, int bm) {
  constexpr int LANES = BN / 4, ROWS = 256 / LANES;
  const int per_tile = bm / ROWS;
  const int t = blockIdx.x / per_tile, part = blockIdx.x % per_tile, left = a.tiles_m * a.tiles_n - a.whole;
  int tile_m, tile_n;
  block_tile_at(a, a.whole + ((left & 7) == 0 ? (t & 7) * (left >> 3) + (t >> 3) : t), tile_m, tile_n);
  const int ml = part * ROWS + threadIdx.x / LANES, nl = threadIdx.x % LANES * 4;
  const int m = tile_m * bm + ml, n = tile_n * BN + nl;
  if (m >= a.M || n >= a.N) return;
  const float* p = a.ws + ((long)t * a.split * bm + ml) * BN + nl;
  bf32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int z = 0; z < a.split; ++z) v += *reinterpret_cast<const bf32x4*>(p + (long)z * bm * BN);
  const int cnt = min(4, a.N - n);
  float o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = v[i] + (a.bias && i < cnt ? block_bias(a.bias, a.out_dtype, n + i) : 0.f);
  block_store4(a.C, a.out_dtype, (long)m * a.N + n, cnt, o);
}

}  // namespace wqaa
