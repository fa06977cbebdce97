// wqaa_block_pp_kernel.h - the block-scaled product's member for many rows: 256 x 256 tiles, two role groups of four waves.
//
// The matrix unit is to run without a pause, and each of its results has four fmas behind it (the block's scale onto the running
// sum): 32 matrix cycles next to 16 vector cycles, which fit under the NEXT result's matrix cycles of the same wave.  Everything
// else - operand reads, copies, scales, barriers - happens in the other role group's time:
//   * waves 0-3 and 4-7 (one of each on every SIMD) run the same instruction stream one barrier apart: while one is in a COMPUTE
//     segment (16 matrix instructions), its partner is in a LOAD segment (operands of its next 16 from LDS, its share of the copies);
//   * wave grid 2 (m) x 4 (n): a wave owns 128 activation rows x 64 weight rows, 8 x 4 fragments, two segments per k-block;
//   * every byte of A and W arrives by LDS-DMA: rings of 3 activation and 2 weight tiles of 32 KiB, the CU's whole 160 KiB.  W(t + 2) goes into
//     W(t)'s slot from load segment 1 of block t on - behind both groups' reads of W(t), which are in segment 0, two barriers and one barrier
//     earlier - and A(t + 2) into A(t - 1)'s slot from load segment 0 of block t on.  A wave issues 8 pieces per block in one order, so
//     "block t + 1 has landed" is vmcnt(8) at the end of segment 1: at most block t + 2's pieces are then in flight, and every other
//     load of the wave is older than they are or makes the wait stricter;
//   * row scales: which 16 of a wave's 128 rows a fragment takes is free, and fragment f takes rows 8 r + f: lane r then needs the scales
//     of 8 neighbouring rows, two 16-byte loads a block (a block ahead) and no exchange between lanes (with rows in order, two 4-byte
//     loads and lane swaps, 4096 x 28672 x 8192 took 790 us instead of 768); the weight tile's scale is a scalar.  In LDS a fragment's rows
//     lie together, so the copies permute them: LDS row 16 f + r of a 128-row half holds row 8 r + f.
#pragma once
#include "wqaa_block_gemm_kernel.h"

namespace wqaa {

typedef bi32x4 bi32x4_at2 __attribute__((aligned(2)));

struct BlockPP {
  static constexpr int BM = 256, BN = 256, THREADS = 512;
  static constexpr int SLOT = 256 * 128, W_OFF = 3 * SLOT, LDS = 5 * SLOT;
  static_assert(LDS == 160 * 1024 && LDS >= BM * BN * 2, "the rings fill LDS; the epilogue stages the tile there");
};

// TAIL: K is no multiple of 128 (pieces of the last block beyond K are fetched from outside the buffer, which reads as zero)
template <int WF, int AF, bool TAIL>
__global__ void __launch_bounds__(BlockPP::THREADS) wq_block_pp_kernel(const BlockGemmArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using P = BlockPP;
  typedef __attribute__((address_space(3))) void* lds_t;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = wave >> 2, nq = wave & 3;
  const int r = lane & 15, q = lane >> 4;

  const BlockShare share = block_share(a);
  const int m0 = share.tile_m * P::BM, n0 = share.tile_n * P::BN;
  const int nt = share.end - share.first, k0 = share.first * kBlock;     // a slice: everything below starts at its first block

  const long a_bytes = (long)min(P::BM, a.M - m0) * a.K - k0, w_bytes = (long)min(P::BN, a.N - n0) * a.K - k0;
  const auto a_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(a.A + (long)m0 * a.K + k0), 0, (int)a_bytes, 0x00020000);
  const auto w_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(a.W + (long)n0 * a.K + k0), 0, (int)w_bytes, 0x00020000);
  constexpr uint32_t OUT = 0xC0000000u;
  const int g0 = (lane & 7) ^ ((lane >> 4) & 7);
  // first row of the wave's pieces: W's rows in order, A's as LDS rows 32 wave + 8 j + lane / 8 hold them (j & 1: 64 rows on, j / 2: one)
  const uint32_t w_row = wave * 32 + (lane >> 3), a_row = grp * 128 + (lane >> 3) * 8 + nq * 2;
  const int tail = a.K - k0 - (nt - 1) * kBlock;                          // (a slice that is not the last: more than a block)
  const bool cut0 = TAIL && g0 * 16 >= tail, cut1 = TAIL && (g0 ^ 4) * 16 >= tail;

  auto piece = [&](const auto& rsrc, uint32_t row, unsigned char* dst, int tt, int j) {
    const int tc = min(tt, nt - 1);                                       // (beyond the last block: it again, never used)
    uint32_t v = row * (uint32_t)a.K + ((j & 1) ? g0 ^ 4 : g0) * 16;
    if constexpr (TAIL) v = (tc == nt - 1 && ((j & 1) ? cut1 : cut0)) ? OUT : v;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_t)(dst + (wave * 32 + j * 8) * 128), 16, v, tc * kBlock, 0, 0);
  };
  auto dma_a = [&](int tt, int slot, int j) { piece(a_rsrc, a_row + (j & 1) * 64 + (j >> 1), smem + slot * P::SLOT, tt, j); };
  auto dma_w = [&](int tt, int slot, int j) { piece(w_rsrc, w_row + j * 8, smem + P::W_OFF + slot * P::SLOT, tt, j); };

  const uint32_t srow = (uint32_t)(m0 + grp * 128 + r * 8) * 4u;
  bf32x4 raw[2];
  auto fetch_scales = [&](int tt) {                                       // rows beyond M are outside the buffer: zero
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.sa + (long)(share.first + min(tt, nt - 1)) * a.sa_ld), 0, a.M * 4, 0x00020000);
    raw[0] = __builtin_bit_cast(bf32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, srow, 0, 0));
    raw[1] = __builtin_bit_cast(bf32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, srow + 16u, 0, 0));
  };
  const int nb = min((n0 + nq * 64) / kBlock, (a.N - 1) / kBlock);
  const auto* swp = (const __attribute__((address_space(4))) float*)(a.sw + (long)nb * a.KB + share.first);

  const int swl = (r >> 1) & 7;
  const int rd0 = r * 128 + ((q ^ swl) * 16), rd1 = r * 128 + (((4 + q) ^ swl) * 16);
  bf32x4 acc[8][4];
#pragma unroll
  for (int f = 0; f < 8; ++f)
#pragma unroll
    for (int g = 0; g < 4; ++g) acc[f][g] = bf32x4{0.f, 0.f, 0.f, 0.f};
  bi32x4 af[4][2], wf[4][2];
  float s[8] = {};

  fetch_scales(0);
  float sw = swp[0];
#pragma unroll
  for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
    for (int j = 0; j < 4; ++j) dma_a(tt, tt, j);
#pragma unroll
    for (int j = 0; j < 4; ++j) dma_w(tt, tt, j);
  }
  block_wait_vm<8>();
  WQ_BLOCK_BARRIER();
  if (grp == 1) WQ_BLOCK_BARRIER();
  auto scale4 = [&](bf32x4 v, float* to) {
#pragma unroll
    for (int f = 0; f < 4; ++f) to[f] = v[f] * sw;
  };
  scale4(raw[0], s);

  bf32x4 d[3] = {};
  auto scaled = [&](auto PH, int j) {                               // result j of segment PH onto its sums
    constexpr int p = decltype(PH)::value;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[p * 4 + (j >> 2)][j & 3][e] = __builtin_fmaf(d[j % 3][e], s[p * 4 + (j >> 2)], acc[p * 4 + (j >> 2)][j & 3][e]);
  };
  // the last two results of a compute segment are still in the matrix unit at its barrier: their fmas are the next load segment's
  auto finish = [&](auto PH) {
    scaled(PH, 14);
    scaled(PH, 15);
  };
  int slot = 0;
  auto load_segment = [&](auto PH, int t) {
    constexpr int p = decltype(PH)::value;
    if constexpr (p == 0) {
      const unsigned char* ws = smem + P::W_OFF + (t & 1) * P::SLOT + nq * 8192;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        wf[g][0] = *reinterpret_cast<const bi32x4*>(ws + g * 2048 + rd0);
        wf[g][1] = *reinterpret_cast<const bi32x4*>(ws + g * 2048 + rd1);
      }
    }
    const unsigned char* as = smem + slot * P::SLOT + (grp * 8 + p * 4) * 2048;
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      af[f][0] = *reinterpret_cast<const bi32x4*>(as + f * 2048 + rd0);
      af[f][1] = *reinterpret_cast<const bi32x4*>(as + f * 2048 + rd1);
    }
    const int dslot = slot + 2 >= 3 ? slot - 1 : slot + 2;
    float hi[4];                                                          // (segment 0: this block's second half; segment 1: not used)
    scale4(raw[1], hi);
    if constexpr (p == 0) {
      fetch_scales(t + 1);
      sw = swp[min(t + 1, nt - 1)];
      dma_a(t + 2, dslot, 0);
      dma_a(t + 2, dslot, 1);
    } else {
      dma_a(t + 2, dslot, 2);
      dma_a(t + 2, dslot, 3);
#pragma unroll
      for (int j = 0; j < 4; ++j) dma_w(t + 2, t & 1, j);
    }
    // vector work in the shadow of the operand reads: the last two results of the segment before, then the scales whose fragments
    // are through - the second half's in segment 0, the next block's first half's in segment 1
    __builtin_amdgcn_sched_barrier(0);
    finish(std::integral_constant<int, 1 - p>{});                        // (block 0, segment 0: the results are zero)
    if constexpr (p == 0) {
#pragma unroll
      for (int f = 0; f < 4; ++f) s[4 + f] = hi[f];
    } else {
      scale4(raw[0], s);
    }
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (p == 1) block_wait_vm<8>();
    WQ_BLOCK_BARRIER();
  };
  auto compute_segment = [&](auto PH) {
    constexpr int p = decltype(PH)::value;
#pragma unroll
    for (int i = 0; i < 16; ++i) {                                        // result i's fmas two matrix instructions behind it
      d[i % 3] = block_mfma<WF, AF>(wf[i & 3], af[i >> 2]);
      __builtin_amdgcn_sched_barrier(0);
      if (i >= 2) scaled(PH, i - 2);
      __builtin_amdgcn_sched_barrier(0);
    }
    WQ_BLOCK_BARRIER();
  };
  for (int t = 0; t < nt; ++t) {
    load_segment(std::integral_constant<int, 0>{}, t);
    compute_segment(std::integral_constant<int, 0>{});
    load_segment(std::integral_constant<int, 1>{}, t);
    compute_segment(std::integral_constant<int, 1>{});
    slot = slot == 2 ? 0 : slot + 1;
  }
  finish(std::integral_constant<int, 1>{});
  if (grp == 0) WQ_BLOCK_BARRIER();
  block_wait_vm<0>();                                                     // no copy may land in what the epilogue stages
  WQ_BLOCK_BARRIER();

  if (share.part >= 0) {                                                  // a slice: the whole tile, rows and columns beyond the matrix included
    float* const o = a.ws + share.part * (P::BM * P::BN) + (grp * 128 + r * 8) * P::BN + nq * 64 + q * 4;
#pragma unroll
    for (int f = 0; f < 8; ++f)
#pragma unroll
      for (int g = 0; g < 4; ++g) *reinterpret_cast<bf32x4*>(o + f * P::BN + g * 16) = acc[f][g];
    return;
  }
  // the tile leaves through LDS, whole rows per store: row m at 512 m, its 8-byte unit u (four n) at u ^ 4 (m / 8 mod 16) - the 64
  // lanes of a write, 16 rows 8 apart, then meet every bank twice, and 16-byte pieces stay whole
  const bool f16 = a.out_dtype == WQAA_F16;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int n = n0 + nq * 64 + g * 16 + q * 4;
    float bias[4] = {0.f, 0.f, 0.f, 0.f};
    if (a.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[e] = block_bias(a.bias, a.out_dtype, min(n + e, a.N - 1));
    }
#pragma unroll
    for (int f = 0; f < 8; ++f) {
      const int m = grp * 128 + r * 8 + f;
      uint16_t b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = acc[f][g][e] + bias[e];
        b[e] = f16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : block_bf16(v);
      }
      *reinterpret_cast<bu32x2*>(smem + m * 512 + ((nq * 16 + g * 4 + q) ^ (r << 2)) * 8) = bu32x2{b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16};
    }
  }
  __syncthreads();
  const int h = lane >> 5, c = lane & 31;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int m = wave * 32 + i * 2 + h, n = n0 + c * 8;
    const bi32x4 x = *reinterpret_cast<const bi32x4*>(smem + m * 512 + (c ^ ((m >> 3 & 15) << 1)) * 16);
    if (m0 + m >= a.M || n >= a.N) continue;
    uint16_t* o = reinterpret_cast<uint16_t*>(a.C) + (long)(m0 + m) * a.N + n;
    if (n + 8 <= a.N) {                                                   // (an odd N puts the piece on any boundary)
      __builtin_nontemporal_store(x, reinterpret_cast<bi32x4_at2*>(o));
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (n + e < a.N) o[e] = (uint16_t)((uint32_t)x[e >> 1] >> (16 * (e & 1)));
    }
  }
#endif
}

}  // namespace wqaa
