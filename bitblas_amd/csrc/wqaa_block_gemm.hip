// wqaa_block_gemm.hip - the block-scaled 8-bit product: which member a call takes, and its launch.
#include "wqaa_block_gemm_kernel.h"
#include "wqaa_block_pp_kernel.h"

namespace wqaa {

namespace {

struct Choice {
  int stream;            // > 0: the streaming member, which form of it (kStream, launch_pair)
  int bm;                // tile members: activation rows of a tile (256: the ping-pong member, whose tiles are 256 weight rows wide)
  int groups;            // tile member: groups of four waves in a workgroup (BlockTile::G)
  int tiles_m, tiles_n, whole, split, split_len;      // whole: tiles with a workgroup each; the others have `split`
  long tiles() const { return (long)tiles_m * tiles_n; }
  long grid() const { return whole + (tiles() - whole) * split; }
  int bn() const { return bm == 256 ? 256 : kBlock; }
};

Choice choose(const wqaa_block_desc& d, int m) {
  Choice c = {};
  const int kb = (d.K + kBlock - 1) / kBlock;
  auto stream = [&](int form, int rows, int nf) {
    c.stream = form;
    c.tiles_m = (m + rows - 1) / rows, c.tiles_n = (d.N + 16 * nf - 1) / (16 * nf), c.split = 1, c.split_len = kb;
    return c;
  };
  // few rows: W streams once.  Weight fragments of a wave: at more than 4 rows the activations' reads weigh as much as W's, and a wave that
  // takes 4 (2) fragments cuts them to a quarter (half) as long as the workgroups still fill the chip: 16 x 28672 x 8192 47 us with 4, 54
  // with 2, 57 with 1; 16 x 8192 x 28672 45 us with 2, 57 with 1, 68 with 4; 16 x 4096 x 4096 6.0 us with 1, 7.4 with 2; one row 39.5 us with 1,
  // 48 with 2 (28672 x 8192).  One fragment: 16 waves a block ahead where each has blocks to run through (one row, 28672 x 8192: 38.8 us
  // against 39.5 for 8 waves with 4 blocks at once; 4096 x 4096 5.0 against 4.7).
  if (m <= 16) return m > 4 && d.N >= 10240 ? stream(4, 16, 4) : m > 4 && d.N >= 7168 ? stream(3, 16, 2) : kb >= 64 ? stream(2, 16, 1) : stream(1, 16, 1);
  // 32 rows a workgroup, more of them along y: small products are through before tiles and their partial sums would be.  One fragment
  // while that is about a workgroup per CU (77 x 1001 x 1040 3.2 us against 3.8 with two and 8.4 for tiles; 128 x 1024 x 4096 7.7, 9.7 and
  // 11.1), else two while they take a round of the chip, or up to four on short K (64 x 4096 x 4096 10.0 us against 13.7 for tiles, 64 x 6144 x 4096
  // 17.2 against 13.4; 256 x 2048 x 2048 10.0 against 12.0; 333 x 2048 x 1024, three rounds, 8.6 against 11.1;
  // 600 x 1024 x 2048 13.6 against 12.6).  Up to 32 rows there is nothing W could be shared with: 24 x 6144 x 4096 9.5 us
  // with two, 12.0 with one; 32 x 11008 x 4096 14.6 us with four, 17.2 with two.  But where the 64-row tiles are a round of the chip or nearly,
  // their copies through LDS ask for more of W at once: 32 x 20480 x 8192, 160 tiles, 43 us against 53 with four fragments; 24 x 28672 x 8192 50
  // against 55; 20 x 50000 x 1024 14 against 23 (on short K two fragments stream: 24 x 22000 x 768 8.1 us, 9.7 in tiles).
  const long chunks = (m + 31) / 32, one = chunks * ((d.N + 15) / 16), two = chunks * ((d.N + 31) / 32), rounds2 = (two + 255) / 256;
  if (one <= 288 && (m <= 32 || kb <= 48)) return stream(5, 32, 1);
  const bool thin = m <= 32 && d.N < 160 * kBlock;
  if (thin && d.N >= 10240) return stream(7, 32, 4);
  if (thin || (rounds2 <= 4 && rounds2 * kb <= 32)) return stream(6, 32, 2);
  auto tiles_of = [&](int bm, int bn) {
    c.bm = bm, c.tiles_m = (m + bm - 1) / bm, c.tiles_n = (d.N + bn - 1) / bn;
    c.split = 1, c.split_len = kb, c.whole = (int)c.tiles();
    return c.tiles();
  };
  auto slices = [&](long whole, long split) {    // the tiles behind the first `whole` of them in K slices
    c.split_len = (int)((kb + split - 1) / split);
    c.split = (kb + c.split_len - 1) / c.split_len;
    if (c.split > 1) c.whole = (int)whole;
  };
  // many rows: the ping-pong member, a 256 x 256 tile per CU at a time.  The tiles of a last round that is not full (or of the only one) may
  // leave in K slices, so that it takes a half to a quarter of a round: saves 1.5 us for every k-block it is shorter, costs 0.09 us for
  // every partial tile, to memory and back, and 6 us for the launch that adds them: 4096 x 4352 x 4096, 272 tiles, 112 us whole, 98 with the last 16 in 2
  // slices, 91 in 4, 94 in 7; 4096 x 5120 x 5120, 320 tiles, 141, 136 and 126 in 4; 3000 x 8192 x 8192, 384 tiles, 236 and 223 in 2; 4096 x
  // 9472 x 2048, 592 tiles, 115, 117 in 2, 134 in 4; 512 x 8192 x 28672, 64 tiles in 4, 123, in 128-row tiles 154
  const long t128 = tiles_of(128, kBlock);
  const long big = tiles_of(256, 256), rounds = (big + 255) / 256, rest = big % 256;
  if (t128 > 0x3fffffffl) return c;               // (block_gemm_check refuses it)
  long split = 1, saved = 0;                      // units of 0.1 us
  for (long z = 2; z <= 4 && rest * z <= 256; ++z) {
    const long gain = 15 * (kb - (kb + z - 1) / z) - rest * z * 9 / 10 - 60;
    if (rest > 0 && gain > saved) split = z, saved = gain;
  }
  // taken where the tile members' rounds would take longer: a k-block of a round of 128-row tiles (two a CU) takes 1.13 us, of up to one a CU
  // 0.62: 1100 x 8192 x 8192, 160 tiles, 105 us, 130 in 576 tiles of 128 rows; 300 x 8192 x 28672, 64 tiles in 4 slices, 116, 139 in 192;
  // 2048 x 28672 x 8192, 896 tiles, 435, 517.  1024 x 8192 x 8192 would take 77 in 2 slices by that reckoning: 512 of 128 rows, 73
  const long tile_time = kb * (t128 > 256 ? 113 * ((t128 + 511) / 512) : t128 >= 192 ? 62 : 62 * t128 / 192) / 10;
  if (m > 128 && 15 * kb * rounds - saved < tile_time) {
    if (split > 1) slices(big - rest, split);
    return c;
  }
  // tiles of 128 rows where they are a tile per CU or nearly, or more than two of 64 rows per CU: 512 x 8192 x 8192, 256 of them, 43 us
  // against 50 for 512 of 64 rows; 128 x 28672 x 8192, 224 of them, 65 against 70; 700 x 8192 x 4096, 704 of 64 rows, 36 against 41
  (void)tiles_of(128, kBlock);
  const bool one_each = t128 >= 192 && t128 <= 256;
  const long t64 = (long)((m + 63) / 64) * c.tiles_n;
  // 64 rows, two of them a CU, and little more than a round: that in 4 slices, which fill the chip once up to 64 tiles (of K = 4096, in slices against
  // tiles of 128 rows: 384 x 11008, 516 tiles, 33.4 us against 37.6; 384 x 11520, 540, 33.7 and 38.0; 1000 x 4480, 560, 33.6 and 35.3; 384 x 12032,
  // 564, 34.1 and 38.2; 640 x 7296, 570, 35.2 and 38.5; 384 x 12288, 576, 34.3 and 34.7; beyond: 384 x 12800, 600, 38.7 and 38.4; 640 x 7680, 600, 39.4
  // and 38.6; 384 x 13568, 636, 40.0 and 38.7; 640 x 8192, 640, 39.7 and 34.2.  From about K = 8192 on the 256-row tiles above take these)
  if (m > 64 && t64 > 512 && t64 <= 512 + 64 && kb >= 32) {
    (void)tiles_of(64, kBlock);
    c.groups = 1;
    slices(512, 4);
    return c;
  }
  if (m > 64 && (one_each || t64 > 512)) {
    c.groups = one_each ? 2 : 1;
    return c;
  }
  (void)tiles_of(64, kBlock);
  // 64 rows: up to a tile per CU two groups of waves on it (512 x 4096 x 4096, 256 tiles, 17.6 us against 19.8; 256 x 8192 x 8192 29 against 32).
  // Fewer tiles than that: K in slices that fill the chip once, of at least 4 blocks, at most 8 - the partial tiles cost their way to memory
  // and back: 128 x 4096 x 4096, 64 tiles, 4 slices 13.8 us, 2 slices 14.4, 8 over 16; 128 x 8192 x 8192, 128 tiles, 2 slices of two groups
  // 19.7 us, 4 slices of one 21.2; 512 x 1024 x 4096, 64 tiles, 4 slices 13.8 us, none 20
  c.groups = t64 >= 128 && t64 <= 256 ? 2 : 1;
  if (t64 < 160) {
    long z = c.groups == 2 ? 2 : 256 / t64;
    if (z > 8) z = 8;
    if (z > kb / 4) z = kb / 4;
    if (z > 1) slices(0, z);
  }
  return c;
}

template <class P>
void tile_attr() {
  (void)hipFuncSetAttribute(reinterpret_cast<const void*>(wq_block_tile_kernel<P>), hipFuncAttributeMaxDynamicSharedMemorySize, P::LDS);
}
template <class P>
void tile_go(const Choice& c, const BlockGemmArgs& a, hipStream_t s) {
  wq_block_tile_kernel<P><<<dim3((unsigned)c.grid()), dim3(P::THREADS), P::LDS, s>>>(a);
}
template <int WF, int AF, bool TAIL>
void pp_attr() {
  (void)hipFuncSetAttribute(reinterpret_cast<const void*>(wq_block_pp_kernel<WF, AF, TAIL>), hipFuncAttributeMaxDynamicSharedMemorySize, BlockPP::LDS);
}
template <int WF, int AF>
void init_pair() {
  pp_attr<WF, AF, false>();
  pp_attr<WF, AF, true>();
  tile_attr<BlockTile<WF, AF, 64, 3, 1, false>>();
  tile_attr<BlockTile<WF, AF, 64, 3, 1, true>>();
  tile_attr<BlockTile<WF, AF, 64, 3, 2, false>>();
  tile_attr<BlockTile<WF, AF, 64, 3, 2, true>>();
  tile_attr<BlockTile<WF, AF, 128, 2, 1, false>>();
  tile_attr<BlockTile<WF, AF, 128, 2, 1, true>>();
  tile_attr<BlockTile<WF, AF, 128, 2, 2, false>>();
  tile_attr<BlockTile<WF, AF, 128, 2, 2, true>>();
}
struct StreamForm {
  int waves, nf;
};
constexpr StreamForm kStream[] = {{0, 0}, {8, 1}, {16, 1}, {16, 2}, {8, 4}, {8, 1}, {8, 2}, {8, 4}};
template <int WF, int AF>
void launch_pair(const Choice& c, const BlockGemmArgs& a, hipStream_t s) {
  const bool tail = a.K % kBlock != 0;
  const dim3 g(a.tiles_n, a.tiles_m), t(kStream[c.stream].waves * 64);
  if (c.stream == 1) wq_block_stream_kernel<WF, AF, 8, 4, 1, 1, false><<<g, t, 0, s>>>(a);
  else if (c.stream == 2) wq_block_stream_kernel<WF, AF, 16, 1, 1, 1, true><<<g, t, 0, s>>>(a);
  else if (c.stream == 3) wq_block_stream_kernel<WF, AF, 16, 1, 2, 1, true><<<g, t, 0, s>>>(a);
  else if (c.stream == 4) wq_block_stream_kernel<WF, AF, 8, 1, 4, 1, true><<<g, t, 0, s>>>(a);
  else if (c.stream == 5) wq_block_stream_kernel<WF, AF, 8, 1, 1, 2, true><<<g, t, 0, s>>>(a);
  else if (c.stream == 6) wq_block_stream_kernel<WF, AF, 8, 1, 2, 2, true><<<g, t, 0, s>>>(a);
  else if (c.stream == 7) wq_block_stream_kernel<WF, AF, 8, 1, 4, 2, true><<<g, t, 0, s>>>(a);
  else if (c.bm == 64 && c.groups == 2) tail ? tile_go<BlockTile<WF, AF, 64, 3, 2, true>>(c, a, s) : tile_go<BlockTile<WF, AF, 64, 3, 2, false>>(c, a, s);
  else if (c.bm == 64) tail ? tile_go<BlockTile<WF, AF, 64, 3, 1, true>>(c, a, s) : tile_go<BlockTile<WF, AF, 64, 3, 1, false>>(c, a, s);
  else if (c.bm == 128 && c.groups == 2) tail ? tile_go<BlockTile<WF, AF, 128, 2, 2, true>>(c, a, s) : tile_go<BlockTile<WF, AF, 128, 2, 2, false>>(c, a, s);
  else if (c.bm == 128) tail ? tile_go<BlockTile<WF, AF, 128, 2, 1, true>>(c, a, s) : tile_go<BlockTile<WF, AF, 128, 2, 1, false>>(c, a, s);
  else if (tail) wq_block_pp_kernel<WF, AF, true><<<dim3((unsigned)c.grid()), dim3(BlockPP::THREADS), BlockPP::LDS, s>>>(a);
  else wq_block_pp_kernel<WF, AF, false><<<dim3((unsigned)c.grid()), dim3(BlockPP::THREADS), BlockPP::LDS, s>>>(a);
}

}  // namespace

void block_init() {
  init_pair<0, 0>();
  init_pair<0, 1>();
  init_pair<1, 0>();
  init_pair<1, 1>();
}

int block_gemm_check(const wqaa_block_desc& d, int m) {
  constexpr long kThreads = 0xffffffffl;          // of a launch
  bool ok = m < (1 << 29) && d.N <= 0x7fffffff - 256;                    // (row scales of a block: 31 bits of bytes)
  if (ok) {
    const Choice c = choose(d, m);
    const long wide = c.stream ? c.tiles_n : c.grid();
    ok = c.tiles() <= 0x3fffffffl && wide * (c.stream ? kStream[c.stream].waves * 64 : c.bm == 256 ? BlockPP::THREADS : c.groups * 256) <= kThreads;
  }
  if (ok) return WQAA_OK;
  set_error(WQAA_ERR_UNSUPPORTED, "block_matmul: m=%d N=%d is too large", m, d.N);
  return WQAA_ERR_UNSUPPORTED;
}

size_t block_gemm_workspace_bytes(const wqaa_block_desc& d, int m) {
  const Choice c = choose(d, m);
  return c.split > 1 ? (size_t)(c.tiles() - c.whole) * c.split * c.bm * c.bn() * 4 : 0;
}

int block_gemm_plan(const wqaa_block_desc& d, int m, wqaa_plan* plan) {
  if (!plan) return WQAA_OK;
  const Choice c = choose(d, m);
  memset(plan, 0, sizeof(*plan));
  plan->kernel_family = 2;
  plan->block_m = c.stream ? (c.stream <= 4 ? 16 : 32) : c.bm;
  plan->block_n = c.stream ? kStream[c.stream].nf * 16 : c.bm == 256 ? 256 : 128;
  plan->block_k = kBlock;
  plan->threads = c.stream ? kStream[c.stream].waves * 64 : c.bm == 256 ? BlockPP::THREADS : c.groups * 256;
  plan->grid = (int)c.grid();
  plan->split_k = c.split;
  snprintf(plan->name, sizeof(plan->name), "block_matmul_m%dn%dk%d_%sx%s_%s%dx%d%s", m, d.N, d.K, short_dtype(d.a_dtype), short_dtype(d.w_dtype),
           c.stream ? "stream" : c.bm == 256 ? "pp" : "tile", plan->block_m, plan->block_n, c.split > 1 ? "_split" : "");
  return WQAA_OK;
}

int block_gemm_launch(const wqaa_block_desc& d, const void* A, const void* W, const float* sa, int64_t sa_ld, const float* sw, const void* bias,
                      void* C, int m, void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  const Choice c = choose(d, m);
  const uint64_t need = block_gemm_workspace_bytes(d, m);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))) {
    set_error(WQAA_ERR_BAD_DESC, "block_matmul: m=%d needs %llu bytes of 16-byte aligned workspace", m, (unsigned long long)need);
    return WQAA_ERR_BAD_DESC;
  }
  BlockGemmArgs a = {};
  a.A = reinterpret_cast<const unsigned char*>(A), a.W = reinterpret_cast<const unsigned char*>(W);
  a.sa = sa, a.sw = sw, a.sa_ld = sa_ld;
  a.bias = d.with_bias ? bias : nullptr;
  a.C = C, a.ws = reinterpret_cast<float*>(workspace);
  a.M = m, a.N = d.N, a.K = d.K, a.KB = (d.K + kBlock - 1) / kBlock;
  a.out_dtype = d.out_dtype;
  a.tiles_m = c.tiles_m, a.tiles_n = c.tiles_n, a.whole = c.whole, a.split = c.split, a.split_len = c.split_len;
  a.group_m = c.tiles_m < 8 ? c.tiles_m : 8;
  const int wf = d.w_dtype == WQAA_E5M2, af = d.a_dtype == WQAA_E5M2;
  if (wf == 0 && af == 0) launch_pair<0, 0>(c, a, stream);
  else if (wf == 0) launch_pair<0, 1>(c, a, stream);
  else if (af == 0) launch_pair<1, 0>(c, a, stream);
  else launch_pair<1, 1>(c, a, stream);
  if (c.split > 1) {
    const dim3 g((unsigned)((c.tiles() - c.whole) * (c.bm * c.bn() / 1024)));
    if (c.bm == 256) wq_block_reduce_kernel<256><<<g, dim3(256), 0, stream>>>(a, c.bm);
    else wq_block_reduce_kernel<kBlock><<<g, dim3(256), 0, stream>>>(a, c.bm);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error(WQAA_ERR_LAUNCH, "block_matmul: %s", hipGetErrorString(e));
    return WQAA_ERR_LAUNCH;
  }
  return WQAA_OK;
}

}  // namespace wqaa
