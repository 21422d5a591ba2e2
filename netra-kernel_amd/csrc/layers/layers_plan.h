// Which kernel and which grid a call of libnetra_layers.so takes: rules on sizes, types and
// alignment, in plain integers, so that they are also tested on the host.
#pragma once
#include <stdint.h>

namespace nkplan {

// Sizes up to 2^21 keep every grid dimension, tile count and scale index inside its type.
constexpr uint32_t kMaxSize = 1u << 21;

inline uint32_t up(uint32_t v, uint32_t m) { return (v + m - 1u) / m * m; }
inline uint32_t blocks(uint32_t v) { return (v + 127u) / 128u; }

// How a product runs: the streaming kernel, quantising on the way (kFused) or not
// (kStream), with p tiles of 16 columns and q of 16 rows per workgroup, or tiles of p x q
// with splits of the contraction.
enum Form { kFused, kStream, kTiles };
struct ProductPlan {
  Form form;
  uint32_t p, q, splits, split_blocks;
};

// Tiles: time = rounds of workgroups over the 256 CUs x (steps x the step's time + what a
// workgroup takes besides), the step's time hardly depending on how many CUs work (us a step:
// 256x256 1.75, 256x128 1.18, 128x128 0.78, 128x64 0.58, 64x64 0.35, or 0.62 where two workgroups
// share a CU). Splits add a launch and the partial sums' way out and in. Measured as whole calls,
// best and next: T 333, N 2048, K 1024 64x64 10.0 us, 128x64 10.7, 128x128 11.0; T 700, N 2048, K
// 2048 128x64 13.8, 64x64 15.4; T 1500, N 1500, K 1500 128x128 17.3, 64x64 20.4; T 1500, N 4096, K
// 1024 256x128 16.4, 128x128 20.2; T 8192, N 512, K 4096 128x128 40.7, 256x128 in two splits 48.5;
// T 3000, N 6000, K 3000 256x256 81.3, 256x128 83.7, 128x128 92.5; T 4096, N 4096, K 2048 256x256
// 39.8, 256x128 45.9; T 200, N 500, K 8000 64x64 in eight splits 14.6, in two 19.5. The model misses
// by 7% at T 128, N 8192, K 8192: 128x64 in two splits 25.1, 64x64 26.8.
inline ProductPlan product_tiles(uint32_t rows, uint32_t ni, uint32_t nc) {
  struct Shape {
    uint32_t p, q;
    double step_us, group_us;
  };
  static const Shape shapes[] = {
      {256, 256, 1.75, 3.0}, {256, 128, 1.18, 2.0}, {128, 128, 0.78, 1.5}, {128, 64, 0.58, 1.2}, {64, 64, 0.35, 1.0}};
  const uint32_t kb = blocks(nc);
  ProductPlan best{kTiles, 256, 256, 1, kb};
  double best_us = 1e30;
  for (const Shape& s : shapes) {
    const uint64_t tiles = static_cast<uint64_t>((ni + s.p - 1u) / s.p) * ((rows + s.q - 1u) / s.q);
    for (uint32_t splits = 1; splits <= 8u && splits <= (kb + 3u) / 4u; splits *= 2u) {
      if (splits > 1u && tiles * splits > 512u) break;
      const uint32_t each = (kb + splits - 1u) / splits, n = (kb + each - 1u) / each;
      const bool pairs = s.p * s.q == 64u * 64u && tiles * n > 256u;
      const double rounds = static_cast<double>(pairs ? (tiles * n + 511u) / 512u : (tiles * n + 255u) / 256u);
      double us = rounds * (each * (pairs ? 0.62 : s.step_us) + s.group_us);
      if (n > 1u) us += 3.0 + static_cast<double>(rows) * ni * (8.0 * n) / 5e6;  // 5 TB/s
      if (us < best_us) {
        best_us = us;
        best = {kTiles, s.p, s.q, n, each};
      }
    }
  }
  return best;
}

inline ProductPlan product_plan(uint32_t rows, uint32_t ni, uint32_t nc, bool bf16) {
  if (rows > 64u) return product_tiles(rows, ni, nc);
  // Two tiles of columns per workgroup: fused they halve the quantisation (T 16, N 8192, K 8192:
  // 21.7 us -> 16.2; of more than two tiles of rows they do not fit the registers), else the
  // activations are read half as often (T 64, N 8192, K 8192: 24.1 us -> 20.3).
  const uint32_t pt = (ni + 15u) / 16u, q = (rows + 15u) / 16u, kb = blocks(nc), wide = pt >= 512u ? 2u : 1u;
  const uint32_t p = q <= 2u ? wide : 1u;  // of a fused workgroup
  // Quantising on the way saves a launch (10.7 us -> 6.7 at one row) and costs every
  // workgroup the quantisation of its waves' blocks. One tile of rows always quantises on the
  // way: at worst it costs 3% (T 16, N 28672, K 8192: 50.5 us, with the launch 49.0), few rows
  // gain most (T 1: 40.2 against 48.6). Two do up to seven tile-blocks per wave and CU (T 32, N
  // 8192, K 8192, sixteen: 23.5 against 17.5). With three or four a CU holds one workgroup at a
  // time, and what pays falls with the rounds that the columns take (us, fused / with the launch):
  //   one round      T 48, K 1152  9.1 / 10.3    K 2048 11.0 / 10.2    T 64, K 2048 12.1 / 10.4
  //   N 8192, two    T 64, K 512  10.1 / 10.4    T 48, K 768 11.8 / 10.5    K 2048 20.0 / 10.4
  //   N 12288        T 64, K 128  10.0 / 10.5    K 256  11.4 / 10.5
  //   N 16384        T 48, K 128  11.8 / 10.4
  const uint32_t rounds = ((pt + p - 1u) / p + 255u) / 256u, each = q * ((kb + 7u) / 8u);
  const uint32_t all = q * (kb < 8u ? kb : (kb + 7u) / 8u * 8u);  // tile-blocks that a workgroup quantises
  const bool few = q <= 2u ? static_cast<uint64_t>(rounds) * each < 8u
                           : bf16 && all <= (rounds == 1u ? 48u : rounds == 2u ? 16u : rounds == 3u ? 4u : 0u);
  if (q == 1u || few) return {kFused, p, q <= 2u ? q : 4u, 1, 0};
  return {kStream, wide, 4, 1, 0};
}

// The same for rows that are quantised already: nothing to do on the way.
inline ProductPlan codes_plan(uint32_t rows, uint32_t ni, uint32_t nc) {
  if (rows > 64u) return product_tiles(rows, ni, nc);
  return {kStream, (ni + 15u) / 16u >= 512u ? 2u : 1u, 4, 1, 0};
}

// Tile and split of the weight gradient, chosen as product_tiles' (steps of 64 tokens: 256x256
// 1.55 us, 128x256 0.93, 128x128 0.48, one workgroup per CU each). As whole calls, best and
// next: T 333, N 1024, K 2048 128x128 8.3 us, 128x256 11.8; T 4096, N 4096, K 2048 128x256 64,
// 128x128 82; T 4096, N 1024, K 1024 128x128 in four splits 21.3, in two 23.9; T 8192, N 4096,
// K 4096 256x256 216, 128x256 249.
struct OuterPlan {
  uint32_t p, q;  // columns of x and of dy per workgroup
  uint32_t splits, split_rows;
};
inline OuterPlan outer_plan(uint32_t rows, uint32_t n, uint32_t k) {
  struct Shape {
    uint32_t p, q;
    double step_us;
  };
  static const Shape shapes[] = {{256, 256, 1.55}, {128, 256, 0.93}, {128, 128, 0.48}};
  const uint32_t steps = (rows + 63u) / 64u;
  OuterPlan best{256, 256, 1, up(rows, 64u)};
  double best_us = 1e30;
  for (const Shape& s : shapes) {
    const uint64_t tiles = static_cast<uint64_t>((k + s.p - 1u) / s.p) * ((n + s.q - 1u) / s.q);
    for (uint32_t splits = 1; splits <= 16u && splits <= (steps + 3u) / 4u; splits *= 2u) {
      if (splits > 1u && tiles * splits > 512u) break;
      const uint32_t each = (steps + splits - 1u) / splits, count = (steps + each - 1u) / each;
      double us = static_cast<double>((tiles * count + 255u) / 256u) * each * s.step_us;
      if (count > 1u) us += 3.0 + static_cast<double>(n) * k * 4.0 * (2.0 * count + 1.0) / 6e6;  // 6 TB/s
      if (us < best_us) {
        best_us = us;
        best = {s.p, s.q, count, each * 64u};
      }
    }
  }
  return best;
}

// Workgroups that copy an operand of the weight gradient [rows, pitch] to the workspace: a multiple of
// the 512-column parts of a row, four rows at a time, 2^18 at most (they loop over the rows).
inline uint32_t copy_groups(uint32_t rows, uint32_t pitch) {
  const uint32_t across = (pitch + 511u) / 512u, most = across <= 64u ? 4096u : (1u << 18) / across;
  const uint32_t down = (rows + 3u) / 4u;
  return across * (down < most ? down : most);
}
// Workgroups that quantise [rows, n] in a launch with the copies.
inline uint32_t quant_groups(uint32_t rows, uint32_t n) { return (rows + 15u) / 16u * ((blocks(n) + 3u) / 4u); }
// Workgroups of a product [rows, ni] in tiles and of a weight gradient: a multiple of the eight XCDs.
inline uint64_t tile_groups(uint64_t a, uint32_t p, uint64_t b, uint32_t q, uint32_t splits) {
  return ((a + p - 1u) / p * ((b + q - 1u) / q) * splits + 7u) / 8u * 8u;
}
// A launch's threads in one dimension have 32 bits.
inline bool launchable(uint64_t groups, uint32_t threads) { return groups * threads < (1ull << 32); }

// Whether a backward pass runs both products in one launch, dx in tiles of 64 x 64 then: passes of
// small tiles (T 333, N 1024, K 2048 13.3 us, in two 16.9; T 3584, N 360, K 189 16.3, 20.7; T 1200,
// N 1000, K 1000 18.3, 24.5; T 3000, N 500, K 500 21.3, 24.1); with larger tiles most lose by it (T
// 5000, N 600, K 1000 36.6, 33.5).
inline bool backward_in_one(const ProductPlan& product, const OuterPlan& outer) {
  return product.form == kTiles && product.p * product.q <= 128u * 64u && product.splits == 1u &&
         outer.p * outer.q == 128u * 128u;
}

// Counting is shared out over workgroups of 256 threads where one would take longer
// than a second launch; each counts `each` tokens, one a thread while `most` workgroups reach (the
// loss kernel's workgroups all add up all parts: few of them, with more threads).
struct CountPlan {
  uint32_t groups, each;
};
inline CountPlan count_plan(uint32_t tokens, uint32_t few, uint32_t most) {
  if (tokens <= few) return {0, tokens};
  const uint32_t groups = (tokens - 1u) / 256u + 1u;
  CountPlan plan{groups > most ? most : groups, 0};
  plan.each = (tokens + plan.groups - 1u) / plan.groups;
  return plan;
}
// Tokens one workgroup counts (1024 of 9 ids: 7.3 us, in two launches 9.5; 2048: 10.0, 9.5; 3500:
// 14.2, 9.6).
constexpr uint32_t kFewCounts = 2048;
constexpr uint32_t kBalanceGrid = 256;
// One workgroup takes 32768 logits through the loss, 256 tokens at most (128 x 256: 11.7 us, shared
// out 13.6; 256 x 16: 9.9, 13.6; 512 x 16: 13.3, 13.7; 64 x 512: 11.2, 13.6; 64 x 1024: 16.0, 13.6).
// More parts than 64 cost their summing up what they gain (32768 x 256 24.1 us with 128, 24.7 with
// 64; x 500 33.8, 32.3; with 32 27.7, 32.9).
inline CountPlan balance_plan(uint32_t tokens, uint32_t experts) {
  const uint32_t few = 32768u / (experts ? experts : 1u);
  return count_plan(tokens, few < 256u ? few : 256u, 64u);
}

// Bytes that the cache behind the L2s holds: what moves more than these finds nothing of it there.
constexpr uint64_t kInfinityCache = 256ull << 20;
constexpr uint64_t kL2 = 4ull << 20;  // of one of the eight XCDs

// Norms: waves a row and eight columns a lane so many times, rows a workgroup takes at once, and
// workgroups (they loop over the rows).
struct NormPlan {
  uint32_t waves, chunks, rows, threads, groups;
};
inline NormPlan norm_shape(uint32_t cols) {
  if (cols <= 512u) return {1, 1, 4, 256, 0};
  if (cols <= 1024u) return {1, 2, 4, 256, 0};
  const uint32_t waves = cols <= 2048u ? 4u : cols <= 4096u ? 8u : 16u;
  return {waves, cols <= 8192u ? 1u : 2u, 1, 64u * waves, 0};
}
inline NormPlan norm_plan(uint32_t rows, uint32_t cols) {
  NormPlan p = norm_shape(cols);
  const uint32_t groups = (rows + p.rows - 1u) / p.rows, most = 8192u * 64u / p.threads;
  p.groups = groups < most ? groups : most;
  return p;
}
// Each workgroup leaves a partial sum of dw.
inline NormPlan norm_gradients_plan(uint32_t rows, uint32_t cols) {
  NormPlan p = norm_shape(cols);
  const uint32_t groups = (rows + p.rows - 1u) / p.rows, most = p.waves == 16u ? 256u : 512u;
  p.groups = groups < most ? groups : most;
  return p;
}

// Tokens of the routing: with four a workgroup the launch's threads still fit their 32 bits.
constexpr uint32_t kMaxRouted = 1u << 25;
// Workgroups of the routing's gradient: each takes so many tokens at a time and loops past a whole chip's worth of waves.
inline uint32_t select_groups(uint32_t tokens, uint32_t at_once) {
  const uint32_t groups = (tokens - 1u) / at_once + 1u;
  return groups < 4096u ? groups : 4096u;
}

// Adapters: 16-rank parts as the kernels have them; tokens a tile; tiles that a batch has at most (one
// short one for each adapter in use and for the tokens without); splits of k's 128-blocks where the tiles are few, and
// groups of 256 columns that a workgroup of the second product takes.
inline uint32_t adapter_ranks(uint32_t rank) { return rank <= 16u ? 1u : rank <= 32u ? 2u : rank <= 64u ? 4u : 8u; }
// (Tiles of 32 share what is read of A and B and fill fewer CUs: us, of 16 / of 32,
//   K 4096   T 4096, N 4096, rank 64  40 / 48    T 8192, N 8192, rank 16  79 / 85, 64  111 / 104, 128  152 / 132
//   K 3008   T 3333, N 5440, rank 48  36 / 45    T 8192, N 4096, 60 adapters of rank 64  110 / 90
// The plan does not know the rank.)
inline uint32_t adapter_tile(uint32_t tokens, uint32_t adapters) {
  return tokens >= 8192u && tokens / 64u >= adapters ? 32u : 16u;
}
inline uint32_t adapter_tiles(uint32_t tokens, uint32_t adapters) {
  const uint32_t tile = adapter_tile(tokens, adapters), parts = adapters + 1u;
  return (tokens + tile - 1u) / tile + (parts < tokens ? parts : tokens) - 1u;
}
struct AdapterPlan {
  uint32_t tiles, splits, split_blocks, wide;
  bool fused;
};
inline AdapterPlan adapter_plan(uint32_t tokens, uint32_t adapters, uint32_t rank, uint32_t n, uint32_t k) {
  AdapterPlan p{adapter_tiles(tokens, adapters), 1, blocks(k), 1, false};
  // One launch, in which each workgroup of 512 columns works u out for itself, where the workgroups find a CU
  // each and A is short (us, in one launch / in two; a launch takes the host 3.5 besides):
  //   A  64 KB  T 64, 32 adapters, N 2048: 144 workgroups 4.7 / 6.7    T 1000, 30, 2048: 372, 11.3 / 8.3
  //   A 128 KB  T 16, 16, N 4096: 136, 5.6 / 7.1    T 64, 16, 4096: 160, 5.6 / 7.2    T 256, 32, 4096: 384, 11.7 / 8.2
  //   A 256 KB  T 64, 16, N 4096: 160, 9.2 / 8.2
  const uint64_t a_bytes = 32ull * adapter_ranks(rank) * up(k, 128u);  // of one adapter
  if (adapter_tile(tokens, adapters) == 16u && a_bytes <= 131072u &&
      static_cast<uint64_t>(p.tiles) * ((n + 511u) / 512u) <= 256u) {
    p.fused = true;
    p.split_blocks = blocks(k);
    return p;
  }
  // A workgroup reads and packs its tile's u before its first columns: up to eight groups of columns share that, the fewer
  // the less there is of u, as more workgroups end more evenly. us at N 4096, K 4096, T 8192, of 1024 / 2048 / 4096 workgroups
  // or more: rank 16 56 / 53 / 52, 32 61 / 57 / 60, 64 74 / 74 / 82, 128 94 / 97 / 112.
  const uint64_t groups = static_cast<uint64_t>(p.tiles) * ((n + 255u) / 256u);
  const uint32_t ranks = adapter_ranks(rank), least = ranks <= 4u ? 4096u / ranks : 1024u;
  while (p.wide < 8u && groups / (2u * p.wide) >= least) p.wide *= 2u;
  while (p.splits < 16u && p.tiles * p.splits * 2u <= 512u && blocks(k) / (p.splits * 2u) >= 8u) p.splits *= 2u;
  p.split_blocks = (blocks(k) + p.splits - 1u) / p.splits;
  p.splits = (blocks(k) + p.split_blocks - 1u) / p.split_blocks;
  return p;
}
// Whether y and out go past the caches: together they are more than the one behind the L2s holds, or than all L2s hold while
// B would fill one (4 MB). us without / with, of 8 adapters and K 4096:
//   268 MB  T 8192, N 8192, rank 16  82 / 81    32 87 / 80    64 103 / 92    128 130 / 122
//   134 MB  T 4096, N 8192: B of 2 MB 42.7 / 43.6    4 50.1 / 47.5    8 66.0 / 59.2    16 85.8 / 84.4
//           T 8192, N 4096: B of 1 MB 51.3 / 55.6    2 57.3 / 56.5    4 72.9 / 66.7     8 94.0 / 90.7
inline bool adapter_once(uint32_t tokens, uint32_t adapters, uint32_t rank, uint32_t n) {
  const uint64_t moved = 4ull * tokens * n, b = 32ull * adapter_ranks(rank) * n * adapters;
  return moved > kInfinityCache || (moved > 8u * kL2 && b >= kL2);
}

}  // namespace nkplan
