// ipc_token_plan.h - how a softmax call over tokens runs, by its sizes and type: the terms of its operands, its
// pieces and tiles, what lies where in the workspace.  Host code that needs no HIP (of the package's
// headers the DT_ and ACT_ codes alone), so that a test can look at every plan.
#pragma once

#include <algorithm>

namespace ipc {

// Tiles of the logits' products (TOKEN_STATS, _KEEP, _ERROR): rows (of W) and columns of a workgroup, and the rows of a wave, whose
// largest values and sums are kept (unit; ways: terms of f(X), side by side in a tile; with three
// TILE_128_64 and TILE_64 alone, each 96 columns wide).
enum { TILE_256 = 0, TILE_128 = 1, TILE_128_64 = 2, TILE_64 = 3 };
inline int token_unit(int tile, int ways) {
  return tile == TILE_256 ? 128 : tile == TILE_128 ? 64 : tile == TILE_128_64 ? (ways == 2 ? 32 : 64) : 32;
}

constexpr int TOKEN_ONE_ROWS = 128;  // of TOKEN_ONE, at most
inline int token_fix_rows(int D, bool vec) { return vec ? (D + 15) / 16 : (D + 3) / 4; }
inline long long token_tail_tiles(int V, int D, int B) { return (D + 63LL) / 64 * ((B + 63LL) / 64 + (V + 63LL) / 64); }

constexpr long long TOKEN_PIECE_BYTES = 1LL << 30;  // of a piece's errors, and of its rows of W where those are laid out
constexpr long long TOKEN_OPERAND = (1LL << 31) - 1;                  // of an operand of a product with all its terms
// 16-bit updates of at most so many errors and multiplications are `fine`.
constexpr long long TOKEN_FINE_ERRORS = 1LL << 23, TOKEN_FINE_WORK = 1LL << 31;
// And in bf16 those of few words: there probabilities are not small, and rounding them to 8 bits leaves the
// next loss off in its fifth digit.  The next loss's error and us, one term / fine, 4000 features, 1024 samples: 2048 words
// 1.9e-5 / 7.6e-7, 159 / 235; 4096 8.5e-6 / 3.3e-7, 194 / 423; 8192 5.8e-6 / 8.4e-7, 301 / 798.  4000 samples: 512 words
// 2.3e-5 / 1.4e-6, 288 / 400; 2048 1.0e-5 / 1.5e-6, 436 / 977.  From 2048 words on, or with more errors, one term keeps the loss
// to five digits and a fine update costs twice the time.  (600 x 8000 x 1000 and 1201 x 4040 x 2744 with one: 5e-5 and
// 4e-5.)  In fp16 one term leaves 3.4e-6 at 512 words, 2.0e-6 at 2048.
constexpr int TOKEN_FINE_WORDS = 2048;

// A column's errors in one workgroup, up to so many; of more, one for each 2048.
constexpr int TOKEN_ERROR_RUN = 8192;
inline long long token_error_blocks(int Bk, int Vp) { return (long long)Bk * (Vp <= TOKEN_ERROR_RUN ? 1 : (Vp + 2047) / 2048); }
// Workgroups of the launch that makes the targets' errors good, for G and for W.
inline long long token_rest_blocks(int D, int B) { return (D + 63LL) / 64 * ((B + 63LL) / 64); }
inline long long token_hot_blocks(int Dp, int B) { return (long long)B * ((Dp + 255) / 256); }
constexpr long long TOKEN_LAUNCH = (1LL << 32) - 1;  // work-items of a launch

struct TokenPlan {
  int terms, Dp, Bk;
  bool copy;          // W laid out per piece: fp32, 16-bit rows of an odd length, or for `tail`
  int ways;           // terms of f(X) in the logits, in 16 bits
  bool fine;          // the update in 16 bits, small: errors and f(X) in `ways` terms
  bool mend;          // the update in 16 bits, large: targets' errors made good in fp32 (for G in a slice of its own)
  bool fix;           // and the loss corrected
  int ft_terms, f_terms, e_terms;
  bool keep;          // one piece, its exponentials kept
  bool one;           // one tile: losses (and errors) at once
  bool tail;          // the gradient and W's update in one launch, from W's copy
  int cut;            // slices of the batch in that
  int rows, Vp;       // of a piece (the last may have fewer), ET's row length
  int tile, unit;     // of the logits
  int grad_tile, grad_ways, slices;  // of the gradient; its terms of the errors
  long long f, ft, et, kept, ws, part, stats, logit, norm, fixes, order, key, slot, hot, bytes;  // offsets in the workspace
};

// Whether there is a kernel for so many terms of f(X) in the logits (kept: TOKEN_KEEP, else TOKEN_STATS).
inline bool token_ways(int storage, int ways, bool kept) {
  return ways == 1 || (storage != DT_F32 && (kept ? ways == (storage == DT_F16 ? 2 : 3) : ways == 2 || (storage == DT_BF16 && ways == 3)));
}

// false: sizes that the kernels do not take
inline bool plan_token(int V, int D, int B, int storage, int act, bool update, TokenPlan& o) {
  auto up = [](long long v, long long m) { return (v + m - 1) / m * m; };
  o = TokenPlan{};
  o.terms = storage == DT_F32 ? 3 : 1;
  if (D > (1 << 26) || B > (1 << 26)) return false;
  o.Dp = (int)up(D, 32);
  o.Bk = (int)up(B, 32);
  const bool inexact = storage != DT_F32 && act != ACT_IDENTITY && act != ACT_RELU;
  const long long work = (long long)V * B;
  const int most = storage == DT_BF16 ? 3 : 2;
  const long long state = 2LL * o.Dp * o.Bk;
  // (all of an operand's terms lie in one buffer: where f(X)'s do not fit, the call is not a small one)
  const bool few = storage != DT_F32 && state * most <= TOKEN_OPERAND && work <= TOKEN_FINE_ERRORS &&
                   (work * D <= TOKEN_FINE_WORK || (update && storage == DT_BF16 && V <= TOKEN_FINE_WORDS));
  // (V within a tile: a launch less against half as many workgroups at long sums: us, at once / kept first, bf16
  // 64 x 300 x 200 update 21.7 / 25.8, fp32 128 x 512 x 4000 89 / 98, 26 x 2000 x 30 36.6 / 40.7; 128 x 1000 x 100 39 / 37,
  // 100 x 4001 x 16 77 / 64; the loss alone, 64 x 300 x 200 11.6 / 13.7, 100 x 90 x 64 12.8 / 11.9)
  const bool within = V <= TOKEN_ONE_ROWS / 2 || (update && V <= TOKEN_ONE_ROWS && D <= 512);
  const bool tail = update && (few || storage == DT_F32) && V <= 480 && (long long)V * D <= 1 << 20 && token_tail_tiles(V, D, B) <= 256;
  o.copy = storage == DT_F32 || D % 2 != 0 || tail;
  // the rows of a piece, 0 for sizes that the kernels do not take
  auto pieces = [&](bool fine) -> long long {
    o.fine = fine;
    o.mend = update && storage != DT_F32 && !fine;
    o.fix = inexact && o.mend;
    o.ways = fine || (inexact && !update) ? few ? most : 2 : 1;
    o.ft_terms = storage == DT_F32 ? 3 : o.fix ? 2 : o.ways;
    o.f_terms = o.e_terms = storage == DT_F32 ? 3 : fine ? o.ways : 1;
    if (state * o.ft_terms > TOKEN_OPERAND) return 0;
    const long long row_w = 2LL * (o.copy ? o.terms * o.Dp : D), row_e = update ? 2LL * o.e_terms * o.Bk : 1;
    long long rows = std::min((o.copy ? TOKEN_PIECE_BYTES : TOKEN_OPERAND) / row_w, TOKEN_PIECE_BYTES / row_e) / 256 * 256;
    if (rows < 256) rows = 256;
    rows = std::min<long long>(rows, V);
    return up(rows, 32) * std::max(row_w, row_e) > TOKEN_OPERAND ? 0 : rows;
  };
  long long rows = pieces(update && few);
  if (o.fine && rows < V) rows = pieces(false);  // (weights of more than a piece: not a small call)
  if (rows == 0) return false;
  o.rows = (int)rows;
  o.Vp = (int)up(o.rows, 32);
  o.keep = update && o.rows == V && (storage != DT_F32 || (long long)o.Bk * o.Vp * 10 <= TOKEN_PIECE_BYTES);
  o.one = within && (update ? o.keep && !o.mend : o.rows == V && (storage == DT_F32 || (few && o.ways == most)));
  auto tiles = [&](long long m, long long n, long long e) { return ((m + e - 1) / e) * ((n + e - 1) / e); };
  const long long columns = (long long)o.ways * B;
  // (the largest tile that gives the CUs one each; fp32: us, 64 wide / 128 x 64, 4000 x 4000 x 512 update 355 / 336,
  // 10007 x 515 x 77 77 / 72)
  if (o.ways == 3) o.tile = (o.rows + 127LL) / 128 * ((B + 31LL) / 32) >= 256 ? TILE_128_64 : TILE_64;
  else if (columns <= 64) o.tile = o.rows >= 32768 ? TILE_128_64 : TILE_64;
  else o.tile = storage != DT_F32 && tiles(o.rows, columns, 256) >= 192 ? TILE_256 : tiles(o.rows, columns, 128) > 128 ? TILE_128 : storage == DT_F32 && (o.rows + 127LL) / 128 * ((columns + 63) / 64) >= 128 ? TILE_128_64 : TILE_64;
  o.unit = token_unit(o.tile, o.ways);
  // (few tiles: narrow ones, with longer slices: us, fp32 10007 x 515 x 77 70.4 / 70.0, bf16 1000 x 1000 x 128 35.7 / 34.2)
  o.grad_tile = storage != DT_F32 && D >= 256 && B >= 256 ? 256 : D > 64 && tiles(D, B, 128) > 8 ? 128 : 64;
  o.grad_ways = o.fine ? 2 : 1;
  const long long gt = o.grad_tile == 256 ? (D + 255LL) / 256 * ((B + 256 / o.grad_ways - 1LL) / (256 / o.grad_ways))
                       : o.grad_tile == 128 ? (D + 127LL) / 128 * (B > 64 ? (B + 127LL) / 128 : 1) : tiles(D, B, 64);
  const long long stages = o.Vp / 32;
  o.slices = (int)std::max<long long>(1, std::min({256 / gt, stages / 8, 64LL}));
  o.tail = tail && o.keep && !o.mend && o.slices == 1;
  // (W's product: as many slices of eight steps and more as give every CU a workgroup, three at least: us, cut / whole, bf16
  // 6 x 73 x 3026 21.7 / 45, 329 x 3 x 4059 40 / 66, 26 x 40 x 2000 21.3 / 29.2; two: 256 x 256 x 512 27.2 / 25.6)
  o.cut = (int)std::min<long long>(o.Bk / 256, (256 - tiles(D, B, 64)) / tiles(V, D, 64));
  if (o.cut < 3) o.cut = 1;
  // (the other launches have fewer work-items than an operand has bytes)
  if (o.keep && !o.one && 256 * token_error_blocks(o.Bk, o.Vp) > TOKEN_LAUNCH) return false;
  if (o.mend && (256 * (token_rest_blocks(D, B) + token_hot_blocks(o.Dp, B)) > TOKEN_LAUNCH || 2LL * V + 1024 > TOKEN_LAUNCH)) return false;
  long long at = 0;
  auto take = [&](long long bytes) {
    const long long here = at;
    at += up(bytes, 256);
    return here;
  };
  o.ft = take(state * o.ft_terms);
  o.logit = take(4LL * B);
  o.norm = take(8LL * B);
  o.stats = take(8LL * B * (((long long)V + o.unit - 1) / o.unit));
  if (o.copy) o.ws = take((long long)o.terms * o.Vp * o.Dp * 2);
  if (update) {
    o.f = take(state * o.f_terms);
    o.et = take((long long)o.e_terms * o.Bk * o.Vp * 2);
    o.part = o.tail ? o.cut > 1 ? take(4LL * o.cut * V * D) : 0 : take(4LL * (o.slices + (o.mend ? 1 : 0)) * D * B);
    o.kept = o.e_terms == 1 ? o.et : o.keep && !o.one ? take(4LL * o.Bk * o.Vp) : 0;
    o.fixes = o.fix ? take(4LL * B * token_fix_rows(D, false)) : 0;
    if (o.mend) {
      o.order = take(4LL * B);
      o.key = take(4LL * (B + 1));
      o.slot = take(4LL * V);
      o.hot = take(4LL * B * o.Dp);
    }
  }
  o.bytes = at;
  return true;
}

// Of the gradient's contraction over a piece of `rows` rows: as many slices as a whole piece has, but of one stage of
// 32 at least.  (A later piece adds to the first so many sums; the others have theirs.)
inline int token_piece_slices(const TokenPlan& o, int rows) { return std::min(o.slices, (rows + 31) / 32); }

}  // namespace ipc
