// pz_lmtile.h -- which LM-head path and tile shape a call takes (host only).
#pragma once
#include <stddef.h>
#include <stdint.h>

// Weights the Infinity Cache (256 MB) cannot hold from one call to the next
// are loaded non-temporally: 128256 x 2560 at batch 1 114 -> 98 us, at 8
// (matrix cores) 116 -> 107; 50257 x 1024, which it can hold, 18.2 -> 19.5.
inline bool lm_once(int V, int n) { return (size_t)V * n * 2 > ((size_t)256 << 20); }

// One tile shape of the GEMM: its batch block, rows per workgroup (one
// workgroup per CU, by LDS), and the time of one round of workgroups on every
// CU at n = 2560 (us, measured at V = 128256).
struct LmTile {
  int cols, rows;
  float round_us;
};
constexpr LmTile LM_TILE_SHAPES[] = {
    {256, 256, 192.0f}, {128, 256, 107.0f}, {64, 256, 83.0f}, {32, 256, 64.0f},
    {16, 256, 59.0f}};
constexpr int LM_TILE_COUNT = sizeof(LM_TILE_SHAPES) / sizeof(LM_TILE_SHAPES[0]);

// The shape with the least time for nb batch rows: rounds of workgroups times
// a round's time.  most: batch rows the workspace holds (a multiple of 16).
inline int lm_tile_for(int V, int nb, int most, int n_cu) {
  int best = LM_TILE_COUNT - 1;
  float best_us = __builtin_inff();
  for (int i = 0; i < LM_TILE_COUNT; i++) {
    const LmTile& t = LM_TILE_SHAPES[i];
    if ((nb + t.cols - 1) / t.cols * t.cols > most) continue;  // parts past the workspace
    const long wgs = (long)((V + t.rows - 1) / t.rows) * ((nb + t.cols - 1) / t.cols);
    const float us = (float)((wgs + n_cu - 1) / n_cu) * t.round_us;
    if (us < best_us) {
      best = i;
      best_us = us;
    }
  }
  return best;
}

// Batches of 4 to 32 whose workgroups make the parts themselves: where the
// launch that makes them once takes longer than it saves.  One round of
// 256-row workgroups: rows of up to 256 (us, own / once, as the kernel that
// staged the parts in every workgroup before: 4 x 128 x 8000 5.4 / 7.9, 5.6;
// 32 x 256 x 50257 12.5 / 13.4, 13.7; but 32 x 512 x 50257 18.3 / 17.2, 21.5).
// More rounds, where a ring per workgroup also fills and drains too often: up
// to 1024, past the Infinity Cache 768 (32 x 256 x 128256 15.6 / 20.7, 20.9;
// fused 32 x 1024 x 128256 44.0 / 48.3, 46.1; 16 x 768 x 200000 68.7 / 74.9,
// 75.0; but 32 x 1024 x 200000 107.7 / 99.3, 109.6).
inline bool lm_own_parts(int V, int n, int B, int n_cu) {
  if (B > 32) return false;
  if (V <= 256 * n_cu) return n <= 256;
  return n <= (lm_once(V, n) ? 768 : 1024);
}

// The 8-bit head's shapes (pz_lmhead_i8.hip): batch rows and rows of W of a
// workgroup's tile, and the longest W, in rows per CU, that takes the shape
// before the next of its batch rows does.  Few rows take small tiles whose waves
// share k; every bound lies between two sizes at which the neighbours were
// timed (us at 256 CUs, each with both): 16 batch rows 8000 x 4096 7.7 / 9.1,
// 14000 x 2560 9.9 / 8.7; 32 4000 x 2560 4.7 / 5.6, 8000 x 4096 8.7 / 7.9, 14000 x
// 2560 9.3 / 10.6, 22000 x 2560 12.7 / 11.7; 64 4000 x 2560 6.2 / 7.1, 8000 x 4096
// 14.2 / 10.4 / 14.9, 14000 x 2560 13.8 / 11.2, 40000 x 2560 28.4 / 29.5, 50257 x
// 1024 19.8 / 17.9 / 18.5, 128256 x 2560 83 / 67; 128 4000 x 2560 8.7 / 9.0, 8000 x
// 4096 21.8 / 13.5 / 23.0, 22000 x 2560 24.8 / 19.6 / 23.3, 40000 x 2560 40.4 / 32.9;
// 256 4000 x 2560 14.3 / 16.4, 8000 x 4096 25.2 / 27.2, 14000 x 2560 24.5 / 19.7 /
// 23.9, 22000 x 2560 28.1 / 24.8 / 38.0, 50257 x 1024 47.9 / 44.0.  Shape 2 in place
// of 1 from 5 batch rows: 64000 x 2560 8 rows 34.4 / 31.9, 16 37.0 / 33.5.
struct I8Tile {
  int cols, rows, most;
};
constexpr I8Tile I8_TILE_SHAPES[] = {
    {16, 16, 40},   {16, 32, 160},  {16, 64, 0},    // (0 - 2)
    {32, 16, 24},   {32, 32, 60},   {32, 128, 0},   // (3 - 5)
    {64, 16, 24},   {64, 32, 40},   {64, 64, 180},  {64, 128, 280}, {64, 256, 0},    // (6 - 10)
    {128, 16, 24},  {128, 32, 60},  {128, 64, 140}, {128, 256, 0},                   // (11 - 14)
    {256, 16, 24},  {256, 32, 40},  {256, 64, 70},  {256, 128, 140}, {256, 256, 0}}; // (15 - 19)
constexpr int I8_TILE_COUNT = sizeof(I8_TILE_SHAPES) / sizeof(I8_TILE_SHAPES[0]);

// The first shape of its batch rows that takes a W of V rows (cols: of a tile; more
// batch rows are as many more workgroups).
inline int i8_shape_for(const I8Tile* shapes, int count, int cols, int V, int B, int n_cu) {
  const double rows = (double)V * ((B + cols - 1) / cols) / n_cu;
  for (int i = 0; i < count; i++)
    if (shapes[i].cols == cols && (shapes[i].most == 0 || rows <= shapes[i].most)) return i;
  return count - 1;
}
// Workgroups of a launch of tiles of `rows` x `cols`: the row tiles in eights, one
// for each XCD.
inline int64_t i8_workgroups(int V, int B, int rows, int cols) {
  const int64_t nrt = ((int64_t)V + rows - 1) / rows, ncb = ((int64_t)B + cols - 1) / cols;
  return (nrt + 7) / 8 * 8 * ncb;
}
inline int i8_tile_for(int V, int B, int n_cu) {
  const int cols = B <= 16 ? 16 : B <= 32 ? 32 : B <= 64 ? 64 : B <= 128 ? 128 : 256;
  const int i = i8_shape_for(I8_TILE_SHAPES, I8_TILE_COUNT, cols, V, B, n_cu);
  return i == 2 && B <= 4 ? 1 : i;
}

// The same where rows are off 16 bytes and go through registers, at k = 2565: the
// batch's rows cost as much as W's, so that tiles of more rows pay earlier.  8
// batch rows 10000 14.6 / 15.5, 20000 19.4 / 17.9; 64 5000 18.3 / 25.2 / 32.9, 10000
// 20.4 / 25.6, 20000 29.6 / 27.8 / 34.7, 60000 89 / 69 / 60; 200 2000 24.6 / 28.0, 5000
// 33.6 / 28.0 / 35.2, 10000 49.5 / 49.9 / 35.9, 60000 - / 208 / 126 (256-row tiles
// 124, but 5000 48.2).
constexpr I8Tile I8_ODD_SHAPES[] = {
    {16, 32, 48},  {16, 32, 0},                       // (0, 1: k shared by 4 waves, by 2)
    {64, 32, 60},  {64, 64, 140}, {64, 128, 0},       // (2 - 4)
    {128, 32, 24}, {128, 64, 56}, {128, 128, 0}};     // (5 - 7)
constexpr int I8_ODD_COUNT = sizeof(I8_ODD_SHAPES) / sizeof(I8_ODD_SHAPES[0]);
inline int i8_odd_tile_for(int V, int B, int n_cu) {
  return i8_shape_for(I8_ODD_SHAPES, I8_ODD_COUNT, B <= 16 ? 16 : B <= 64 ? 64 : 128, V, B, n_cu);
}
