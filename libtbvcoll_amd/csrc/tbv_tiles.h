// Which of its kernels an int8 product takes (tbv_matmul.hip): host arithmetic only, so that a test can ask for the choice
// without a GPU.
#pragma once
#include <stddef.h>

namespace tbv {

// The kernels a product of whole 16-byte pieces can take, as tiles: rows of x by rows of w.  `step` is what 128 bytes of k cost
// with 256 tiles, one for each CU, and `end` the rest, in us, with operands that no cache holds; where a CU holds several blocks
// at a time (`shared`) they fill one another's gaps and the work counts, otherwise whole rounds of 256 tiles do.  128 x 128 comes
// twice: three steps ahead and a block to a CU where one round does (`once`), two steps ahead and two blocks to a CU beyond
// (1024 x 4096 x 8192: 41.6 and 50.5; 2048 x 4096 x 4096: 45.2 and 39.7).  Fitted to 138 products of 1 .. 4096 rows by 2048 .. 28672
// channels of 1024 .. 14336: the estimate is 14 % (rms) off, the tile it picks within 8 % of the best one of all, with operands
// in the caches too.  In us, without the caches, chosen one first, channels and k 4096: 16 rows 16x16 5.9, 16x32 6.8; 32 rows
// 16x32 6.7, 16x16 7.8; 64 rows 32x32 8.0, 16x64 8.8; 128 rows 64x32 10.0, 32x32 10.8; 192 rows 64x64 12.7, 128x64 15.7;
// 384 rows 128x64 17.0, 128x128 21.5; 1024 rows 128x128 24.3 (two steps ahead 28.4); 2048 rows 128x256 38.8, 128x128 41.4;
// 4096 rows 256x256 61.4, 128x256 75.4; 16 x 14336 x 4096 16x64 12.6, 16x32 12.7.
struct Tile { unsigned rows, cols; float end, step; bool ring, shared, once; };
constexpr Tile kTiles[] = {
    {16, 16, 2.9f, 0.092f, true, true, false}, {16, 32, 2.4f, 0.127f, true, true, false}, {16, 64, 1.8f, 0.241f, true, true, false},
    {32, 32, 2.4f, 0.158f, true, true, false}, {64, 32, 2.5f, 0.177f, true, false, false}, {64, 64, 2.9f, 0.281f, false, false, false},
    {128, 64, 2.9f, 0.401f, false, false, false}, {128, 128, 3.1f, 0.574f, false, false, true}, {128, 128, 2.7f, 0.624f, false, false, false},
    {128, 256, 5.8f, 0.882f, false, false, false}, {256, 256, 9.1f, 1.287f, false, false, false}};
// The same for rows that start anywhere (45 products; 14 % and 9 %), 4096 channels of 4097: 16 rows 16x16 7.4, 16x32 9.9; 32 rows
// 16x32 9.5, 16x16 10.6; 64 rows 32x32 11.3, 16x32 14.0; 256 rows 64x64 21.2, 32x32 29.9; 1024 rows 128x128 42.9, 64x64 59.4.
constexpr Tile kAnyTiles[] = {
    {16, 16, 2.7f, 0.105f, true, true, false}, {16, 32, 2.4f, 0.173f, true, true, false}, {32, 32, 2.9f, 0.21f, true, true, false}, {64, 64, 3.2f, 0.489f, true, false, false},
    {128, 128, 5.5f, 1.08f, false, false, false}};

template <int N> inline int pick_tile(const Tile (&tiles)[N], unsigned m, unsigned n, unsigned k)
{
    const float steps = (float)((k + 127) / 128);
    int best = N - 1;
    float least = 0.0f;
    for (int i = 0; i < N; i++) {
        const Tile& t = tiles[i];
        const size_t tm = ((size_t)m + t.rows - 1) / t.rows, tn = ((size_t)n + t.cols - 1) / t.cols;
        if (t.ring && (tm > 65535 || tn > (1u << 20))) continue;      // a grid's y and x
        if (t.once && tm * tn > 256) continue;
        const float rounds = tm * tn <= 256 ? 1.0f : t.shared ? (float)(tm * tn) / 256 : (float)((tm * tn + 255) / 256);
        const float us = t.shared ? t.end + rounds * steps * t.step : rounds * (t.end + steps * t.step);
        if (least == 0.0f || us < least) { best = i; least = us; }
    }
    return best;
}

}  // namespace tbv
