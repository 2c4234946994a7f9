// Matrices in 4 bits: codes are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte with the even column in the low half,
// and consecutive columns of a row share a scale in groups.
//   SMAT_FP4_NV  groups of 16, scale e4m3 (bit 7 clear), times an fp32 scale of the row
//   SMAT_FP4_MX  groups of 32, scale 2^(code - 127)
// Dense matrix (activations, [rows][K]):
//   codes   row r at r * fp4_pitch(K) bytes; columns from K to the next multiple of 64 are zeros
//   scales  tiles of 128 rows x 64 columns, 512 bytes each, tile (r / 128, k / 64) at index (r / 128) * fp4_quads(K) + k / 64;
//           the four bytes of a row stand at (r % 32) * 16 + (r % 128) / 32 * 4: the order in which a block-scaled MMA finds the
//           scales of 128 rows in tensor memory, so a tile goes there as it is.  SMAT_FP4_NV uses all four (one for 16 columns),
//           SMAT_FP4_MX the first two (one for 32 columns), the others are zeros.
// Block matrix: block p has its codes at p * 128 (16 rows of 8 bytes) and 16 scales at p * 16, one for each of its rows; of
// SMAT_FP4_MX, the two blocks of an aligned pair of block-columns have equal scales.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "smat_internal.h"

namespace smat {

// Columns are handled 64 at a time: K of one block-scaled MMA, 32 bytes of codes, one scale tile.
inline size_t fp4_quads(size_t K) { return (K + 63) / 64; }
inline size_t fp4_pitch(size_t K) { return fp4_quads(K) * 32; }

// Products with B in 4 bits walk groups of 16 block-rows in steps of 256 columns; steps in which a group has no block are left out (a
// group without any has one, with an empty mask).  Every step has two tiles, one for each half of the group: 128 rows x 256 columns
// as they lie in shared memory, 16384 bytes of codes (128 bytes a row, its 16-byte pieces in the order piece ^ row % 8) and four
// scale tiles of 128 rows x 64 columns, zeros where no block is stored.
constexpr size_t kFp4GroupRows = 16, kFp4StepColumns = 256;
constexpr uint32_t kFp4TileCodes = 16384, kFp4TileBytes = kFp4TileCodes + 2048;
// A step is one word: bits [8, 32) say that its columns begin at 256 times that number (K below 2^26), bit 4 h + q that half h of the
// group has blocks in columns 64 q to 64 q + 63 of them.
struct Fp4Where {         // of what the tiles of a step are made
    int group;            // whose step it is
    int begin[16];        // first block of each block-row in these columns
    uint16_t blocks[16];  // bit c: the block-row has a block in columns 16 c to 16 c + 15 of these
};

// Products with B in 16 bits walk a block-row four blocks at a time, kept by the plan in the order in which a warp's lanes use them:
// 512 bytes of codes (lane l: 16 bytes, a word for each block: columns 4 (l % 4) to + 3 of rows 2 (l / 4) and 2 (l / 4) + 1), 64 bytes
// of scales (8 for each pair of rows: two a block) and four block columns.  The last four of a block-row may be fewer; the rest is
// zeros, with the column of the last block.
constexpr size_t kFp4FourBytes = 512 + 64 + 16;
struct Fp4Row {
    int first, blocks;  // four to begin with, number of blocks
};

// A stored matrix of 16 x 16 blocks in 4 bits and what a plan worked out about block-rows [brow_begin, brow_end).  Device memory.
struct Fp4View {
    const uint8_t* codes = nullptr;
    const uint8_t* scales = nullptr;
    const float* row_scale = nullptr;  // of the whole matrix, or null: ones
    const int* colidx = nullptr;
    const Fp4Row* rows = nullptr;    // of the range; empty where the arrays were inconsistent
    const uint8_t* fours = nullptr;
    int fmt = 0;
    size_t K = 0, brow_begin = 0, block_rows = 0;
    const uint32_t* steps = nullptr;  // null: the plan has no tiles
    const uint8_t* tiles = nullptr;  // two of a step
    const int* gsp = nullptr;        // first step of every group, and the number of all
    const int* h_gsp = nullptr;      // the same on the host
    size_t total_steps = 0;
    size_t blocks = 0, longest = 0;  // stored blocks of the range, and of its longest block-row
};

// Dense right-hand side: 16-bit values [N][K], or 4 bits as above.
struct Fp4Rhs {
    const void* data = nullptr;      // values, or codes
    const uint8_t* scales = nullptr;  // 4 bits
    const float* row_scale = nullptr;  // 4 bits; may be null
    int dtype = 0;                   // SMAT_F16 or SMAT_BF16, or kFp4Rhs
};
constexpr int kFp4Rhs = 3;

int launch_fp4_stream(const Fp4View& A, const Fp4Rhs& B, void* C, int c_dtype, size_t N, cudaStream_t stream);

// selftest: waits for codes run out (smat_selftest_fp4_plan_wait_timeout).
int launch_fp4_tile(const Fp4View& A, const Fp4Rhs& B, void* C, int c_dtype, size_t N, cudaStream_t stream, bool selftest = false);

}  // namespace smat
