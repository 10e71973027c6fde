// Moves of whole rows within buffers [layers, rows, ...]: pages of a cache (forked for another request), rows of
// fixed-size states (beams that change places).
//
//   buffer[l, dst[i], :] = old buffer[l, src[i], :]      for every i and layer l, as if all at once
//
// A row may be a source and a destination in the same call (a permutation, cycles included): a workgroup owns a range
// of columns of one layer for all of the call's moves, has every piece it reads in registers before it stores the
// first one, and no other workgroup touches those columns.  So nothing is staged in memory: a source piece is read for
// each move that it is the source of, and each destination piece written once, which is what bounds the kernel.
#include "common.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

#define ROWS_MAX_BUFFERS 8
// Pieces that a thread holds.  Few of them, in workgroups of 512 threads, keep more workgroups on a compute unit, some
// loading while others store (12 layers of 64 states of 512 KB: 146 us, 4.5 TB/s; with 16 pieces in 256 threads 174);
// long lists take what registers there are, so that a row's columns come in whole lines for up to 2,048 moves (beyond,
// pieces of a line to a workgroup, 16 bytes at 16,384).
#define ROWS_PIECES 4
#define ROWS_THREADS 512
#define ROWS_PIECES_MANY 16
#define ROWS_THREADS_MANY 1024
#define ROWS_MAX_MOVES (ROWS_THREADS_MANY * ROWS_PIECES_MANY)

struct RowBuffers {
  char* base[ROWS_MAX_BUFFERS];
  int64_t layer_bytes[ROWS_MAX_BUFFERS];     // from one layer to the next
  int64_t row_stride[ROWS_MAX_BUFFERS];      // from one row to the next, bytes
  int64_t pieces[ROWS_MAX_BUFFERS];          // pieces of a row
  int64_t first_block[ROWS_MAX_BUFFERS + 1]; // of each buffer in the grid
  int rows[ROWS_MAX_BUFFERS];
  int count;
};

// Thread t holds the pieces t, t + THREADS, ... of the (move, column) table of its workgroup, 1 << wide columns to a move.
template <typename P, int THREADS, int PIECES>
__global__ __launch_bounds__(THREADS) void move_rows_kernel(RowBuffers bufs, const int* __restrict__ src,
                                                            const int* __restrict__ dst, int moves, int wide) {
  int b = 0;
  while (b + 1 < bufs.count && (int64_t)blockIdx.x >= bufs.first_block[b + 1]) ++b;
  const int64_t block = (int64_t)blockIdx.x - bufs.first_block[b];
  const int64_t spans = (bufs.pieces[b] + (1 << wide) - 1) >> wide;
  const int64_t layer = block / spans, column0 = (block % spans) << wide;
  char* base = bufs.base[b] + layer * bufs.layer_bytes[b];
  const int rows = bufs.rows[b];
  P held[PIECES];
  char* to[PIECES];
#pragma unroll
  for (int r = 0; r < PIECES; ++r) {
    const int i = threadIdx.x + r * THREADS;
    const int move = i >> wide;
    const int64_t column = column0 + (i & ((1 << wide) - 1));
    to[r] = nullptr;
    if (move < moves && column < bufs.pieces[b]) {
      const int s = src[move], d = dst[move];
      if (s != d && s >= 0 && s < rows && d >= 0 && d < rows) {
        held[r] = *reinterpret_cast<const P*>(base + s * bufs.row_stride[b] + column * (int64_t)sizeof(P));
        to[r] = base + d * bufs.row_stride[b] + column * (int64_t)sizeof(P);
      }
    }
  }
  // every load of the workgroup has returned before any thread stores
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int r = 0; r < PIECES; ++r)
    if (to[r]) *reinterpret_cast<P*>(to[r]) = held[r];
}

template <typename P, int THREADS, int PIECES>
static void launch_move_rows(RowBuffers& bufs, const int* src, const int* dst, int moves, int wide, int64_t blocks,
                             hipStream_t stream) {
  move_rows_kernel<P, THREADS, PIECES><<<(uint32_t)blocks, THREADS, 0, stream>>>(bufs, src, dst, moves, wide);
}

// spec: of each of the `count` buffers, on the host, its address, the bytes from layer to layer, from row to row and of a
// row, its layers and rows.
MI_EXPORT int mi_move_rows(int count, const int64_t* spec, const int* src, const int* dst, int moves, hipStream_t stream) {
  MI_REQUIRE(count >= 1 && count <= ROWS_MAX_BUFFERS, "move_rows: %d buffers, 1 to %d are taken", count, ROWS_MAX_BUFFERS);
  MI_REQUIRE(moves >= 0 && moves <= ROWS_MAX_MOVES, "move_rows: %d moves, at most %d are taken", moves, ROWS_MAX_MOVES);
  if (moves == 0) return 0;
  uint64_t align = 0;
  for (int b = 0; b < count; ++b) {
    const int64_t* s = spec + 6 * b;
    MI_REQUIRE(s[3] >= 0 && s[2] >= s[3] && s[4] >= 0 && s[5] >= 0 && s[5] <= INT32_MAX, "move_rows: bad sizes of buffer %d", b);
    align |= (uint64_t)s[0] | (uint64_t)s[1] | (uint64_t)s[2] | (uint64_t)s[3];
  }
  const int piece = align % 16 == 0 ? 16 : align % 4 == 0 ? 4 : align % 2 == 0 ? 2 : 1;
  // Columns to a workgroup: as many as its registers hold for all moves.
  const bool many = moves > ROWS_THREADS * ROWS_PIECES / 8;
  const int room = many ? ROWS_THREADS_MANY * ROWS_PIECES_MANY : ROWS_THREADS * ROWS_PIECES;
  int wide = 0;
  while (wide < 12 && ((int64_t)moves << (wide + 1)) <= room) ++wide;
  RowBuffers bufs;
  bufs.count = count;
  int64_t blocks = 0;
  for (int b = 0; b < count; ++b) {
    const int64_t* s = spec + 6 * b;
    bufs.base[b] = (char*)s[0];
    bufs.layer_bytes[b] = s[1];
    bufs.row_stride[b] = s[2];
    bufs.pieces[b] = s[3] / piece;
    bufs.rows[b] = (int)s[5];
    bufs.first_block[b] = blocks;
    blocks += s[4] * ((bufs.pieces[b] + (1 << wide) - 1) >> wide);
  }
  bufs.first_block[count] = blocks;
  MI_REQUIRE(blocks <= 0x7fffffff, "move_rows: %lld workgroups are too many for one launch", (long long)blocks);
  if (blocks == 0) return 0;
#define LAUNCH(P) (many ? launch_move_rows<P, ROWS_THREADS_MANY, ROWS_PIECES_MANY>(bufs, src, dst, moves, wide, blocks, stream) \
                        : launch_move_rows<P, ROWS_THREADS, ROWS_PIECES>(bufs, src, dst, moves, wide, blocks, stream))
  if (piece == 16) LAUNCH(u32x4);
  else if (piece == 4) LAUNCH(uint32_t);
  else if (piece == 2) LAUNCH(uint16_t);
  else LAUNCH(uint8_t);
#undef LAUNCH
  MI_CHECK_LAUNCH("move_rows");
  return 0;
}
