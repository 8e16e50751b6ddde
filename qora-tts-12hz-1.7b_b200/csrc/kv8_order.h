// kv8_order.h -- the barrier and the parity of the waits of a tile CTA
// (kv8_tile.cu) that more than one part takes, apart from the kernel so that a
// host program can walk through every order in which the parts may run.
//
// A wait by parity tells a phase from the one before and the one after it, no
// more: it holds up for the right phase only if, whenever it is made, the
// phase before has ended and the one after has not.
#pragma once

#ifdef __CUDACC__
#define QTTS_TILE_HD __host__ __device__ __forceinline__
#else
#define QTTS_TILE_HD inline
#endif

namespace qtts {

struct TileTurn {
  int bar;          // which of a pair of barriers
  unsigned parity;  // of the phase
};

// "The products into O of the half's n-th tile are done."  16-bit rows: a barrier
// a half, as the next tile's products wait for the half's softmax, which has
// waited for these.  f32 rows: a barrier for each of the two buffers of O.  Who
// adds the tiles up may be a tile behind the products; the next phase of the
// buffer's barrier begins only when it has given the buffer back (o_free).
QTTS_TILE_HD TileTurn o_full_turn(bool split, int half, int n) {
  return split ? TileTurn{n & 1, (unsigned)(n >> 1) & 1u} : TileTurn{half, (unsigned)n & 1u};
}
// f32 rows: "the n-th tile has been added up, its buffer of O is free."
QTTS_TILE_HD TileTurn o_free_turn(int n) { return TileTurn{n & 1, (unsigned)(n >> 1) & 1u}; }

// f32 rows: "all tiles of the n-th segment that has any are added up", which the
// softmax waits for before it reads the sums.  (o_free of the last tile would not
// do: the tile of that buffer before may still be on its way then, and the wait
// would take its parity for the one that is meant.)
QTTS_TILE_HD unsigned summed_parity(int n) { return (unsigned)n & 1u; }

}  // namespace qtts
