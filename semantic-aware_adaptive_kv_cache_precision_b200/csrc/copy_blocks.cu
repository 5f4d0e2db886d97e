// Copies of cache blocks, and of rows of per-sequence state, to other places of their pools or into
// other pools: the partly filled last block of a forked sequence, its state, the blocks of a cache that
// is given another size.
//
//   to[e][target[n]] = from[e][source[n]]      for entries e, pairs n, several tensors in one launch
//
// Nothing is computed; what bounds it is memory: a source read once, a target written once. A thread
// block takes a piece of one (tensor, entry, pair) of up to kPiece bytes, every thread with four 16-byte
// reads in flight before its first write. The pairs travel as arguments of the launch, so a copy needs no
// transfer of its own and no memory on the device. Of a block whose last positions are not filled only
// the filled rows of every head are copied: a "chunk" of the block, `chunk_bytes` of every `chunk_pitch`.
//
// The order of the pieces is free: targets are distinct, and none is a source.
#include <string.h>

#include "common.cuh"

namespace {

constexpr int kMaxTensors = 16;
constexpr int kMaxPairs = 1024;      // 8 KB of the 32 KB that a launch's arguments may take
constexpr int kThreads = 256;
constexpr int kUnroll = 4;           // reads in flight a thread

struct Tensor {
  const uint8_t* from;
  uint8_t* to;
  long long from_entry, to_entry;    // bytes from entry to entry
  long long block;                   // bytes from block to block
  int entries;
  int units;                         // vectors copied of a block
  int chunk_units;                   // vectors of a chunk
  int chunk_pitch;                   // bytes from chunk to chunk
  int pieces;                        // thread blocks for one block of the cache
};

struct Params {
  Tensor tensor[kMaxTensors];
  long long first[kMaxTensors + 1];  // first thread block of each tensor
  int tensors, pairs;
  int2 pair[kMaxPairs];
};

template <typename V>
__global__ void __launch_bounds__(kThreads)
copy_blocks_kernel(const __grid_constant__ Params p) {
  const long long b = blockIdx.x;
  int t = 0;
  while (t + 1 < p.tensors && b >= p.first[t + 1]) ++t;
  const Tensor& x = p.tensor[t];
  const long long at = b - p.first[t];
  const int piece = static_cast<int>(at % x.pieces);
  const long long item = at / x.pieces;
  // (pairs fastest: copies of one source lie side by side and find it in L2)
  const int2 pair = p.pair[item % p.pairs];
  const long long e = item / p.pairs;
  const uint8_t* from = x.from + e * x.from_entry + pair.x * x.block;
  uint8_t* to = x.to + e * x.to_entry + pair.y * x.block;
  const int begin = piece * (kThreads * kUnroll) + threadIdx.x;
  V v[kUnroll];
  long long where[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int u = begin + i * kThreads;
    const int chunk = u / x.chunk_units;
    where[i] = (long long)chunk * x.chunk_pitch + (long long)(u - chunk * x.chunk_units) * sizeof(V);
    if (u < x.units) v[i] = *reinterpret_cast<const V*>(from + where[i]);
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i)
    if (begin + i * kThreads < x.units) *reinterpret_cast<V*>(to + where[i]) = v[i];
}

}  // namespace

// One tensor's part of the copy, as the host describes it (all in bytes).
struct SakvCopyTensor {
  const void* from;
  void* to;
  long long from_entry, to_entry, block, entries, chunks, chunk_bytes, chunk_pitch;
};

// `tensors` descriptors and `pairs` block numbers to copy from and to, all on the HOST and read before the call
// returns. Numbers lie in [0, blocks) and [0, room), a target is named once and, where the targets lie in the sources'
// own tensors (`within`), is no source: else nothing is copied and the call returns -1.
SAKV_EXPORT int sakv_copy_blocks(const SakvCopyTensor* tensor, int tensors, const int* source, const int* target,
                                 int pairs, int blocks, int room, int within, cudaStream_t stream) {
  if (tensors < 0 || pairs < 0 || blocks < 0 || room < 0) return cudaErrorInvalidValue;
  for (int i = 0; i < pairs; ++i)
    if (source[i] < 0 || source[i] >= blocks || target[i] < 0 || target[i] >= room) return -1;
  if (pairs > 1 || within) {
    const size_t n = within && blocks > room ? blocks : room;       // a byte a block: whether it is taken
    uint8_t few[4096];
    uint8_t* taken = n <= sizeof(few) ? few : static_cast<uint8_t*>(malloc(n));
    if (!taken) return cudaErrorMemoryAllocation;
    memset(taken, 0, n);
    bool good = true;
    if (within)
      for (int i = 0; i < pairs; ++i) taken[source[i]] = 1;
    for (int i = 0; i < pairs && good; ++i) {
      good = !taken[target[i]];
      taken[target[i]] = 1;
    }
    if (taken != few) free(taken);
    if (!good) return -1;
  }
  for (int t0 = 0; t0 < tensors; t0 += kMaxTensors) {
    const int n = tensors - t0 < kMaxTensors ? tensors - t0 : kMaxTensors;
    // the widest vector that every address and size of these tensors is a multiple of
    unsigned long long bits = 0;
    for (int i = 0; i < n; ++i) {
      const SakvCopyTensor& x = tensor[t0 + i];
      if (x.entries <= 0 || x.chunks <= 0 || x.chunk_bytes <= 0 || x.chunk_pitch < x.chunk_bytes ||
          x.chunks * x.chunk_pitch > x.block || x.chunk_pitch > 0x7fffffffLL ||
          x.chunks * x.chunk_bytes > 0x3fffffffLL)
        return cudaErrorInvalidValue;
      bits |= (unsigned long long)(uintptr_t)x.from | (uintptr_t)x.to | x.from_entry | x.to_entry |
              x.block | x.chunk_bytes | (x.chunks > 1 ? x.chunk_pitch : 0);
    }
    const int size = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
    Params p;
    p.tensors = n;
    for (int first = 0; first < pairs; first += kMaxPairs) {
      p.pairs = pairs - first < kMaxPairs ? pairs - first : kMaxPairs;
      for (int i = 0; i < p.pairs; ++i) p.pair[i] = make_int2(source[first + i], target[first + i]);
      long long blocks = 0;
      for (int i = 0; i < n; ++i) {
        const SakvCopyTensor& x = tensor[t0 + i];
        Tensor& y = p.tensor[i];
        y.from = static_cast<const uint8_t*>(x.from);
        y.to = static_cast<uint8_t*>(x.to);
        y.from_entry = x.from_entry;
        y.to_entry = x.to_entry;
        y.block = x.block;
        y.entries = static_cast<int>(x.entries);
        y.units = static_cast<int>(x.chunks * x.chunk_bytes / size);
        y.chunk_units = static_cast<int>(x.chunk_bytes / size);
        y.chunk_pitch = static_cast<int>(x.chunk_pitch);
        y.pieces = (y.units + kThreads * kUnroll - 1) / (kThreads * kUnroll);
        p.first[i] = blocks;
        blocks += (long long)y.pieces * p.pairs * x.entries;
      }
      p.first[n] = blocks;
      if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
      const dim3 grid((unsigned)blocks), block(kThreads);
      int e;
      if (size == 16) e = launch_ordered(copy_blocks_kernel<uint4>, grid, block, 0, stream, p);
      else if (size == 4) e = launch_ordered(copy_blocks_kernel<uint32_t>, grid, block, 0, stream, p);
      else if (size == 2) e = launch_ordered(copy_blocks_kernel<uint16_t>, grid, block, 0, stream, p);
      else e = launch_ordered(copy_blocks_kernel<uint8_t>, grid, block, 0, stream, p);
      if (e) return e;
    }
  }
  return 0;
}
