// Log-probabilities of given tokens under the output head, without keeping the logits:
//
//   z_v = cap(scale (x . w_v + b_v)),   cap(z) = c tanh(z / c) where c > 0
//   lse = m + log sum_v e^(z_v - m),  m = max_v z_v;    logprob = z_target - lse
//
// The vocabulary is taken in pieces: a piece leaves (m, sum e^(z - m)) a row (m in natural units: the type's lowest
// value, a common mask, times log2(e) would be -inf), and whoever meets the target's column leaves z_target;
// `join_kernel` merges the pieces. 2,048 tokens over 151,936 logits would be 1.2 GB written and read again; the pieces
// are 10 MB.
//
// Ways to a piece. bfloat16 operands: tcgen05 on PAIRS of SMs (`cta_group::2`), the softmax's sums in the
// epilogue. A pair takes a tile of the head's rows (up to 128 a block) against
//   256 tokens   tokens on tensor memory's lanes, the head's rows its columns: thread = token row, so that no sum
//                crosses a thread, or
//   a rest       of up to 96 tokens the other way round, the head's rows on the lanes and the tokens, rounded up to
//                32, the columns: a few tokens do not pay for 256. 32 columns are reduced over 32 lanes in 31
//                exchanges (each step hands half of what is left to the neighbour), and a warp keeps its running
//                sums for the whole kernel, or
//   both         257 to 384 tokens: what comes of the head into shared memory serves both products (what L2 gives
//                an SM bounds tiles of this size), at the price of one accumulator instead of two.
//   warp 0     TMA: boxes of x and of the head (64 wide) into a ring of stages (each block of the pair fetches
//              its own half of both; no multicast),
//   warp 1     tensor memory; in the pair's first block lane 0 issues the products,
//   warps 2-9  epilogue of a tile under the products of the next (two accumulators of 256 columns): two warps for
//              every 32 lanes of tensor memory, each with every other run of columns.
// Tiles of one piece of the head lie side by side in time, so the head comes from memory once. Up to some 256
// tokens its bytes bound the kernel, above the tensor cores. The tile's height is chosen so that the last round
// of tiles is not nearly empty (see the launcher).
// float32 operands: each number as three of bfloat16 on the tensor cores (`split_logprob_kernel`), or plain multiply-adds
// where the head's rows are not aligned; each sum over k and each row's sums over the vocabulary in one order whatever
// rows are beside it, as in the other 32-bit products. bfloat16 rows that TMA cannot take come as copies that it can
// (`pad_kernel`).
//
// Sums and maxima are fp32. Every mbarrier wait is bounded, and a pair leaves together.
// The reference keeps all logits (`src/microinfer/model.py:388-402`).
#include "common.cuh"
#include "mma.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace {

constexpr int BM = 128;                          // rows of an operand that a block holds at most
constexpr int BK = 64;
constexpr int kMaxStages = 12;
constexpr int kWBytes = BM * BK * 2;             // room for the head's rows in a stage
constexpr int kXBytes = BM * BK * 2;
constexpr int kMaxTokens = 256;                  // tokens of a tile
// Tokens behind the last 256 up to which they are a rest; more are a tile of 256 that is not full. Measured
// (us, rest / tile of 256; the sums over lanes cost the rest more where K is small): 97 tokens alone, vocabulary
// x K 151936 x 1536 95 / 98, 50257 x 2048 62 / 52, 50257 x 768 35 / 33, 152064 x 3584 200 / 215; 129 100 / 100,
// 54 / 52, 37 / 33, 232 / 218; 65 behind 512 tokens 291 / 263, 110 / 114, 52 / 51, 560 / 599; 140 behind them
// 280 / 268, 118 / 116, 60 / 51, 658 / 645.
constexpr int kRestMost = 96;
// Tokens behind 256 up to which one tile takes both, where K is at most kLongK. Measured likewise (both / two tiles of
// 256): 32 170 / 178, 70 / 84, 39 / 40, 375 / 394; 77 172 / 177, 76 / 84, 44 / 41, 380 / 394; 128 180 / 181, 79 / 85, 46 / 41, 367 /
// 408; 160 189 / 182, 83 / 86, 49 / 41, 435 / 409.
constexpr int kBothMost = 128;
// The tensor cores cut where they add, always the same way: K is taken in chunks of at most kLongK, added up in fp32 by
// the epilogue (512 tokens and K = 4,096: relative error 5.9e-7, in one sum 2.7e-6; 64 and 1,536: 2.1e-7, 4.5e-7; the
// time is the same). 257 to 384 tokens in one tile have no registers left for that: above kLongK they are two tiles
// (333 tokens, K = 2,048, 50,257 rows: 85 us; one tile took 1 to 4 % more, with an error of 8e-7 instead of 3e-7).
constexpr int kLongK = 1024;
constexpr int kEpilogueThreads = 256;            // two warps a quarter of tensor memory's lanes, each half the columns
constexpr int kThreads = 64 + kEpilogueThreads;
constexpr uint32_t kTmemCols = 512;
constexpr uint16_t kBoth = 3;
constexpr float kLog2e = 1.4426950408889634f;

// two floats in a register pair, and arithmetic on them (sm_100: one instruction for both)
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ uint64_t both(float a) { return two(a, a); }
__device__ __forceinline__ void apart_two(uint64_t d, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
}
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul_two(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// What becomes of a product x . w before the softmax.
struct Shape {
  const void* bias;          // or null
  int bias_bf16;
  float scale;
  float cap, over_cap;       // 0: none; 1 / cap
};

__device__ __forceinline__ float bias_at(const Shape& f, int v) {
  return f.bias_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(f.bias)[v])
                     : reinterpret_cast<const float*>(f.bias)[v];
}

// The tensor-core kernel works on logits in a unit of its own, so that what shapes them costs little: with a cap a
// logit is c tanh(y), y = (x . w + b) scale / c, and t = tanh(y) stands for it in maxima and exponents, whose factor
// takes the cap up; without one it stands for itself.
struct Unit {
  float mul;             // y or z = mul (x . w) + mul b
  float size;            // natural units in one (the cap, or 1)
  float rate;            // log2(e) size
};
__device__ __forceinline__ Unit unit_of(const Shape& f) {
  const float size = f.cap > 0.f ? f.cap : 1.f;
  return Unit{f.cap > 0.f ? f.scale * f.over_cap : f.scale, size, kLog2e * size};
}

// tanh(y) = 1 - 2 / (e^2y + 1), and below 1/4, where that difference would cancel, the series y - y^3/3 + 2 y^5/15
// - 17 y^7/315 + 62 y^9/2835 (the next term is below 2^-26 of y there). Logits are mostly all near zero or not: a
// run of them takes the series alone where it may.
constexpr float kNear = 0.25f;
template <int N>
__device__ __forceinline__ void tanh_all(float (&y)[N]) {
  float big[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; i += 8)
#pragma unroll
    for (int q = 0; q < 4; ++q) big[q] = mma::max3(big[q], fabsf(y[i + 2 * q]), fabsf(y[i + 2 * q + 1]));
  const bool far = !(fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3])) < kNear);      // (NaN is itself in the series)
  if (__any_sync(0xffffffffu, far)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // (2 log2(e) y is kept below 2^7, where the quotient is still one; NaN stays)
      const float e = y[i] > 40.f ? 40.f : y[i], q = y[i] * y[i];
      const float t = 1.f - __fdividef(2.f, 1.f + mma::exp2_fast(e * (2.f * kLog2e)));
      const float s = fmaf(y[i] * q, fmaf(q, fmaf(q, fmaf(q, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), y[i]);
      y[i] = fabsf(y[i]) < kNear ? s : t;
    }
  } else {
    const uint64_t c9 = both(62.f / 2835.f), c7 = both(-17.f / 315.f), c5 = both(2.f / 15.f), c3 = both(-1.f / 3.f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint64_t v = two(y[i], y[i + 1]), q = mul_two(v, v);
      const uint64_t s = fma_two(q, fma_two(q, fma_two(q, c9, c7), c5), c3);
      apart_two(fma_two(mul_two(v, q), s, v), y[i], y[i + 1]);
    }
  }
}

struct Params {
  int M, N, K;               // tokens, vocabulary, inner size
  int full, rest, rest_cols; // tiles of 256 tokens; tokens behind them, and those rounded up to 32
  int both;                  // one tile takes 256 tokens AND the rest (full is 1)
  int chunk;                 // steps of BK that go into one sum
  int w_rows;                // rows of the head a block takes of a tile
  int n_tiles;               // tiles of 2 w_rows rows of the head
  int stages, stage_bytes;
  const int32_t* targets;
  float2* part;              // [n_tiles][256 full], then [blocks][rest]: (maximum, sum)
  float* mine;               // [M]: the targets' logits
  Shape form;
  int* error;
};

struct Barriers {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem;
};

// Behind the ring: barriers, a tile's biases twice, the rest's targets, and the warps' running sums of the rest.
struct Tail {
  Barriers bar;
  alignas(16) float bias[2][2 * BM];
  alignas(16) int32_t target[kMaxTokens];
  float2 run[4][kMaxTokens];
  float2 share[BM];
};
constexpr int kSmemMost = 232448;                // 227 KB
constexpr int kRingMost = kSmemMost - 1024 - static_cast<int>(sizeof(Tail));

// Which tile a pair takes in a round. (Shifted by one a round: with an even number of pairs and of token tiles
// each pair would otherwise meet the same kind of tile every time.)
struct Tiles {
  int per, total;
  __device__ explicit Tiles(const Params& p)
      : per(p.both ? 1 : p.full + (p.rest > 0)), total(per * p.n_tiles) {}
  __device__ int at(int round, int pair, int pairs) const { return round * pairs + (pair + round) % pairs; }
};

__device__ __forceinline__ void ld_32x32b_x32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
      "%23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// e^(size (z - top)), rate = log2(e) size; right where the difference is: top may be -inf only beside z = -inf (0) or
// NaN (NaN)
__device__ __forceinline__ float weight_of(float z, float top, float rate) {
  return mma::exp2_fast((z - (top == -INFINITY ? 0.f : top)) * rate);
}
// Below this a maximum's product with log2(e) leaves the type's range, or nearly.
constexpr float kLow = -2e38f;

// 64 columns of a row joined to the row's running (maximum, sum).
__device__ __forceinline__ void take_up(const float (&z)[64], float rate, float& top, float& sum) {
  float big4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 64; c += 8)
#pragma unroll
    for (int q = 0; q < 4; ++q) big4[q] = mma::max3(big4[q], z[c + 2 * q], z[c + 2 * q + 1]);
  const float big = fmaxf(fmaxf(big4[0], big4[1]), fmaxf(big4[2], big4[3]));
  if (big > top) {
    sum = sum == 0.f ? 0.f : sum * weight_of(top, big, rate);
    top = big;
  }
  if (top < kLow) {                    // nothing so far, or values that a mask made the type's lowest
#pragma unroll
    for (int c = 0; c < 64; ++c) sum += weight_of(z[c], top, rate);
    return;
  }
  const float base = top * rate;
  float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 64; c += 2) {
    float e0, e1;
    mma::fma2(e0, e1, z[c], z[c + 1], rate, -base);
    mma::add2(s4[c & 2], s4[(c & 2) + 1], mma::exp2_fast(e0), mma::exp2_fast(e1));
  }
  sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
}

// 32 values a lane reduced over the lanes: lane i gets the i-th's. Each step a lane keeps half of its values and
// gets its neighbour's share of them.
template <bool kMax>
__device__ __forceinline__ float over_lanes(float (&v)[32], int lane) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const bool upper = lane & s;
#pragma unroll
    for (int i = 0; i < s; ++i) {
      const float keep = upper ? v[i + s] : v[i], give = upper ? v[i] : v[i + s];
      const float got = __shfl_xor_sync(0xffffffffu, give, s);
      v[i] = kMax ? fmaxf(keep, got) : keep + got;
    }
  }
  return v[0];
}

// kPlain: no bias, no scale, no cap; kLong: K in several chunks
template <bool kPlain, bool kCap, bool kLong>
__global__ void __launch_bounds__(kThreads, 1)
logprob_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap rest_map,
               const __grid_constant__ CUtensorMap w_map, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Tail* tail = reinterpret_cast<Tail*>(smem + p.stages * p.stage_bytes);
  Barriers* bar = &tail->bar;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(tma::cluster_rank());
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const Tiles tiles(p);
  const int n_kb = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      tma::mbar_init(&bar->full[s], 1);
      tma::mbar_init(&bar->empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tma::mbar_init(&bar->acc_full[i], 1);
      tma::mbar_init(&bar->acc_empty[i], 2 * kEpilogueThreads);
    }
    tma::fence_barrier_init();
  }
  if (warp == 1) tc::tmem_alloc_pair(&bar->tmem, kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tma::cluster_sync_all();
  tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bar->tmem, 0);      // (known to be the warp's own)
  let_next_kernel_start();       // (with its shared and tensor memory in hand)
  wait_for_previous_kernel();

  if (warp == 0) {
    // ---- TMA: this block's half of the tile's tokens and of its rows of the head -----------------
    if (lane == 0) {
      tma::prefetch_map(&w_map);
      int stage = 0, phase = 0;
      bool ok = true;
      for (int round = 0; round * pairs < tiles.total && ok; ++round) {
        const int tile = tiles.at(round, pair, pairs);
        if (tile >= tiles.total) continue;
        const int m_tile = tile % tiles.per, n_tile = tile / tiles.per;     // tokens fastest
        const bool wide = m_tile < p.full, rest = !wide || p.both;
        const int w_row = (2 * n_tile + rank) * p.w_rows;
        const int x_row = m_tile * kMaxTokens + rank * BM;
        const int rest_row = p.full * kMaxTokens + rank * (p.rest_cols / 2);
        const int rest_at = kWBytes + (wide ? kXBytes : 0);
        const uint32_t bytes = 2 * (p.w_rows + (wide ? BM : 0) + (rest ? p.rest_cols / 2 : 0)) * BK * 2;
        for (int kb = 0; kb < n_kb; ++kb) {
          if (!tma::mbar_wait(&bar->empty[stage], phase ^ 1, p.error, 801)) {
            ok = false;
            break;
          }
          uint8_t* dst = smem + stage * p.stage_bytes;
          const uint32_t full = tma::cluster_address(tma::smem_u32(&bar->full[stage]), 0);
          if (rank == 0) tma::mbar_expect_tx(&bar->full[stage], bytes);
          tma::load_2d_pair(dst, &w_map, kb * BK, w_row, full);
          if (wide) tma::load_2d_pair(dst + kWBytes, &x_map, kb * BK, x_row, full);
          if (rest) tma::load_2d_pair(dst + rest_at, &rest_map, kb * BK, rest_row, full);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // before this block may leave: every stage it filled has been given back
      for (int s = 0; s < p.stages && ok; ++s) {
        ok = tma::mbar_wait(&bar->empty[stage], phase ^ 1, p.error, 805);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // ---- products, issued in the pair's first block: the whole warp walks and one lane issues, and no turn of the loops
    // depends on what a lane saw, so that the operands stay in uniform registers (5 to 10 % of the kernel's time) ----
    if (rank == 0) {
      const uint32_t elected = tc::elect_lane();
      const uint64_t first = tc::smem_desc_k_major_sw128(tma::smem_u32(smem));      // (descriptors count 16 bytes)
      const uint32_t wide_desc = tc::idesc_bf16_f32(2 * BM, 2 * p.w_rows);
      const uint32_t rest_desc = tc::idesc_bf16_f32(2 * BM, p.rest_cols);
      int stage = 0, phase = 0, count = 0;
      bool ok = true;
      for (int round = 0; round * pairs < tiles.total; ++round) {
        const int tile = tiles.at(round, pair, pairs);
        if (tile >= tiles.total) continue;
        const bool wide = tile % tiles.per < p.full, rest = !wide || p.both;
        for (int chunk = 0; chunk < n_kb; chunk += p.chunk) {
          // (both: 256 tokens in the first half of tensor memory, the rest in the second, one sum at a time)
          const int buf = p.both ? 0 : count & 1, use = p.both ? count : count >> 1;
          const uint32_t wide_acc = tmem + buf * kMaxTokens, rest_acc = tmem + (p.both ? 1 : buf) * kMaxTokens;
          ok = ok && (use < 1 || tma::mbar_wait(&bar->acc_empty[buf], (use - 1) & 1, p.error, 802));
          const int end = min(chunk + p.chunk, n_kb);
          for (int kb = chunk; kb < end; ++kb) {
            ok = ok && tma::mbar_wait(&bar->full[stage], phase, p.error, 803);
            __syncwarp();
            tc::fence_after_sync();
            const uint32_t go = elected && ok;
            const uint64_t w = first + stage * (p.stage_bytes >> 4), x = w + (kWBytes >> 4);
            const uint64_t xr = x + (wide ? kXBytes >> 4 : 0);
            if (wide) {
#pragma unroll
              for (int k = 0; k < BK / 16; ++k)
                tc::mma_ss_pair_if(go, wide_acc, x + 2 * k, w + 2 * k, wide_desc, kb > chunk || k > 0);
            }
            if (rest) {
#pragma unroll
              for (int k = 0; k < BK / 16; ++k)
                tc::mma_ss_pair_if(go, rest_acc, w + 2 * k, xr + 2 * k, rest_desc, kb > chunk || k > 0);
            }
            tc::commit_pair_if(go, &bar->empty[stage], kBoth);
            if (++stage == p.stages) {
              stage = 0;
              phase ^= 1;
            }
          }
          tc::commit_pair_if(elected && ok, &bar->acc_full[buf], kBoth);
          ++count;
        }
      }
    }
  } else {
    // ---- epilogue -------------------------------------------------------------------------------
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const int thread = quarter * 32 + lane;                          // lane of tensor memory
    const int worker = half * BM + thread;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const Unit unit = kPlain ? Unit{1.f, 1.f, kLog2e} : unit_of(p.form);
    const int first_rest = p.full * kMaxTokens;
    float2* run = tail->run[quarter];        // (a warp's own columns of it)
    for (int c = worker; c < kMaxTokens; c += kEpilogueThreads)
      tail->target[c] = c < p.rest ? p.targets[first_rest + c] : -1;
    for (int c = half * 32 + lane; c < kMaxTokens; c += 64) run[c] = make_float2(-INFINITY, 0.f);
    asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueThreads) : "memory");
    int count = 0, wide = 0;       // sums so far, and tiles of 256 tokens among theirs
    bool ok = true;
    // the sums of all chunks of K, `width` columns a run, this thread's runs from half `width` on, every other one
    auto add_up = [&](auto& sums, int cols, int real) {
      constexpr int kRuns = sizeof(sums) / sizeof(sums[0]), kWidth = sizeof(sums[0]) / sizeof(float);
#pragma unroll
      for (int r = 0; r < kRuns; ++r)
#pragma unroll
        for (int i = 0; i < kWidth; ++i) sums[r][i] = 0.f;
      for (int kb = 0; kb < n_kb; kb += p.chunk) {
        const int buf = count & 1;
        ok = ok && tma::mbar_wait(&bar->acc_full[buf], (count >> 1) & 1, p.error, 804);
        ok = __all_sync(0xffffffffu, ok);
        tc::fence_after_sync();
#pragma unroll
        for (int r = 0; r < kRuns; ++r) {
          const int c = (2 * r + half) * kWidth;
          if (c < cols && c < real && ok) {
#pragma unroll
            for (int i = 0; i < kWidth; i += 16) {
              float some[16];
              tc::ld_32x32b_x16(lane_base + buf * kMaxTokens + c + i, some);
#pragma unroll
              for (int j = 0; j < 16; j += 2) mma::add2(sums[r][i + j], sums[r][i + j + 1], some[j], some[j + 1]);
            }
          }
        }
        tc::fence_before_sync();
        tma::mbar_arrive_cluster(tma::cluster_address(tma::smem_u32(&bar->acc_empty[buf]), 0));
        ++count;
      }
    };
    for (int round = 0; round * pairs < tiles.total; ++round) {
      const int tile = tiles.at(round, pair, pairs);
      if (tile >= tiles.total) continue;
      const int m_tile = tile % tiles.per, n_tile = tile / tiles.per;
      const int buf = p.both ? 0 : count & 1, use = p.both ? count : count >> 1;
      const int n0 = n_tile * 2 * p.w_rows;
      if (m_tile < p.full) {
        // tokens on the lanes: this thread's row against 2 w_rows rows of the head
        const int cols = 2 * p.w_rows;
        const int m = m_tile * kMaxTokens + rank * BM + thread;
        const int target = m < p.M ? p.targets[m] : -1;
        // (a warp that comes here has seen every other one behind the barrier of the wide tile before, and so
        // done with the one before that, whose biases these replace)
        const float* biases = tail->bias[wide & 1];
        if (!kPlain && p.form.bias) {
          for (int c = worker; c < cols; c += kEpilogueThreads)
            tail->bias[wide & 1][c] = n0 + c < p.N ? bias_at(p.form, n0 + c) * unit.mul : 0.f;
          asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueThreads) : "memory");
        }
        ++wide;
        float top = -INFINITY, sum = 0.f;
        auto take = [&](float (&z)[64], int c) {
          if (!kPlain) {
            if (p.form.bias) {
#pragma unroll
              for (int i = 0; i < 64; i += 4) {
                const float4 b = *reinterpret_cast<const float4*>(biases + c + i);
                apart_two(fma_two(two(z[i], z[i + 1]), both(unit.mul), two(b.x, b.y)), z[i], z[i + 1]);
                apart_two(fma_two(two(z[i + 2], z[i + 3]), both(unit.mul), two(b.z, b.w)), z[i + 2], z[i + 3]);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 64; i += 2) mma::mul2(z[i], z[i + 1], unit.mul);
            }
            if (kCap) tanh_all(z);
          }
          const int real = min(cols, p.N - n0) - c;         // columns of the 64 that are tokens' of this tile
          if (real < 64) {
#pragma unroll
            for (int i = 0; i < 64; ++i) z[i] = i < real ? z[i] : -INFINITY;
          }
          const int at = target - (n0 + c);
          const bool here = at >= 0 && at < min(real, 64);
          if (__any_sync(0xffffffffu, here)) {
            float found = 0.f;
#pragma unroll
            for (int i = 0; i < 64; ++i) found = at == i ? z[i] : found;
            if (here) p.mine[m] = found * unit.size;       // (a row behind the last token has no target)
          }
          take_up(z, unit.rate, top, sum);
        };
        if (kLong) {
          float sums[2][64];
          add_up(sums, cols, p.N - n0);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int c = (2 * r + half) * 64;
            if (c < cols && ok && n0 + c < p.N) take(sums[r], c);
          }
        } else {
          ok = ok && tma::mbar_wait(&bar->acc_full[buf], use & 1, p.error, 804);
          tc::fence_after_sync();
          const uint32_t acc = lane_base + buf * kMaxTokens;
#pragma unroll 1
          for (int c = half * 64; c < cols && ok && n0 + c < p.N; c += 128) {
            float z[64];
            tc::ld_32x32b_x64(acc + c, z);
            take(z, c);
          }
        }
        // the second warp of the quarter hands its share to the first
        if (half) tail->share[thread] = make_float2(top, sum);
        asm volatile("bar.sync %0, 64;" ::"r"(2 + quarter) : "memory");
        if (!half) {
          const float2 other = tail->share[thread];
          const float big = fmaxf(top, other.x);
          sum = (sum == 0.f ? 0.f : sum * weight_of(top, big, unit.rate)) +
                (other.y == 0.f ? 0.f : other.y * weight_of(other.x, big, unit.rate));
          if (ok && m < p.M) p.part[(long long)n_tile * first_rest + m] = make_float2(big * unit.size, sum);
        }
        asm volatile("bar.sync %0, 64;" ::"r"(2 + quarter) : "memory");
      }
      if (m_tile == p.full || p.both) {
        // rows of the head on the lanes: this thread's row against the rest of the tokens
        const int v = n0 + rank * p.w_rows + thread;
        const bool real = thread < p.w_rows && v < p.N;
        const float bias = !kPlain && p.form.bias && real ? bias_at(p.form, v) * unit.mul : 0.f;
        auto take = [&](float (&z)[32], int c) {
          if (!kPlain) {
#pragma unroll
            for (int i = 0; i < 32; ++i) z[i] = fmaf(z[i], unit.mul, bias);
            if (kCap) tanh_all(z);
          }
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const int4 t = *reinterpret_cast<const int4*>(&tail->target[c + i]);
            const int of[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (of[j] == v && real) p.mine[first_rest + c + i + j] = z[i + j] * unit.size;
              z[i + j] = real ? z[i + j] : -INFINITY;
            }
          }
          float most[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) most[i] = z[i];
          const float2 old = run[c + lane];
          const float top = fmaxf(old.x, over_lanes<true>(most, lane));
          const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int i = 0; i < 32; ++i) z[i] = mma::exp2_fast((z[i] - __shfl_sync(0xffffffffu, base, i)) * unit.rate);
          const float sum = over_lanes<false>(z, lane);
          run[c + lane] = make_float2(top, (old.y == 0.f ? 0.f : old.y * weight_of(old.x, top, unit.rate)) + sum);
        };
        if (kLong) {
          float sums[kBothMost / 64][32];
          add_up(sums, p.rest_cols, p.rest_cols);
#pragma unroll
          for (int r = 0; r < kBothMost / 64; ++r) {
            const int c = (2 * r + half) * 32;
            if (c < p.rest_cols && ok) take(sums[r], c);
          }
        } else {
          if (!p.both) {           // (else it has been waited for)
            ok = ok && tma::mbar_wait(&bar->acc_full[buf], use & 1, p.error, 806);
            tc::fence_after_sync();
          }
          const uint32_t acc = lane_base + (p.both ? 1 : buf) * kMaxTokens;
#pragma unroll 1
          for (int c = half * 32; c < p.rest_cols && ok; c += 64) {
            float z[32];
            ld_32x32b_x32(acc + c, z);
            take(z, c);
          }
        }
      }
      if (kLong) continue;         // (given back chunk by chunk)
      tc::fence_before_sync();
      // (given back whatever happened: the issuing lane counts 256 arrivals a tile)
      tma::mbar_arrive_cluster(tma::cluster_address(tma::smem_u32(&bar->acc_empty[buf]), 0));
      ++count;
    }
    // the warps' sums of the rest, joined
    asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueThreads) : "memory");
    float2* part = p.part + (long long)p.n_tiles * first_rest + (long long)blockIdx.x * p.rest;
    for (int c = worker; c < p.rest; c += kEpilogueThreads) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, tail->run[w][c].x);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 v = tail->run[w][c];
        sum += v.y == 0.f ? 0.f : v.y * weight_of(v.x, top, unit.rate);
      }
      part[c] = make_float2(top * unit.size, sum);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tma::cluster_sync_all();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc_pair(tmem, kTmemCols);
  }
}

// 16-bit rows that TMA cannot take, copied to rows that it can: `padded` (a multiple of 8) numbers apart, zeros behind the
// K of each. A warp takes a row, a lane two neighbouring numbers at a time (they may begin at any of their own
// multiples), written as one; 151,936 rows of 1,535 take 177 us, at the rate of memory 145.
constexpr int kPadWarps = 8;
__global__ void __launch_bounds__(32 * kPadWarps)
pad_kernel(const uint16_t* __restrict__ from, long long stride, long long rows, int K, int padded, uint32_t* __restrict__ to) {
  const long long row = (long long)blockIdx.x * kPadWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const uint16_t* in = from + row * stride;
  uint32_t* out = to + row * (padded / 2);
#pragma unroll 4
  for (int c = threadIdx.x & 31; c < padded / 2; c += 32) {
    const uint32_t low = 2 * c < K ? in[2 * c] : 0, high = 2 * c + 1 < K ? in[2 * c + 1] : 0;
    out[c] = low | high << 16;
  }
}

// The product and its softmax in 32 bits where the head's rows do not begin at multiples of 16 bytes, which TMA cannot
// take: plain multiply-adds. A block takes 8 TM rows of x and kCols rows of the head, K in steps of 16
// through a ring copied with cp.async; thread (ty, tx) of 8 x 16 has rows ty + 8 i and columns tx + 16 j, so that
// the column's threads, and with them the order of a row's sums, are the same for every TM. Two multiply-adds an
// instruction: a sum is one over the even k's and one over the odd ones, whose operands lie side by side as they
// are read. Bound by reads of shared memory (16 bytes a lane take four cycles whatever the lanes share) and copies of
// four bytes beside the multiply-adds: 64 rows of 1,023 over 32,768 take 142 us, 58 us at the multiply-adds' rate.
constexpr int kCols = 128, kF32Threads = 128, kF32K = 16, kF32Stages = 4, kLd = kF32K + 4;

// d += a * b in both halves
__device__ __forceinline__ void fma_pair(uint64_t& d, uint64_t a, uint64_t b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(b));
}

__device__ __forceinline__ void copy_f32(uint32_t dst, const float* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(real ? 4 : 0) : "memory");
}

template <int TM>
__global__ void __launch_bounds__(kF32Threads, TM == 8 ? 2 : 3)
f32_kernel(const float* __restrict__ x, long long x_stride, const float* __restrict__ head, int M, int N, int K,
           int m_tiles, const int32_t* __restrict__ targets, float2* __restrict__ part,
           float* __restrict__ mine, const Shape form) {
  constexpr int kRows = 8 * TM, kStages = kF32Stages;
  extern __shared__ __align__(16) float ring[];            // [stages][kRows + kCols][kLd]
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int m0 = blockIdx.x % m_tiles * kRows, piece = blockIdx.x / m_tiles;      // tokens fastest
  const long long n0 = (long long)piece * kCols;
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  const int steps = (K + kF32K - 1) / kF32K;
  // a thread copies one place of K (of a step) in rows kAt, kAt + kStep, ... of x and of the head
  constexpr int kStep = kF32Threads / kF32K;
  const int kc = threadIdx.x % kF32K, row = threadIdx.x / kF32K;
  const float* from_x = x + (m0 + row) * x_stride + kc;
  const float* from_w = head + (n0 + row) * K + kc;
  const uint32_t to0 = base + (row * kLd + kc) * 4;
  auto fill = [&](int step) {
    const uint32_t to = to0 + (step % kStages) * ((kRows + kCols) * kLd * 4);
    const bool in_k = step * kF32K + kc < K;
#pragma unroll
    for (int r = 0; r < kRows; r += kStep) {
      const bool real = in_k && m0 + row + r < M;
      copy_f32(to + r * kLd * 4, real ? from_x + r * x_stride : head, real);
    }
#pragma unroll
    for (int r = 0; r < kCols; r += kStep) {
      const bool real = in_k && n0 + row + r < N;
      copy_f32(to + (kRows + r) * kLd * 4, real ? from_w + (long long)r * K : head, real);
    }
    from_x += kF32K;
    from_w += kF32K;
  };
  uint64_t sums[TM][8];              // (sum over even k, sum over odd k)
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[i][j] = 0;
  for (int s = 0; s < kStages - 1; ++s) {
    if (s < steps) fill(s);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  for (int step = 0; step < steps; ++step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncthreads();
    if (step + kStages - 1 < steps) fill(step + kStages - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const float* xs = ring + (step % kStages) * (kRows + kCols) * kLd;
    const float* ws = xs + kRows * kLd;
#pragma unroll
    for (int k = 0; k < kF32K; k += 4) {
      ulonglong2 a[TM], w[8];
#pragma unroll
      for (int i = 0; i < TM; ++i) a[i] = *reinterpret_cast<const ulonglong2*>(xs + (ty + 8 * i) * kLd + k);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = *reinterpret_cast<const ulonglong2*>(ws + (tx + 16 * j) * kLd + k);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) fma_pair(sums[i][j], a[i].x, w[j].x);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) fma_pair(sums[i][j], a[i].y, w[j].y);
    }
  }
  float acc[TM][8];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      acc[i][j] = __uint_as_float(static_cast<uint32_t>(sums[i][j])) + __uint_as_float(static_cast<uint32_t>(sums[i][j] >> 32));
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + ty + 8 * i;
    const int target = m < M ? targets[m] : -1;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long v = n0 + tx + 16 * j;
      float z = -INFINITY;
      if (v < N) {
        z = acc[i][j];
        if (form.bias) z += bias_at(form, static_cast<int>(v));
        z *= form.scale;
        if (form.cap > 0.f) z = form.cap * tanhf(z * form.over_cap);
        if (v == target) mine[m] = z;
      }
      acc[i][j] = z;
      top = fmaxf(top, z);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float from = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n0 + tx + 16 * j < N) sum += expf(acc[i][j] - from);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (tx == 0 && m < M) part[(long long)piece * M + m] = make_float2(top, sum);
  }
}

template <int TM>
int launch_f32(const float* x, long long x_stride, const float* head, int M, int N, int K, const int32_t* targets,
               float2* part, float* mine, const Shape& form, cudaStream_t stream) {
  constexpr int kSmem = kF32Stages * (8 * TM + kCols) * kLd * 4;
  static PerDeviceOnce configured;
  if (configured.needs()) {
    const cudaError_t e = cudaFuncSetAttribute(f32_kernel<TM>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return (int)e;
    configured.done();
  }
  const long long m_tiles = (M + 8 * TM - 1) / (8 * TM), pieces = ((long long)N + kCols - 1) / kCols;
  if (m_tiles * pieces > 0x7fffffffLL) return cudaErrorInvalidValue;
  return launch_ordered(f32_kernel<TM>, dim3((unsigned)(m_tiles * pieces)), dim3(kF32Threads), kSmem, stream, x,
                        x_stride, head, M, N, K, (int)m_tiles, targets, part, mine, form);
}

// ---- 32 bits on the tensor cores ----------------------------------------------------------------
// A number of 24 bits is the sum of three bfloat16 numbers h + m + l, each the upper half of what the ones before
// leave (exact: 8 bits each, cut off); a product is h h' + (h m' + m h') + (h l' + m m' + l h'), and what is left out
// is below 2^-21 of it. The six are products on the tensor cores. These cut where they add, always the same way: sums
// of h h' are taken off them every kChunk steps and added up in fp32 by the epilogue. The largest error over 64 tokens
// and K = 1,536 is 1.6e-6 to 2.6e-6 so (every second step; every fourth: 3.1e-6 and 4 % less time), 1.2e-5 with one
// sum for all of K, 3.5e-6 to 6.9e-6 with the library's product. Sums that are NaN are taken again with
// plain multiply-adds: the parts of an infinity are infinity and NaN.
// A block takes a tile of `rows` rows of the head, on the lanes of tensor memory, against up to 96 tokens, its columns:
//   warp 0       TMA: the head as it is (boxes of 32 floats) into a ring,
//   warp 1       tensor memory, and the products,
//   warp 2       TMA: the tokens' numbers in three, which `split_kernel` has left in a scratch,
//   warp 3       has waited for those before the warp that issues looks,
//   warps 4-15   epilogue: for every 32 lanes a warp for each 32 tokens. Sums stay in registers, so that the next
//                tile's products run under the softmax,
//   warps 16-23  the head's numbers in three, four warps a step in turns: a thread takes a row's floats and writes them
//                to tensor memory, as the products' left operand (no second trip through shared memory, which their
//                right one fills).
// The right operand is h', m', l' side by side, or two of them (a product's width is 256 at most): three products or
// four a 16 of K instead of six, since issuing one takes some 55 cycles whatever its width. The height of a tile
// depends on the vocabulary and the device alone and every tile leaves a partial: a row's sums are the same to the bit
// whatever rows are beside it.
// Measured: 64 tokens, K 1,024, 32,768 rows 44 us (21 at the memory's rate, 15 the products at the tensor cores'; the
// multiply-adds below took 131); 64, 1,536, 151,936 240 us (145, 107); 185, 1,704, 94,657 334 us (100, 214; 1,480). A
// step of 64 takes 0.9 to 1.2 us, of which the floats' arrival is 0.7: cutting them in three and the products, each a
// chain of waits, share what is left (without the products 0.86, without the cutting 0.9).
constexpr int kSplitThreads = 768, kSplitTokens = 96, kSplitEpilogue = 4 * kSplitTokens, kSplitRaw = BM * BK * 4;
constexpr int kSplitRawMost = 6, kSplitXMost = 4, kSplitConverters = 4, kSplitMerged = 64, kChunk = 2;
constexpr uint32_t kSplitA = 3 * BK / 2;         // columns of tensor memory for a step's left operands
constexpr uint32_t kSplitAcc = 2 * kSplitA;      // where the sums begin
static_assert(kSplitAcc + 3 * kSplitTokens <= kTmemCols && 3 * kSplitMerged <= 256, "tensor memory, and a product's width");

struct SplitParams {
  int M, N, K;
  int m_tiles, cols;         // tiles of `cols` tokens (a multiple of 32)
  int rows, n_tiles;         // tiles of `rows` rows of the head
  int raw_stages, x_stages;
  const float *x, *head;     // as they are, for sums that are NaN in three parts
  long long x_stride;
  const int32_t* targets;
  float2* part;              // [n_tiles][M]
  float* mine;
  Shape form;
  int* error;
};

struct SplitTail {
  uint64_t raw_full[kSplitRawMost], raw_empty[kSplitRawMost], x_full[kSplitXMost];
  uint64_t a_full[2], done[kSplitXMost], acc_full, acc_empty;
  uint32_t tmem;
  alignas(16) int32_t target[2][kSplitTokens];
  float2 share[2][4][kSplitTokens];
};

// A place in a ring and the parity of its use.
struct Place {
  int at = 0, phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++at == stages) {
      at = 0;
      phase ^= 1;
    }
  }
};

// The upper halves of two numbers side by side, and what they leave.
__device__ __forceinline__ uint32_t cut_two(float& a, float& b) {
  const uint32_t upper = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
  mma::add2(a, b, -__uint_as_float(upper << 16), -__uint_as_float(upper & 0xffff0000u));
  return upper;
}

// x [M, K] in three: out [3][rows][padded], zeros behind M and K; a thread takes four numbers.
__global__ void __launch_bounds__(256)
split_kernel(const float* x, long long x_stride, int M, int K, int rows, int padded, int wide,
             uint2* __restrict__ out) {
  wait_for_previous_kernel();
  let_next_kernel_start();       // (in this order: the next one reads the head before it waits for this one)
  const int per = padded / 4;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x, all = (long long)rows * per;
  if (i >= all) return;
  const int k = static_cast<int>(i % per) * 4;
  const long long m = i / per;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (k < K && m < M) {      // (K is a multiple of four)
    const float* from = x + m * x_stride + k;
    if (wide) {
      read4(from, v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = from[j];
    }
  }
#pragma unroll
  for (int piece = 0; piece < 3; ++piece) {
    const uint32_t a = cut_two(v[0], v[1]);
    out[piece * all + i] = make_uint2(a, cut_two(v[2], v[3]));
  }
}

// A row's (maximum, sum) over a warp's rows of the head, from plain multiply-adds: for sums that came out NaN, since the
// three parts of an infinity are infinity and NaN. A row that has a NaN of its own, which all lanes look for together,
// keeps it. `target`: the row's; `v`: the lane's token, of those that are `real`.
__device__ __noinline__ float2 plain_row(const SplitParams* p, int m, int target, int v, bool real) {
  const float* x = p->x + m * p->x_stride;
  bool none = true;
  for (int k = threadIdx.x & 31; k < p->K; k += 32) none &= x[k] == x[k];
  if (!__all_sync(0xffffffffu, none)) return make_float2(-INFINITY, NAN);
  float z = -INFINITY;
  if (real) {
    const float* w = p->head + (long long)v * p->K;
    z = 0.f;
    for (int k = 0; k < p->K; ++k) z = fmaf(x[k], w[k], z);
    if (p->form.bias) z += bias_at(p->form, v);
    z *= p->form.scale;
    if (p->form.cap > 0.f) z = p->form.cap * tanhf(z * p->form.over_cap);
    if (v == target) p->mine[m] = z;
  }
  const float top = warp_max(z);
  return make_float2(top, warp_sum(expf(z - (top == -INFINITY ? 0.f : top))));
}

// 16 columns of this warp's 32 lanes are written (no wait).
__device__ __forceinline__ void put_x16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

__global__ void __launch_bounds__(kSplitThreads, 1)
split_logprob_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                     const __grid_constant__ SplitParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* raw = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* xs = raw + p.raw_stages * kSplitRaw;
  const int x_piece = p.cols * BK * 2, x_bytes = 3 * x_piece;
  SplitTail* tail = reinterpret_cast<SplitTail*>(xs + p.x_stages * x_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total = p.m_tiles * p.n_tiles, n_kb = (p.K + BK - 1) / BK;
  const long long steps = ((long long)total - blockIdx.x + gridDim.x - 1) / gridDim.x * n_kb;   // of this block

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSplitRawMost; ++s) {
      tma::mbar_init(&tail->raw_full[s], 1);
      tma::mbar_init(&tail->raw_empty[s], kSplitConverters);
    }
    for (int s = 0; s < kSplitXMost; ++s) {
      tma::mbar_init(&tail->x_full[s], 1);
      tma::mbar_init(&tail->done[s], 1);
    }
    for (int i = 0; i < 2; ++i) tma::mbar_init(&tail->a_full[i], kSplitConverters + 1);
    tma::mbar_init(&tail->acc_full, 1);
    tma::mbar_init(&tail->acc_empty, kSplitEpilogue);
    tma::fence_barrier_init();
  }
  if (warp == 1) tc::tmem_alloc(&tail->tmem, kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tail->tmem, 0);     // (known to be the warp's own)
  let_next_kernel_start();       // (with its shared and tensor memory in hand)
  // (what comes before `split_kernel` is done once that one lets this one start; only the warp that reads what it
  // writes waits for it, and all others wait for that warp before they write)

  if (warp == 0 || warp == 2) {
    // ---- TMA: the head's rows, or the tokens' -------------------------------------------------
    if (lane == 0) {
      const bool head = warp == 0;
      const CUtensorMap* map = head ? &w_map : &x_map;
      uint64_t *full = head ? tail->raw_full : tail->x_full, *empty = head ? tail->raw_empty : tail->done;
      const int stages = head ? p.raw_stages : p.x_stages;
      tma::prefetch_map(map);
      if (!head) wait_for_previous_kernel();
      Place place;
      long long issued = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
        const int row = head ? tile / p.m_tiles * p.rows : tile % p.m_tiles * p.cols;
        for (int kb = 0; kb < n_kb; ++kb) {
          ok = tma::mbar_wait(&empty[place.at], place.phase ^ 1, p.error, 811);
          if (!ok) break;
          uint64_t* bar = &full[place.at];
          if (head) {
            // (the floats as pairs of 16-bit numbers, 64 to a box)
            uint8_t* dst = raw + place.at * kSplitRaw;
            tma::mbar_expect_tx(bar, 2 * p.rows * BK * 2);
            tma::load_2d(dst, map, kb * 2 * BK, row, bar);
            tma::load_2d(dst + kSplitRaw / 2, map, kb * 2 * BK + BK, row, bar);
          } else {
            uint8_t* dst = xs + place.at * x_bytes;
            tma::mbar_expect_tx(bar, x_bytes);
            for (int piece = 0; piece < 3; ++piece)
              tma::load_2d(dst + piece * x_piece, map, kb * BK, piece * p.m_tiles * p.cols + row, bar);
          }
          ++issued;
          place.next(stages);
        }
      }
      // before this block may leave: what was asked for has arrived
      for (long long i = issued > stages ? issued - stages : 0; i < issued; ++i)
        if (!tma::mbar_wait(&full[i % stages], (i / stages) & 1, p.error, 812)) break;
    }
  } else if (warp == 1) {
    // ---- products: the whole warp walks and one lane issues, and no turn of the loops depends on what a lane saw, so
    // that the operands stay in uniform registers, which the instruction reads --------------------------------
    const uint32_t one = tc::idesc_bf16_f32(BM, p.cols), two = tc::idesc_bf16_f32(BM, 2 * p.cols);
    const uint32_t three = tc::idesc_bf16_f32(BM, 3 * p.cols);
    const bool merged = p.cols <= kSplitMerged;
    const uint32_t elected = tc::elect_lane();
    // columns: h h' | h m' + m h' | h l' + m m' + l h'
    const uint32_t s0 = tmem + kSplitAcc, s1 = s0 + p.cols, s2 = s1 + p.cols;
    const uint64_t x0 = tc::smem_desc_k_major_sw128(tma::smem_u32(xs));
    Place x, a, acc;
    bool ok = true;
    for (int tile = blockIdx.x; tile < total; tile += gridDim.x) {
      for (int kb = 0; kb < n_kb; ++kb) {
        ok = ok && tma::mbar_wait(&tail->a_full[a.at], a.phase, p.error, 815) &&
             (kb % kChunk || tma::mbar_wait(&tail->acc_empty, acc.phase ^ 1, p.error, 813));
        __syncwarp();
        tc::fence_after_sync();
        const uint32_t go = elected && ok;
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) {
          const uint32_t h = tmem + a.at * kSplitA + k * 8, m = h + BK / 2, l = m + BK / 2;
          // (descriptors count 16 bytes)
          const uint64_t xh = x0 + ((x.at * x_bytes + k * 32) >> 4), xm = xh + (x_piece >> 4);
          const bool begun = kb % kChunk || k, others = kb || k;      // h h' so far, and the others
          // (the order of what adds up in a column is the same either way)
          if (merged && begun == others) {
            tc::mma_ts_if(go, s0, h, xh, three, begun);
          } else {
            tc::mma_ts_if(go, s0, h, xh, one, begun);
            tc::mma_ts_if(go, s1, h, xm, two, others);
          }
          tc::mma_ts_if(go, s1, m, xh, two, true);
          tc::mma_ts_if(go, s2, l, xh, one, true);
        }
        tc::commit_if(go, &tail->done[x.at]);
        if (kb % kChunk == kChunk - 1 || kb + 1 == n_kb) {
          tc::commit_if(go, &tail->acc_full);
          acc.next(1);
        }
        x.next(p.x_stages);
        a.next(2);
      }
    }
  } else if (warp == 3) {
    // ---- the tokens' numbers have arrived (the warp that issues has no time to wait for more than one barrier) ------
    if (lane == 0) {
      Place x, a, free;          // free: the step before the last one's, whose place in `a` a step takes
      bool ok = true;
      for (long long step = 0; step < steps && ok; ++step) {
        if (step >= 2) {
          ok = tma::mbar_wait(&tail->done[free.at], free.phase, p.error, 819);
          free.next(p.x_stages);
        }
        ok = ok && tma::mbar_wait(&tail->x_full[x.at], x.phase, p.error, 814);
        if (ok) tma::mbar_arrive(&tail->a_full[a.at]);
        x.next(p.x_stages);
        a.next(2);
      }
    }
  } else if (warp >= 16) {
    // ---- the head's numbers in three ------------------------------------------------------------
    const int quarter = warp & 3, row = quarter * 32 + lane, turn = (warp - 16) >> 2;
    const uint32_t to = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + turn * kSplitA;
    Place r, free;
    if (turn) {
      r.next(p.raw_stages);
      free.next(p.x_stages);
    }
    bool ok = true;
    for (long long step = turn; step < steps; step += 2) {
      ok = __all_sync(0xffffffffu, tma::mbar_wait(&tail->raw_full[r.at], r.phase, p.error, 816));
      if (!ok) break;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint8_t* from = raw + r.at * kSplitRaw + half * (kSplitRaw / 2) + row * 128;
        float v[32];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float4 f = *reinterpret_cast<const float4*>(from + ((c ^ (row & 7)) << 4));
          v[4 * c] = f.x; v[4 * c + 1] = f.y; v[4 * c + 2] = f.z; v[4 * c + 3] = f.w;
        }
        if (half) {
          __syncwarp();
          if (lane == 0) tma::mbar_arrive(&tail->raw_empty[r.at]);
        } else if (step >= 2) {
          ok = __all_sync(0xffffffffu, tma::mbar_wait(&tail->done[free.at], free.phase, p.error, 817));
          if (!ok) break;
          free.next(p.x_stages);
          free.next(p.x_stages);
          tc::fence_after_sync();
        }
#pragma unroll
        for (int piece = 0; piece < 3; ++piece) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = cut_two(v[2 * i], v[2 * i + 1]);
          put_x16(to + piece * (BK / 2) + half * 16, w);
        }
      }
      if (!ok) break;
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tma::mbar_arrive(&tail->a_full[turn]);
      r.next(p.raw_stages);
      r.next(p.raw_stages);
    }
  } else if (warp >= 4) {
    // ---- epilogue -------------------------------------------------------------------------------
    const int quarter = warp & 3, thread = quarter * 32 + lane, worker = threadIdx.x - 4 * 32;
    const int c = (warp - 4) / 4 * 32;         // this warp's tokens of a tile
    const bool mine = c < p.cols;
    const uint32_t sums = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + kSplitAcc + c;
    Place acc, turn;
    bool ok = true;
    for (int tile = blockIdx.x; tile < total; tile += gridDim.x) {
      const int m0 = tile % p.m_tiles * p.cols, n_tile = tile / p.m_tiles;
      const int v = n_tile * p.rows + thread;
      const bool real = thread < p.rows && v < p.N;
      const bool token = worker < p.cols && m0 + worker < p.M;
      int32_t* target = tail->target[turn.at];
      if (worker < kSplitTokens) target[worker] = token ? p.targets[m0 + worker] : -1;
      const float bias = p.form.bias && real ? bias_at(p.form, v) : 0.f;
      asm volatile("bar.sync 1, %0;" ::"n"(kSplitEpilogue) : "memory");
      float z[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) z[j] = 0.f;
      for (int kb = 0; kb < n_kb; kb += kChunk) {
        ok = __all_sync(0xffffffffu, ok && tma::mbar_wait(&tail->acc_full, acc.phase, p.error, 818));
        tc::fence_after_sync();
        if (mine && ok) {
#pragma unroll 1
          for (int part = kb + kChunk < n_kb ? 0 : 2; part >= 0; --part) {      // (the largest last)
            float some[32];
            ld_32x32b_x32(sums + part * p.cols, some);
#pragma unroll
            for (int j = 0; j < 32; j += 2) mma::add2(z[j], z[j + 1], some[j], some[j + 1]);
          }
        }
        tc::fence_before_sync();
        tma::mbar_arrive(&tail->acc_empty);
        acc.next(1);
      }
      if (mine && ok) {
        if (p.form.bias) {
#pragma unroll
          for (int j = 0; j < 32; ++j) z[j] += bias;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] *= p.form.scale;
        if (p.form.cap > 0.f) {
#pragma unroll
          for (int j = 0; j < 32; ++j) z[j] = p.form.cap * tanhf(z[j] * p.form.over_cap);
        }
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const int4 t = *reinterpret_cast<const int4*>(&target[c + j]);
          const int of[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (of[q] == v && real) p.mine[m0 + c + j + q] = z[j + q];
            z[j + q] = real ? z[j + q] : -INFINITY;
          }
        }
        float most[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) most[j] = z[j];
        const float top = over_lanes<true>(most, lane);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] = expf(z[j] - __shfl_sync(0xffffffffu, base, j));
        float2 share = make_float2(top, over_lanes<false>(z, lane));
        for (unsigned odd = __ballot_sync(0xffffffffu, share.y != share.y); odd; odd &= odd - 1) {
          const int j = __ffs(odd) - 1;
          if (m0 + c + j >= p.M) continue;
          const float2 plain = plain_row(&p, m0 + c + j, target[c + j], v, real);
          if (lane == j) share = plain;
        }
        tail->share[turn.at][quarter][c + lane] = share;
      }
      // (what a tile leaves in shared memory stays until the one after the next, past the next one's barriers)
      asm volatile("bar.sync 1, %0;" ::"n"(kSplitEpilogue) : "memory");
      if (token && ok) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) top = fmaxf(top, tail->share[turn.at][q][worker].x);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 other = tail->share[turn.at][q][worker];
          sum += other.y == 0.f ? 0.f : other.y * expf(other.x - top);
        }
        p.part[(long long)n_tile * p.M + m0 + worker] = make_float2(top, sum);
      }
      turn.next(2);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

// lse and log-probability of every row from its partials: rows below `full` have `pieces` of them, [pieces][full],
// the others `rest_pieces`, [rest_pieces][M - full] behind them. A block has 32 rows, all of one kind; a warp takes
// every 32nd piece of all of them (lane = row: neighbouring rows' partials are neighbours in memory).
constexpr int kJoinWarps = 32;
__global__ void __launch_bounds__(32 * kJoinWarps)
join_kernel(const float2* part, const float* mine, const int32_t* targets,
            float* __restrict__ logprob, float* __restrict__ lse, int M, int N, int full, int pieces,
            int rest_pieces) {
  constexpr int kRound = 8;
  let_next_kernel_start();
  wait_for_previous_kernel();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m = blockIdx.x * 32 + lane;
  const bool in_full = m < full;               // (full is a multiple of 256, past M where the last tile is not, or M)
  const int width = in_full ? full : M - full, count = in_full ? pieces : rest_pieces;
  const float2* mine_part = part + (in_full ? (long long)m : (long long)pieces * full + m - full);
  float top = -INFINITY, sum = 0.f;
  if (m < M)
    for (int s0 = warp; s0 < count; s0 += kJoinWarps * kRound) {
      float2 v[kRound];
#pragma unroll
      for (int i = 0; i < kRound; ++i) {
        const int s = s0 + i * kJoinWarps;
        v[i] = s < count ? mine_part[(long long)s * width] : make_float2(-INFINITY, 0.f);
      }
      float big = top;
#pragma unroll
      for (int i = 0; i < kRound; ++i) big = fmaxf(big, v[i].x);
      sum = sum == 0.f ? 0.f : sum * expf(top - big);
      top = big;
#pragma unroll
      for (int i = 0; i < kRound; ++i) sum += v[i].y == 0.f ? 0.f : v[i].y * expf(v[i].x - top);
    }
  __shared__ float2 all[kJoinWarps][32];
  all[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (warp || m >= M) return;
#pragma unroll
  for (int w = 1; w < kJoinWarps; ++w) top = fmaxf(top, all[w][lane].x);
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w)
    sum += all[w][lane].y == 0.f ? 0.f : all[w][lane].y * expf(all[w][lane].x - top);
  const float total = sum == 0.f ? -INFINITY : top + logf(sum);
  const int target = targets[m];
  lse[m] = total;
  // (a row that asks for nothing: 0; a target that is no token: NaN)
  logprob[m] = target < 0 ? 0.f : target < N ? mine[m] - total : __int_as_float(0x7fc00000);
}

__device__ int g_error;

// Where the current device has it (asked once a device).
int* error_word() {
  static int* known[PerDeviceOnce::kDevices] = {};
  const int device = PerDeviceOnce::current();
  if (device < 0 || device >= PerDeviceOnce::kDevices) return nullptr;
  if (!known[device]) {
    void* at = nullptr;
    if (cudaGetSymbolAddress(&at, g_error) != cudaSuccess) return nullptr;
    known[device] = static_cast<int*>(at);
  }
  return known[device];
}

int resident_pairs() {
  static int known[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 0;
  if (known[device]) return known[device] - 1;
  int clusters = 0;
  auto allow = [](auto kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost) == cudaSuccess;
  };
  if (allow(logprob_kernel<true, false, false>) && allow(logprob_kernel<false, false, false>) &&
      allow(logprob_kernel<false, true, false>) && allow(logprob_kernel<true, false, true>) &&
      allow(logprob_kernel<false, false, true>) && allow(logprob_kernel<false, true, true>)) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(2 * sm_count());
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kSmemMost;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&clusters, logprob_kernel<true, false, true>, &config) != cudaSuccess) clusters = 0;
    cudaGetLastError();
  }
  known[device] = clusters + 1;
  return clusters;
}

// Whether one tile takes the 256 tokens and the rest of M tokens.
bool both_of(int M, int K, int full) { return full == 1 && M > kMaxTokens && K <= kLongK; }

// The join of `pieces` partials [pieces][full] of rows below `full` and `rest_pieces` [.][M - full] of the others, which
// lie behind them (full: a multiple of 256, perhaps past M, or M).
int join(const float* part, const float* mine, const int32_t* targets, float* logprob, float* lse, int M, int N,
         int full, int pieces, int rest_pieces, cudaStream_t stream) {
  return launch_overlapped(join_kernel, dim3((M + 31) / 32), dim3(32 * kJoinWarps), 0, stream, 1,
                           reinterpret_cast<const float2*>(part), mine, targets, logprob, lse, M, N, full, pieces,
                           rest_pieces);
}

Shape shape_of(const void* bias, int bias_bf16, float scale, float cap) {
  Shape f;
  f.bias = bias; f.bias_bf16 = bias_bf16; f.scale = scale; f.cap = cap;
  f.over_cap = cap > 0.f ? 1.f / cap : 0.f;
  return f;
}

}  // namespace

// Rows of the head a piece of the 32-bit kernel has.
SAKV_EXPORT int sakv_logprob_f32_columns() { return kCols; }

// The log-probabilities of x [M, K] (rows `x_stride` apart) against the head [N, K] in float32: scratch part
// [ceil(N / 128)][M] pairs, mine [M].
SAKV_EXPORT int sakv_logprob_f32(const float* x, long long x_stride, const float* head, int M, int N, int K,
                                 const int32_t* targets, float* part, float* mine, const void* bias, int bias_bf16,
                                 float scale, float cap, float* logprob, float* lse, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || x_stride < K || M > 0x7fffffff - 64 || !(cap >= 0.f)) return cudaErrorInvalidValue;
  const Shape form = shape_of(bias, bias_bf16, scale, cap);
  float2* to = reinterpret_cast<float2*>(part);
#define SAKV_F32(TM) launch_f32<TM>(x, x_stride, head, M, N, K, targets, to, mine, form, stream)
  const int e = M <= 8 ? SAKV_F32(1) : M <= 16 ? SAKV_F32(2) : M <= 32 ? SAKV_F32(4) : SAKV_F32(8);
#undef SAKV_F32
  return e ? e : join(part, mine, targets, logprob, lse, M, N, M, (N + kCols - 1) / kCols, 0, stream);
}

// Pairs of SMs that can hold the tensor-core kernel at one time (0: it cannot run here).
SAKV_EXPORT int sakv_logprob_resident() { return resident_pairs(); }

// How M tokens against N rows of K numbers of the head are cut, for `pairs` pairs of SMs:
// shape = {tiles of 256 tokens, rows of the head a block takes of a tile, tiles of the head, pairs launched}.
// A block takes 128 rows of the head, or fewer where that makes the last round of tiles fuller. A few tokens: bound
// by the head's bytes, so any height serves, the one that gives every block the same number of rows in all. More:
// the height is a multiple of 16 (the products' width, two blocks' rows, is one of 32), and a round of tiles costs
// what its operands' rows take from L2.
SAKV_EXPORT int sakv_logprob_shape(int M, int N, int K, int pairs, int* shape) {
  // (row numbers of tiles that reach past the head are 32-bit numbers)
  if (M <= 0 || N <= 0 || K <= 0 || pairs <= 0 || pairs > (1 << 16) || N > 0x7fffffff - 4 * BM * pairs ||
      M > 0x7fffffff - 512)
    return cudaErrorInvalidValue;
  const int most = M > kMaxTokens && M < 2 * kMaxTokens && K <= kLongK ? kBothMost : kRestMost;
  const int full = M / kMaxTokens + (M % kMaxTokens > most ? 1 : 0);
  const int per = both_of(M, K, full) ? 1 : full + (M > full * kMaxTokens);
  int rows = BM;
  if (full == 0) {
    const long long rounds = (N + 2LL * BM * pairs - 1) / (2 * BM * pairs);
    rows = (int)((N + 2 * pairs * rounds - 1) / (2 * pairs * rounds));
  } else {
    const int beside = both_of(M, K, full) ? (M - kMaxTokens + 31) / 32 * 16 : 0;
    long long best = -1;
    for (int r = BM; r >= 96; r -= 16) {
      const long long tiles = (N + 2LL * r - 1) / (2 * r) * per;
      const long long cost = (tiles + pairs - 1) / pairs * (r + BM + beside);
      if (best < 0 || cost < best) {
        best = cost;
        rows = r;
      }
    }
  }
  const long long n_tiles = (N + 2LL * rows - 1) / (2 * rows);
  if (n_tiles * per > 0x3fffffffLL) return cudaErrorInvalidValue;
  shape[0] = full;
  shape[1] = rows;
  shape[2] = (int)n_tiles;
  shape[3] = n_tiles * per < pairs ? (int)(n_tiles * per) : pairs;
  return 0;
}

// A TMA descriptor of a row-major bf16 matrix read in boxes of [box_rows, 64 columns].
static int logprob_map(CUtensorMap* map, const void* base, long long rows, long long cols, long long row_stride,
                       int box_rows) {
  if (rows <= 0 || cols <= 0 || rows > 0x7fffffffLL || (cols % 8) || (row_stride % 8) || row_stride < cols)
    return cudaErrorInvalidValue;
  return tma::make_map_bf16_2d(map, base, (uint64_t)rows, (uint64_t)cols, (uint64_t)row_stride * 2,
                               (uint32_t)box_rows, BK);
}

// Rows of the head in a tile of the 32-bit tensor-core kernel for a vocabulary of N: the height that a device of so many
// SMs gets through in the fewest rows, whatever the tokens.
SAKV_EXPORT int sakv_logprob_split_rows(int N, int sms) {
  if (N <= 0 || sms <= 0) return 0;
  long long best = -1;
  int rows = BM;
  for (int r = BM; r >= 104; r -= 8) {
    const long long tiles = ((long long)N + r - 1) / r, cost = (tiles + sms - 1) / sms * r;
    if (best < 0 || cost < best) {
      best = cost;
      rows = r;
    }
  }
  return rows;
}

// M tokens rounded up to whole tiles of it (0: too many): as few tiles as there can be, of equal width.
SAKV_EXPORT int sakv_logprob_split_tokens(int M) {
  if (M <= 0) return 0;
  const long long tiles = ((long long)M + kSplitTokens - 1) / kSplitTokens;
  const long long rows = ((M + tiles - 1) / tiles + 31) / 32 * 32 * tiles;
  return rows <= 0x7fffffff / 3 ? (int)rows : 0;
}

// The same as sakv_logprob_f32 on the tensor cores, for heads whose rows begin at multiples of 16 bytes: tiles of `rows`
// rows (sakv_logprob_split_rows), scratch part [ceil(N / rows)][M] pairs, mine [M], split [3][M rounded
// up to sakv_logprob_split_tokens][K rounded up to 8] of 16 bits at a multiple of 16 bytes.
SAKV_EXPORT int sakv_logprob_split(const float* x, long long x_stride, const float* head, int M, int N, int K, int rows,
                                   const int32_t* targets, float* part, float* mine, void* split, const void* bias,
                                   int bias_bf16, float scale, float cap, float* logprob, float* lse,
                                   cudaStream_t stream) {
  const int sms = sm_count();
  if (M <= 0 || N <= 0 || K <= 0 || K % 4 || x_stride < K || !(cap >= 0.f) || !sakv_logprob_split_tokens(M) ||
      N > 0x7fffffff - BM || K > 0x3fffffff - BK || rows != sakv_logprob_split_rows(N, sms) || rows <= 0)
    return cudaErrorInvalidValue;
  SplitParams p;
  p.M = M; p.N = N; p.K = K;
  const int padded_rows = sakv_logprob_split_tokens(M);
  p.m_tiles = (M + kSplitTokens - 1) / kSplitTokens;
  p.cols = padded_rows / p.m_tiles;
  p.rows = rows;
  p.n_tiles = (N + rows - 1) / rows;
  if ((long long)p.m_tiles * p.n_tiles > 0x3fffffffLL) return cudaErrorInvalidValue;
  // what is left of shared memory beside up to four steps of the tokens is the head's
  const int x_bytes = 3 * p.cols * BK * 2, room = kSmemMost - 1024 - (int)sizeof(SplitTail);
  p.x_stages = p.cols <= 32 ? 4 : 3;
  p.raw_stages = (room - p.x_stages * x_bytes) / kSplitRaw;
  if (p.raw_stages > kSplitRawMost) p.raw_stages = kSplitRawMost;
  p.x = x; p.head = head; p.x_stride = x_stride;
  p.targets = targets; p.part = reinterpret_cast<float2*>(part); p.mine = mine;
  p.form = shape_of(bias, bias_bf16, scale, cap);
  p.error = error_word();
  if (!p.error || p.raw_stages < 2) return cudaErrorInvalidValue;
  const int padded = (K + 7) / 8 * 8;
  CUtensorMap w_map, x_map;
  int e = logprob_map(&w_map, head, N, 2LL * K, 2LL * K, rows);
  if (!e) e = logprob_map(&x_map, split, 3LL * padded_rows, padded, padded, p.cols);
  if (e) return e;
  const int smem = p.raw_stages * kSplitRaw + p.x_stages * x_bytes + 1024 + (int)sizeof(SplitTail);
  static PerDeviceOnce configured;
  if (configured.needs()) {
    const cudaError_t set =
        cudaFuncSetAttribute(split_logprob_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
    if (set != cudaSuccess) return (int)set;
    configured.done();
  }
  const long long quads = (long long)padded_rows * (padded / 4), blocks = (quads + 255) / 256;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const int wide = x_stride % 4 == 0 && !(reinterpret_cast<uintptr_t>(x) & 15);
  e = launch_overlapped(split_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, 1, x, x_stride, M, K, padded_rows, padded,
                        wide, reinterpret_cast<uint2*>(split));
  const int tiles = p.m_tiles * p.n_tiles;
  if (!e) e = launch_overlapped(split_logprob_kernel, dim3(tiles < sms ? tiles : sms), dim3(kSplitThreads), smem, stream, 1,
                                w_map, x_map, p);
  return e ? e : join(part, mine, targets, logprob, lse, M, N, M, p.n_tiles, 0, stream);
}

// The partials of x [M, K] against the head [N, K] in bf16 (rows of x `x_stride` apart; 16-byte aligned), cut as
// `shape` (sakv_logprob_shape) says, joined: scratch part [shape[2]][256 shape[0]] and, behind it, [2 shape[3]][M - 256
// shape[0]] pairs, mine [M].
SAKV_EXPORT int sakv_logprob_pieces(const void* x, long long x_stride, const void* head, int M, int N, int K,
                                    const int* shape, const int32_t* targets, float* part, float* mine,
                                    const void* bias, int bias_bf16, float scale, float cap, float* logprob,
                                    float* lse, cudaStream_t stream) {
  int expect[4];
  const int here = resident_pairs();
  if (K <= 0 || (K % 8) || !(cap >= 0.f)) return cudaErrorInvalidValue;
  if (here <= 0) return cudaErrorNotSupported;
  const int bad = sakv_logprob_shape(M, N, K, here, expect);
  if (bad) return bad;
  for (int i = 0; i < 4; ++i)
    if (shape[i] != expect[i]) return cudaErrorInvalidValue;
  Params p;
  p.M = M; p.N = N; p.K = K;
  p.full = shape[0]; p.w_rows = shape[1]; p.n_tiles = shape[2];
  p.rest = M > p.full * kMaxTokens ? M - p.full * kMaxTokens : 0;
  p.rest_cols = (p.rest + 31) / 32 * 32;
  p.both = both_of(M, K, p.full);
  p.stage_bytes = kWBytes + (p.full ? kXBytes : 0) + (p.full == 0 || p.both ? p.rest_cols / 2 * BK * 2 : 0);
  p.stages = kRingMost / p.stage_bytes < kMaxStages ? kRingMost / p.stage_bytes : kMaxStages;
  p.targets = targets; p.part = reinterpret_cast<float2*>(part); p.mine = mine;
  p.form = shape_of(bias, bias_bf16, scale, cap);
  p.error = error_word();
  if (!p.error) return cudaErrorInvalidValue;
  CUtensorMap x_map, rest_map, w_map;
  int e = logprob_map(&w_map, head, N, K, K, p.w_rows);
  if (!e) e = logprob_map(&x_map, x, M, K, x_stride, p.full ? BM : p.rest_cols / 2);
  if (!e && p.full && p.rest) e = logprob_map(&rest_map, x, M, K, x_stride, p.rest_cols / 2);
  else rest_map = x_map;
  if (e) return e;
  const int steps = (K + BK - 1) / BK, chunks = (K + kLongK - 1) / kLongK;
  p.chunk = (steps + chunks - 1) / chunks;
  auto kernel = chunks > 1
      ? cap > 0.f ? logprob_kernel<false, true, true>
                  : bias || scale != 1.f ? logprob_kernel<false, false, true> : logprob_kernel<true, false, true>
      : cap > 0.f ? logprob_kernel<false, true, false>
                  : bias || scale != 1.f ? logprob_kernel<false, false, false> : logprob_kernel<true, false, false>;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(2 * shape[3]);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = p.stages * p.stage_bytes + 1024 + sizeof(Tail);
  config.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 2;
  const cudaError_t launched = cudaLaunchKernelEx(&config, kernel, x_map, rest_map, w_map, p);
  if (launched != cudaSuccess) return static_cast<int>(launched);
  return join(part, mine, targets, logprob, lse, M, N, p.full * kMaxTokens, p.n_tiles, 2 * shape[3], stream);
}

// Copies of 16-bit rows (K numbers, `stride` apart) that are `padded` numbers apart at `to`, a multiple of 16 bytes.
SAKV_EXPORT int sakv_logprob_pad(const void* from, long long stride, long long rows, int K, int padded, void* to,
                                 cudaStream_t stream) {
  const long long blocks = (rows + kPadWarps - 1) / kPadWarps;
  if (rows <= 0 || K <= 0 || padded < K || padded % 8 || stride < K || blocks > 0x7fffffffLL ||
      (reinterpret_cast<uintptr_t>(from) & 1) || (reinterpret_cast<uintptr_t>(to) & 15))
    return cudaErrorInvalidValue;
  return launch_ordered(pad_kernel, dim3((unsigned)blocks), dim3(32 * kPadWarps), 0, stream,
                        reinterpret_cast<const uint16_t*>(from), stride, rows, K, padded, reinterpret_cast<uint32_t*>(to));
}

// The join of partials [pieces][M] that calls for pieces of the head have left.
SAKV_EXPORT int sakv_logprob_join(const float* part, const float* mine, const int32_t* targets, float* logprob,
                                  float* lse, int M, int N, int pieces, cudaStream_t stream) {
  if (M <= 0 || pieces < 0) return cudaErrorInvalidValue;
  return join(part, mine, targets, logprob, lse, M, N, M, pieces, 0, stream);
}

SAKV_EXPORT int sakv_logprob_error(int* value) {
  return static_cast<int>(cudaMemcpyFromSymbol(value, g_error, sizeof(int)));
}
