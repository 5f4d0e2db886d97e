// Log-probabilities of given tokens under the output head, without keeping the logits:
//
//   z_v = cap(scale (x . w_v + b_v)),   cap(z) = c tanh(z / c) where c > 0
//   lse = m + log sum_v e^(z_v - m),  m = max_v z_v;    logprob = z_target - lse
//
// The vocabulary is taken in pieces: a piece leaves (m, sum 2^(z - m)) a row, in base 2, and whoever meets the
// target's column leaves z_target; `join_kernel` merges the pieces. 2,048 tokens over 151,936 logits would be
// 1.2 GB written and read again; the pieces are 10 MB.
//
// Two ways to a piece. bfloat16 operands: tcgen05 on PAIRS of SMs (`cta_group::2`), a tile of 256 tokens x 256
// rows of the head, the softmax's sums in the epilogue, thread = token row, so that no sum crosses a thread.
//   warp 0     TMA: boxes of x [128 tokens x 64] and of the head [128 rows x 64] into a ring of six 32 KB
//              stages (each block of the pair fetches its own half of both; no multicast),
//   warp 1     tensor memory; in the pair's first block lane 0 issues the products,
//   warps 2-5  epilogue of a tile under the products of the next (two accumulators of 256 columns).
// Up to 256 tokens the head is read once and that bounds it; above, the tensor cores do.
// float32 operands (and rows that TMA cannot take): `fold_kernel` reads a piece of logits that a product of
// its own left in a scratch.
//
// Sums and maxima are fp32. Every mbarrier wait is bounded, and a pair leaves together.
// The reference keeps all logits (`src/microinfer/model.py:388-402`).
#include "common.cuh"
#include "mma.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace {

constexpr int BM = 128;                          // tokens per block
constexpr int BN = 256;                          // rows of the head a tile
constexpr int BK = 64;
constexpr int kStages = 6;
constexpr int kXBytes = BM * BK * 2;
constexpr int kWBytes = (BN / 2) * BK * 2;
constexpr int kStageBytes = kXBytes + kWBytes;
constexpr int kEpilogueThreads = 128;
constexpr int kThreads = 64 + kEpilogueThreads;
constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 256;
constexpr uint32_t kTmemCols = 512;
constexpr uint16_t kBoth = 3;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// What becomes of a product x . w before the softmax.
struct Shape {
  const void* bias;          // or null
  int bias_bf16;
  float scale;
  float cap, two_over_cap;   // 0: none; 2 log2(e) / cap
};

__device__ __forceinline__ float bias_at(const Shape& f, int v) {
  return f.bias_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(f.bias)[v])
                     : reinterpret_cast<const float*>(f.bias)[v];
}

// tanh(y) = 1 - 2 / (e^2y + 1): off by a few 2^-24 of 1, so z by a few 2^-24 of the cap
template <bool kCap>
__device__ __forceinline__ float shaped(const Shape& f, float z) {
  z *= f.scale;
  if (kCap) {
    const float y = z * f.two_over_cap;          // (kept below 2^126, where the quotient is still one; NaN stays)
    z = f.cap - __fdividef(2.f * f.cap, 1.f + mma::exp2_fast(y > 125.f ? 125.f : y));
  }
  return z;
}

struct Params {
  int M, N, K;               // tokens, vocabulary, inner size
  int m_tiles, n_tiles;
  const int32_t* targets;
  float2* part;              // [n_tiles][M]
  float* mine;               // [M]: the targets' logits
  Shape form;
  int* error;
};

struct Barriers {
  uint64_t full[kStages], empty[kStages];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem;
};

// 64 columns of a row joined to the row's running (maximum, sum) in base 2. `z` in natural units.
__device__ __forceinline__ void take_up(const float (&z)[64], float& top, float& sum) {
  float big4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 64; c += 8)
#pragma unroll
    for (int q = 0; q < 4; ++q) big4[q] = mma::max3(big4[q], z[c + 2 * q], z[c + 2 * q + 1]);
  const float big = fmaxf(fmaxf(big4[0], big4[1]), fmaxf(big4[2], big4[3])) * kLog2e;
  if (big > top) {
    sum *= mma::exp2_fast(top - big);
    top = big;
  }
  const float base = top == -INFINITY ? 0.f : top;
  float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 64; c += 2) {
    float e0, e1;
    mma::fma2(e0, e1, z[c], z[c + 1], kLog2e, -base);
    mma::add2(s4[c & 2], s4[(c & 2) + 1], mma::exp2_fast(e0), mma::exp2_fast(e1));
  }
  sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
}

// kPlain: no bias, no scale, no cap
template <bool kPlain, bool kCap>
__global__ void __launch_bounds__(kThreads, 1)
logprob_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map,
               const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Barriers* bar = reinterpret_cast<Barriers*>(smem + kStages * kStageBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tma::cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = p.m_tiles * p.n_tiles;
  const int n_kb = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
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
  const uint32_t tmem = bar->tmem;
  let_next_kernel_start();       // (with its shared and tensor memory in hand)
  wait_for_previous_kernel();

  if (warp == 0) {
    // ---- TMA: this block's tokens and its half of the tile's rows -----------------------------
    if (lane == 0) {
      tma::prefetch_map(&x_map);
      tma::prefetch_map(&w_map);
      int stage = 0, phase = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        const int m_tile = tile % p.m_tiles, n_tile = tile / p.m_tiles;     // token tiles fastest
        const int x_row = (m_tile * 2 + static_cast<int>(rank)) * BM;
        const int w_row = n_tile * BN + static_cast<int>(rank) * (BN / 2);
        for (int kb = 0; kb < n_kb; ++kb) {
          if (!tma::mbar_wait(&bar->empty[stage], phase ^ 1, p.error, 801)) {
            ok = false;
            break;
          }
          uint8_t* dst = smem + stage * kStageBytes;
          const uint32_t full = tma::cluster_address(tma::smem_u32(&bar->full[stage]), 0);
          if (rank == 0) tma::mbar_expect_tx(&bar->full[stage], 2 * kStageBytes);
          tma::load_2d_pair(dst, &x_map, kb * BK, x_row, full);
          tma::load_2d_pair(dst + kXBytes, &w_map, kb * BK, w_row, full);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // before this block may leave: every stage it filled has been given back
      for (int s = 0; s < kStages && ok; ++s) {
        ok = tma::mbar_wait(&bar->empty[stage], phase ^ 1, p.error, 805);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issue: one lane of the pair's first block ----------------------------------------
    if (rank == 0 && lane == 0) {
      constexpr uint32_t idesc = tc::idesc_bf16_f32(2 * BM, BN);
      int stage = 0, phase = 0, round = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs, ++round) {
        const int buf = round & 1;
        if (round >= 2 && !tma::mbar_wait(&bar->acc_empty[buf], ((round >> 1) - 1) & 1, p.error, 802)) break;
        for (int kb = 0; kb < n_kb && ok; ++kb) {
          if (!tma::mbar_wait(&bar->full[stage], phase, p.error, 803)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const uint32_t a = tma::smem_u32(smem + stage * kStageBytes);
          const uint32_t b = a + kXBytes;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            tc::mma_ss_pair(tmem + buf * BN, tc::smem_desc_k_major_sw128(a + k * 32),
                            tc::smem_desc_k_major_sw128(b + k * 32), idesc, kb > 0 || k > 0);
          tc::commit_pair(&bar->empty[stage], kBoth);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (ok) tc::commit_pair(&bar->acc_full[buf], kBoth);
      }
    }
  } else {
    // ---- epilogue: thread = token row -----------------------------------------------------------
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    int round = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles; tile += pairs, ++round) {
      const int m_tile = tile % p.m_tiles, n_tile = tile / p.m_tiles;
      const int buf = round & 1;
      const int m = (m_tile * 2 + static_cast<int>(rank)) * BM + row;
      const int target = m < p.M ? p.targets[m] : -1;
      ok = ok && tma::mbar_wait(&bar->acc_full[buf], (round >> 1) & 1, p.error, 804);
      tc::fence_after_sync();
      const int n0 = n_tile * BN;
      float top = -INFINITY, sum = 0.f;
      // (a warp whose rows are all beyond the last token has nothing to read)
      const bool any = (m_tile * 2 + static_cast<int>(rank)) * BM + quarter * 32 < p.M;
#pragma unroll 1
      for (int c = 0; c < BN && ok && any && n0 + c < p.N; c += 64) {
        float z[64];
        tc::ld_32x32b_x64(lane_base + buf * BN + c, z);
        if (!kPlain) {
          if (p.form.bias) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (n0 + c + i < p.N) z[i] += bias_at(p.form, n0 + c + i);
          }
#pragma unroll
          for (int i = 0; i < 64; ++i) z[i] = shaped<kCap>(p.form, z[i]);
        }
        if (n0 + c + 64 > p.N) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (n0 + c + i >= p.N) z[i] = -INFINITY;
        }
        const int at = target - (n0 + c);
        if (__any_sync(0xffffffffu, at >= 0 && at < 64)) {
          float found = 0.f;
#pragma unroll
          for (int i = 0; i < 64; ++i) found = at == i ? z[i] : found;
          if (at >= 0 && at < 64 && target < p.N) p.mine[m] = found;
        }
        take_up(z, top, sum);
      }
      if (ok && m < p.M) p.part[(long long)n_tile * p.M + m] = make_float2(top, sum);
      tc::fence_before_sync();
      // (given back whatever happened: the issuing lane counts 256 arrivals a tile)
      tma::mbar_arrive_cluster(tma::cluster_address(tma::smem_u32(&bar->acc_empty[buf]), 0));
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

// A piece of logits that lies in memory: columns [first, first + n) of the vocabulary for M rows, `ld` apart. A
// block takes kFoldColumns columns of a row and leaves their (maximum, sum); blockIdx.y counts them.
constexpr int kFoldThreads = 256, kFoldColumns = 4096;
__global__ void __launch_bounds__(kFoldThreads)
fold_kernel(const float* __restrict__ z, long long ld, int M, int n, int first, int vocab,
            const int32_t* __restrict__ targets, float2* __restrict__ part, float* __restrict__ mine,
            const Shape form) {
  const int m = blockIdx.x;
  const int begin = blockIdx.y * kFoldColumns, end = min(n, begin + kFoldColumns);
  const int target = targets[m] - first;
  const float* row = z + (long long)m * ld;
  __shared__ float scratch[kFoldThreads / 32], sums[kFoldThreads / 32];
  float v[kFoldColumns / kFoldThreads], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kFoldColumns / kFoldThreads; ++i) {
    const int c = begin + threadIdx.x + i * kFoldThreads;
    v[i] = c < end ? row[c] : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < kFoldColumns / kFoldThreads; ++i) {
    const int c = begin + threadIdx.x + i * kFoldThreads;
    if (c < end) {
      if (form.bias) v[i] += bias_at(form, first + c);
      v[i] *= form.scale;
      if (form.cap > 0.f) v[i] = form.cap * tanhf(v[i] / form.cap);
      if (c == target) mine[m] = v[i];
    }
    top = fmaxf(top, v[i]);
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < kFoldThreads / 32; ++w) top = fmaxf(top, scratch[w]);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kFoldColumns / kFoldThreads; ++i)
    if (begin + static_cast<int>(threadIdx.x) + i * kFoldThreads < end) sum += expf(v[i] - base);
  sum = warp_sum(sum);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x) return;
  sum = 0.f;
  for (int w = 0; w < kFoldThreads / 32; ++w) sum += sums[w];
  part[(long long)blockIdx.y * M + m] = make_float2(top * kLog2e, sum);
}

// lse and log-probability of every row from its `pieces` partials [pieces][M]. A block has 32 rows, a warp takes
// every eighth piece of all of them (lane = row: neighbouring rows' partials are neighbours in memory).
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(32 * kJoinWarps)
join_kernel(const float2* __restrict__ part, const float* __restrict__ mine, const int32_t* __restrict__ targets,
            float* __restrict__ logprob, float* __restrict__ lse, int M, int N, int pieces) {
  constexpr int kRound = 8;
  let_next_kernel_start();
  wait_for_previous_kernel();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m = blockIdx.x * 32 + lane;
  float top = -INFINITY, sum = 0.f;
  if (m < M)
    for (int s0 = warp; s0 < pieces; s0 += kJoinWarps * kRound) {
      float2 v[kRound];
#pragma unroll
      for (int i = 0; i < kRound; ++i) {
        const int s = s0 + i * kJoinWarps;
        v[i] = s < pieces ? part[(long long)s * M + m] : make_float2(-INFINITY, 0.f);
      }
      float big = top;
#pragma unroll
      for (int i = 0; i < kRound; ++i) big = fmaxf(big, v[i].x);
      sum = sum == 0.f ? 0.f : sum * exp2f(top - big);
      top = big;
#pragma unroll
      for (int i = 0; i < kRound; ++i) sum += v[i].y == 0.f ? 0.f : v[i].y * exp2f(v[i].x - top);
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
    sum += all[w][lane].y == 0.f ? 0.f : all[w][lane].y * exp2f(all[w][lane].x - top);
  const float total = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  const int target = targets[m];
  lse[m] = total;
  // (a row that asks for nothing: 0; a target that is no token: NaN)
  logprob[m] = target < 0 ? 0.f : target < N ? mine[m] - total : __int_as_float(0x7fc00000);
}

__device__ int g_error;

int resident_pairs() {
  static int known[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 0;
  if (known[device]) return known[device] - 1;
  int clusters = 0;
  auto allow = [](auto kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) == cudaSuccess;
  };
  if (allow(logprob_kernel<true, false>) && allow(logprob_kernel<false, false>) && allow(logprob_kernel<false, true>)) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(2 * sm_count());
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&clusters, logprob_kernel<true, false>, &config) != cudaSuccess) clusters = 0;
    cudaGetLastError();
  }
  known[device] = clusters + 1;
  return clusters;
}

Shape shape_of(const void* bias, int bias_bf16, float scale, float cap) {
  Shape f;
  f.bias = bias; f.bias_bf16 = bias_bf16; f.scale = scale; f.cap = cap;
  f.two_over_cap = cap > 0.f ? 2.f * kLog2e / cap : 0.f;
  return f;
}

}  // namespace

// Rows of the head a piece of the tensor-core kernel has, and columns a piece of the fold has.
SAKV_EXPORT int sakv_logprob_tile() { return BN; }
SAKV_EXPORT int sakv_logprob_fold_columns() { return kFoldColumns; }
// Pairs of SMs that can hold the tensor-core kernel at one time (0: it cannot run here).
SAKV_EXPORT int sakv_logprob_resident() { return resident_pairs(); }

// A TMA descriptor of a row-major bf16 matrix read in boxes of [128 rows, 64 columns].
SAKV_EXPORT int sakv_logprob_map(void* map, const void* base, long long rows, long long cols, long long row_stride) {
  if (rows <= 0 || cols <= 0 || rows > 0x7fffffffLL || (cols % 8) || (row_stride % 8) || row_stride < cols)
    return cudaErrorInvalidValue;
  return tma::make_map_bf16_2d(reinterpret_cast<CUtensorMap*>(map), base, (uint64_t)rows, (uint64_t)cols,
                               (uint64_t)row_stride * 2, BM, BK);
}

// part [ceil(N / 256)][M] and mine [M] for x [M, K] and the head [N, K] in bf16, by their tensor maps.
SAKV_EXPORT int sakv_logprob_pieces(const void* x_map, const void* w_map, int M, int N, int K,
                                    const int32_t* targets, float* part, float* mine, const void* bias,
                                    int bias_bf16, float scale, float cap, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || (K % 8) || N > 0x7fffffff - BN || M > 0x7fffffff - 2 * BM || !(cap >= 0.f))
    return cudaErrorInvalidValue;
  const int here = resident_pairs();
  if (here <= 0) return cudaErrorNotSupported;
  Params p;
  p.M = M; p.N = N; p.K = K;
  p.m_tiles = (M + 2 * BM - 1) / (2 * BM);
  p.n_tiles = (N + BN - 1) / BN;
  if ((long long)p.m_tiles * p.n_tiles > 0x7fffffffLL - here) return cudaErrorInvalidValue;
  p.targets = targets; p.part = reinterpret_cast<float2*>(part); p.mine = mine;
  p.form = shape_of(bias, bias_bf16, scale, cap);
  p.error = nullptr;
  if (cudaGetSymbolAddress(reinterpret_cast<void**>(&p.error), g_error) != cudaSuccess) return cudaErrorInvalidValue;
  const int tiles = p.m_tiles * p.n_tiles;
  const dim3 grid(2 * (tiles < here ? tiles : here));
  const CUtensorMap& xm = *reinterpret_cast<const CUtensorMap*>(x_map);
  const CUtensorMap& wm = *reinterpret_cast<const CUtensorMap*>(w_map);
  auto kernel = cap > 0.f ? logprob_kernel<false, true>
                          : bias || scale != 1.f ? logprob_kernel<false, false> : logprob_kernel<true, false>;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = kSmemBytes;
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
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, xm, wm, p);
  return e != cudaSuccess ? static_cast<int>(e) : launch_status();
}

// The same partials of a piece of logits in memory: z [M, n], columns `first`, first + 1, ... of the vocabulary;
// part [ceil(n / 4096)][M].
SAKV_EXPORT int sakv_logprob_fold(const float* z, long long ld, int M, int n, int first, int vocab,
                                  const int32_t* targets, float* part, float* mine, const void* bias,
                                  int bias_bf16, float scale, float cap, cudaStream_t stream) {
  if (M <= 0 || n <= 0 || first < 0 || first > vocab - n || ld < n || !(cap >= 0.f) ||
      (n + kFoldColumns - 1) / kFoldColumns > 65535)
    return cudaErrorInvalidValue;
  const dim3 grid(M, (n + kFoldColumns - 1) / kFoldColumns);
  return launch_ordered(fold_kernel, grid, dim3(kFoldThreads), 0, stream, z, ld, M, n, first, vocab, targets,
                        reinterpret_cast<float2*>(part), mine, shape_of(bias, bias_bf16, scale, cap));
}

SAKV_EXPORT int sakv_logprob_join(const float* part, const float* mine, const int32_t* targets, float* logprob,
                                  float* lse, int M, int N, int pieces, cudaStream_t stream) {
  if (M <= 0 || pieces < 0) return cudaErrorInvalidValue;
  return launch_overlapped(join_kernel, dim3((M + 31) / 32), dim3(32 * kJoinWarps), 0, stream, 1,
                           reinterpret_cast<const float2*>(part), mine, targets, logprob, lse, M, N, pieces);
}

SAKV_EXPORT int sakv_logprob_error(int* value) {
  return static_cast<int>(cudaMemcpyFromSymbol(value, g_error, sizeof(int)));
}
