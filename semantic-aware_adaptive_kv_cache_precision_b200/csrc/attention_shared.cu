// Decode attention in bfloat16 over blocks that several sequences list: one new token per sequence, and
// what sequences share (they were forked from one another) is read once for all of them.
//
//   s_j = scale q . k_j,  m = max_j s_j,  l = sum_j e^(s_j - m),  out = sum_j e^(s_j - m) v_j / l
//
// for the positions j of a sequence's length. The sum may be cut anywhere and joined: a piece with its own
// (m, l, o = sum e^(s - m) v) enters with weight e^(m - max m). The host's plan cuts the block lists into
// pieces that the same set of sequences lists (ops/shared.py); a unit of work is a piece, up to 64 rows of
// queries (sequences of the piece x query heads of one KV head) and that KV head.
//
//   grid  = units x KV heads, heaviest first; block = 4 warps
//   tile  = one cache block: 64 keys x head_dim by TMA (128-byte swizzle) into a ring of stages
//   NR    = groups of 16 rows the unit has (1, 2 or 4): warp w takes rows 16 (w % NR) .. + 15 and 16 NR keys
//           of every tile from 16 NR (w / NR) on, so that four warps have work however few the rows; warps of
//           the same rows are merged at the end.
//
// Every unit leaves a partial (m, l, o) for each of its (sequence, head); a sequence's partials lie side by
// side, in the order of its positions, and `join_kernel` merges them. Scores, maxima, exponentials and sums
// are fp32; probabilities are rounded to bf16 for the product with the values, as values are stored (an error
// of half a step, 2^-9 of a probability, as in the other attention kernels). Every wait on a copy is bounded.
// The reference reads a sequence's cache for every sequence (`src/core_kernels/attention.cu:754-815`).
#include "common.cuh"
#include "mma.cuh"
#include "tma.cuh"

namespace {

constexpr int KT = kCacheBlock;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;
constexpr int kRows = 64;            // most rows of a unit

template <int D>
struct Smem {
  static constexpr int kBoxes = D / 64;
  static constexpr int kTileBytes = KT * D * 2;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kBytes = kStages * kStageBytes + 1024 + 256;
};

// What the host's plan holds (int32 words, offsets in words): see ops/shared.py.
struct Plan {
  const int32_t* words;
  int unit_at, member_at, first_at;    // units (8 words each), members (2 each), a sequence's first partial
  int unit_capacity;
};

struct Params {
  Plan plan;
  const __nv_bfloat16* q;
  long long q_stride;
  const int32_t* seq_lens;
  const int32_t* block_table;
  int max_blocks, sequences;
  int heads, kv_heads;
  float* part_o;                       // [partials][heads][D]
  float2* part_ml;                     // [partials][heads]: (maximum in base 2, sum)
  int partials;
  float scale_log2e;
  int* error;
};

// Words 0-1 of the plan: units, sequences. A unit's words: the sequence whose block list is read, its first
// block, blocks, first member, members, 0, 0, 0. A member: (sequence, its partial).
template <int D, int NR>
__device__ __forceinline__ void
attend(const Params& p, const CUtensorMap* k_map, const CUtensorMap* v_map, uint8_t* smem, uint64_t* full,
       uint64_t* empty, const int* listed, int g, int row_seq, int col0, int n_tiles, int kv_len,
       const int2* member, int members) {
  using S = Smem<D>;
  constexpr int KW = 16 * NR;          // keys of a tile that a warp takes
  const int group = p.heads / p.kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rg = warp % NR, kp = warp / NR;
  const int rows = members * group;

  auto request = [&](int i) {
    const int stage = i % kStages;
    const int block = i < kThreads ? listed[i] : p.block_table[(long long)row_seq * p.max_blocks + col0 + i];
    const int row0 = (block * p.kv_heads + g) * KT;
    uint8_t* dst = smem + stage * S::kStageBytes;
    tma::mbar_expect_tx(&full[stage], S::kStageBytes);
    for (int x = 0; x < S::kBoxes; ++x) {
      tma::load_2d(dst + x * (KT * 128), k_map, x * 64, row0, &full[stage]);
      tma::load_2d(dst + S::kTileBytes + x * (KT * 128), v_map, x * 64, row0, &full[stage]);
    }
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < min(kStages, n_tiles); ++i) request(i);

  // this warp's 16 query rows; rows that the unit does not have are zero
  uint32_t qf[D / 16][4];
  {
    const int c = (lane & 3) * 2;
    const __nv_bfloat16* at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = rg * 16 + (lane >> 2) + 8 * i;
      at[i] = nullptr;
      if (r < rows) {
        const int j = r / group;
        at[i] = p.q + (long long)member[j].x * p.q_stride + (long long)(g * group + r - j * group) * D + c;
      }
    }
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qf[ks][i] = at[i & 1] ? *reinterpret_cast<const uint32_t*>(at[i & 1] + ks * 16 + (i >> 1) * 8) : 0u;
  }
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  bool alive = true;

  for (int i = 0; i < n_tiles; ++i) {
    const int stage = i % kStages;
    if (!tma::mbar_wait(&full[stage], (i / kStages) & 1, p.error, 152)) {
      alive = false;
      break;
    }
    const uint32_t kbase = tma::smem_u32(smem + stage * S::kStageBytes);
    const uint32_t vbase = kbase + S::kTileBytes;
    const int valid = kv_len - (col0 + i) * KT - kp * KW;      // keys of this warp that exist
    if (valid < KW) {
      // rows behind the sequence's end hold whatever the block held before: zero the value rows of this
      // warp's keys, so that 0 x garbage cannot become NaN (warps of the same keys write the same zeros)
      uint8_t* vt = smem + stage * S::kStageBytes + S::kTileBytes;
      for (int r = max(valid, 0); r < KW; ++r)
        for (int x = 0; x < S::kBoxes; ++x)
          reinterpret_cast<uint32_t*>(vt + x * (KT * 128) + (kp * KW + r) * 128)[lane] = 0u;
      __syncwarp();
    }
    float s[2 * NR][4];
#pragma unroll
    for (int nt = 0; nt < 2 * NR; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
    {
      const int row = kp * KW + (lane & 7) + ((lane >> 4) << 3);
      const int half = (lane >> 3) & 1;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int chunk = ks * 2 + half;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          uint32_t b0, b1, b2, b3;
          mma::ldmatrix_x4(mma::swizzled(kbase + (chunk >> 3) * (KT * 128), row + n * 16, chunk & 7), b0, b1, b2,
                           b3);
          mma::bf16_16816(s[2 * n], qf[ks], b0, b1);
          mma::bf16_16816(s[2 * n + 1], qf[ks], b2, b3);
        }
      }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < 2 * NR; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool seen = nt * 8 + (lane & 3) * 2 + (e & 1) < valid;
        s[nt][e] = seen ? s[nt][e] * p.scale_log2e : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[nt][e]);
      }
    float corr[2], base[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float m_new = fmaxf(m[r], top[r]);
      corr[r] = (m_new == -INFINITY) ? 1.f : mma::exp2_fast(m[r] - m_new);
      m[r] = m_new;
      base[r] = (m_new == -INFINITY) ? 0.f : m_new;       // (2^(-inf - 0) = 0: nothing seen yet)
      l[r] *= corr[r];
    }
    uint32_t pf[NR][4];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int i2 = 0; i2 < 4; ++i2) {
        // registers of the A operand: rows r, r + 8 of keys 0-7, then of keys 8-15
        const int nt = 2 * n + (i2 >> 1), r = i2 & 1;
        const float p0 = mma::exp2_fast(s[nt][2 * r] - base[r]), p1 = mma::exp2_fast(s[nt][2 * r + 1] - base[r]);
        l[r] += p0 + p1;
        pf[n][i2] = mma::pack_bf16(p0, p1);
      }
    {
      const int row = kp * KW + (lane & 7) + (((lane >> 3) & 1) << 3);
      const int half = lane >> 4;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        o[2 * j][0] *= corr[0]; o[2 * j][1] *= corr[0]; o[2 * j][2] *= corr[1]; o[2 * j][3] *= corr[1];
        o[2 * j + 1][0] *= corr[0]; o[2 * j + 1][1] *= corr[0];
        o[2 * j + 1][2] *= corr[1]; o[2 * j + 1][3] *= corr[1];
        const int chunk = j * 2 + half;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          uint32_t b0, b1, b2, b3;
          mma::ldmatrix_x4_trans(mma::swizzled(vbase + (chunk >> 3) * (KT * 128), row + n * 16, chunk & 7), b0, b1,
                                 b2, b3);
          mma::bf16_16816(o[2 * j], pf[n], b0, b1);
          mma::bf16_16816(o[2 * j + 1], pf[n], b2, b3);
        }
      }
    }
    __syncwarp();
    if (lane == 0) {
      tma::mbar_arrive(&empty[stage]);
      if (warp == 0 && i + kStages < n_tiles) {
        if (!tma::mbar_wait(&empty[stage], (i / kStages) & 1, p.error, 151)) alive = false;
        else request(i + kStages);
      }
    }
    alive = __shfl_sync(0xffffffffu, alive, 0);
    if (!alive) break;
  }

  // ---- the warps' shares of a row, merged through shared memory (every tile has been read) ----
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }
  alive = __syncthreads_and(alive);
  if (!alive) {                  // (a copy did not come: see the others land before the memory is given back)
    if (threadIdx.x == 0)
      for (int i = max(0, n_tiles - kStages); i < n_tiles; ++i)
        tma::mbar_wait(&full[i % kStages], (i / kStages) & 1, p.error, 153);
    __syncthreads();
    return;
  }
  constexpr int kRow = D + 8;
  float* sm_o = reinterpret_cast<float*>(smem);                // [warp][16][kRow]
  float* sm_m = sm_o + kWarps * 16 * kRow;                     // [warp][16]
  float* sm_l = sm_m + kWarps * 16;
  {
    const int r0 = lane >> 2, c = (lane & 3) * 2;
#pragma unroll
    for (int nt = 0; nt < D / 8; ++nt) {
      float* row0 = sm_o + (warp * 16 + r0) * kRow + nt * 8 + c;
      *reinterpret_cast<float2*>(row0) = make_float2(o[nt][0], o[nt][1]);
      *reinterpret_cast<float2*>(row0 + 8 * kRow) = make_float2(o[nt][2], o[nt][3]);
    }
    if ((lane & 3) == 0) {
      sm_m[warp * 16 + r0] = m[0]; sm_m[warp * 16 + r0 + 8] = m[1];
      sm_l[warp * 16 + r0] = l[0]; sm_l[warp * 16 + r0 + 8] = l[1];
    }
  }
  __syncthreads();
  // a warp takes rows warp, warp + 4, ...; a lane four sizes of the head
#pragma unroll 2
  for (int r = warp; r < rows; r += kWarps) {
    constexpr int kParts = kWarps / NR;
    const int at = (r >> 4) * 16 + (r & 15);                   // row in the first of its warps
    // (a share that saw nothing has the sum 0; one whose scores are all NaN has a NaN sum, which passes on)
    float big = -INFINITY;
#pragma unroll
    for (int w = 0; w < kParts; ++w) big = fmaxf(big, sm_m[w * NR * 16 + at]);
    float weight[kParts], total = 0.f;
#pragma unroll
    for (int w = 0; w < kParts; ++w) {
      const float mine = sm_m[w * NR * 16 + at];
      const float sum = sm_l[w * NR * 16 + at];
      weight[w] = sum == 0.f ? 0.f : mma::exp2_fast(mine - big);
      total += weight[w] * sum;
    }
    const int j = r / group;
    const long long to = (long long)member[j].y * p.heads + g * group + r - j * group;
    if (lane < D / 4) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kParts; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(sm_o + (w * NR * 16 + at) * kRow + lane * 4);
        acc.x += weight[w] * v.x; acc.y += weight[w] * v.y;
        acc.z += weight[w] * v.z; acc.w += weight[w] * v.w;
      }
      *reinterpret_cast<float4*>(p.part_o + to * D + lane * 4) = acc;
    }
    if (lane == 0) p.part_ml[to] = make_float2(big, total);
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads)
shared_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                        const __grid_constant__ Params p) {
  using S = Smem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * S::kStageBytes);
  uint64_t* empty = full + kStages;
  __shared__ int listed[kThreads];
  __shared__ int2 member[kRows];

  let_next_kernel_start();
  const int unit = blockIdx.x / p.kv_heads, g = blockIdx.x - unit * p.kv_heads;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      tma::mbar_init(&full[s], 1);
      tma::mbar_init(&empty[s], kWarps);
    }
    tma::fence_barrier_init();
    tma::prefetch_map(&k_map);
    tma::prefetch_map(&v_map);
  }
  // (the plan, the block lists and the lengths are the step's inputs: they were written before the kernel
  // before this one began; what that one wrote, queries, keys and values, is read behind the wait)
  const bool live = unit < min(p.plan.words[0], p.plan.unit_capacity);
  int4 what = make_int4(0, 0, 0, 0);
  int members = 0, n_tiles = 0, kv_len = 0;
  if (live) {
    what = *reinterpret_cast<const int4*>(p.plan.words + p.plan.unit_at + unit * 8);
    members = p.plan.words[p.plan.unit_at + unit * 8 + 4];
    const int given = p.seq_lens[what.x];
    kv_len = given < 0 || given > p.max_blocks * KT ? 0 : given;
    n_tiles = min((kv_len + KT - 1) / KT - what.y, what.z);
    if (threadIdx.x < members)
      member[threadIdx.x] = *reinterpret_cast<const int2*>(p.plan.words + p.plan.member_at +
                                                           2 * (what.w + threadIdx.x));
    if (threadIdx.x < n_tiles)
      listed[threadIdx.x] = p.block_table[(long long)what.x * p.max_blocks + what.y + threadIdx.x];
  }
  wait_for_previous_kernel();
  if (!live) return;
  __syncthreads();
  const int group = p.heads / p.kv_heads;
  const int rows = members * group;
  if (n_tiles <= 0) {            // a piece that the sequence has not reached yet: it counts for nothing
    for (int r = threadIdx.x; r < rows; r += kThreads) {
      const int j = r / group;
      p.part_ml[(long long)member[j].y * p.heads + g * group + r - j * group] = make_float2(-INFINITY, 0.f);
    }
    return;
  }
#define SAKV_ATTEND(NR) \
  attend<D, NR>(p, &k_map, &v_map, smem, full, empty, listed, g, what.x, what.y, n_tiles, kv_len, member, members)
  if (rows <= 16) SAKV_ATTEND(1);
  else if (rows <= 32) SAKV_ATTEND(2);
  else SAKV_ATTEND(4);
#undef SAKV_ATTEND
}

// out[b, h] = sum_s w_s o_s / sum_s w_s l_s, w_s = 2^(m_s - max m), over the sequence's partials. A block a
// (sequence, head): D / 4 threads hold four sizes each, the block's groups of them take partials s, s + groups,
// ... with kRound reads in flight, and are merged through shared memory in their order.
template <int D>
__global__ void __launch_bounds__(kThreads)
join_kernel(const Plan plan, const float* __restrict__ part_o, const float2* __restrict__ part_ml,
            __nv_bfloat16* __restrict__ out, int heads) {
  constexpr int kLanes = D / 4, kGroups = kThreads / kLanes, kRound = 4;
  let_next_kernel_start();
  const int b = blockIdx.x / heads, h = blockIdx.x - b * heads;
  const int first = plan.words[plan.first_at + b], end = plan.words[plan.first_at + b + 1];
  const int group = threadIdx.x / kLanes, c = threadIdx.x % kLanes * 4;
  wait_for_previous_kernel();
  float big = -INFINITY, total = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = first + group; s0 < end; s0 += kGroups * kRound) {
    float2 ml[kRound];
    float4 o[kRound];
    float top = big;
    bool any = false;
#pragma unroll
    for (int i = 0; i < kRound; ++i) {
      const int s = s0 + i * kGroups;
      const long long at = (long long)s * heads + h;
      ml[i] = s < end ? part_ml[at] : make_float2(-INFINITY, 0.f);
      o[i] = s < end ? *reinterpret_cast<const float4*>(part_o + at * D + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < kRound; ++i) {
      top = fmaxf(top, ml[i].x);
      any |= ml[i].y != 0.f;
    }
    if (!any) continue;
    const float keep = total == 0.f ? 0.f : exp2f(big - top);
    total *= keep;
    acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
    big = top;
#pragma unroll
    for (int i = 0; i < kRound; ++i) {
      if (ml[i].y == 0.f) continue;             // (a piece of nothing: its output was not written)
      const float w = exp2f(ml[i].x - big);
      total += w * ml[i].y;
      acc.x += w * o[i].x; acc.y += w * o[i].y; acc.z += w * o[i].z; acc.w += w * o[i].w;
    }
  }
  __shared__ float sm_m[kGroups], sm_l[kGroups];
  __shared__ float4 sm_o[kGroups][kLanes];
  if (c == 0) {
    sm_m[group] = big;
    sm_l[group] = total;
  }
  sm_o[group][threadIdx.x % kLanes] = acc;
  __syncthreads();
  if (group) return;
#pragma unroll
  for (int i = 1; i < kGroups; ++i) big = fmaxf(big, sm_m[i]);
  total = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    if (sm_l[i] == 0.f) continue;
    const float w = exp2f(sm_m[i] - big);
    const float4 v = sm_o[i][threadIdx.x];
    total += w * sm_l[i];
    acc.x += w * v.x; acc.y += w * v.y; acc.z += w * v.z; acc.w += w * v.w;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;      // no key at all: zeros
  *reinterpret_cast<uint2*>(out + (long long)blockIdx.x * D + c) =
      make_uint2(mma::pack_bf16(acc.x * inv, acc.y * inv), mma::pack_bf16(acc.z * inv, acc.w * inv));
}

__device__ int g_error;

template <int D>
int launch(const CUtensorMap& k_map, const CUtensorMap& v_map, Params& p, __nv_bfloat16* out, cudaStream_t stream) {
  static PerDeviceOnce configured;
  if (configured.needs()) {
    const cudaError_t e = cudaFuncSetAttribute(shared_attention_kernel<D>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::kBytes);
    if (e != cudaSuccess) return (int)e;
    configured.done();
  }
  if (p.plan.unit_capacity > 0) {
    const int e = launch_overlapped(shared_attention_kernel<D>, dim3((unsigned)(p.plan.unit_capacity * p.kv_heads)),
                                    dim3(kThreads), Smem<D>::kBytes, stream, 1, k_map, v_map, p);
    if (e) return e;
  }
  return launch_overlapped(join_kernel<D>, dim3((unsigned)(p.sequences * p.heads)), dim3(kThreads), 0, stream, 1,
                           p.plan, p.part_o, p.part_ml, out, p.heads);
}

}  // namespace

// `plan`: int32 words on the device (see ops/shared.py for their order), of which `unit_capacity` units at
// word `unit_at`, the members at `member_at` and the sequences' first partials at `first_at`; `partials`: how
// many the scratch holds ([partials][heads][head_dim] and [partials][heads][2] floats).
SAKV_EXPORT int sakv_shared_attention(const void* k_map, const void* v_map, const void* q, long long q_stride,
                                      const int32_t* seq_lens, const int32_t* block_table, int max_blocks,
                                      const int32_t* plan, int unit_at, int unit_capacity, int member_at,
                                      int first_at, void* out, float* part_o, float* part_ml, int partials,
                                      int sequences, int heads, int kv_heads, int head_dim, float scale,
                                      cudaStream_t stream) {
  if (sequences < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads / kv_heads > kRows ||
      max_blocks <= 0 || max_blocks > (1 << 24) || unit_capacity < 0 || partials < 0 || (q_stride & 1) ||
      (unit_at & 3) || (member_at & 1) || (reinterpret_cast<uintptr_t>(q) & 3) ||
      (reinterpret_cast<uintptr_t>(plan) & 15) || (long long)unit_capacity * kv_heads > 0x7fffffffLL ||
      (long long)sequences * heads > 0x7fffffffLL)
    return cudaErrorInvalidValue;
  if (sequences == 0) return 0;
  Params p;
  p.plan = Plan{plan, unit_at, member_at, first_at, unit_capacity};
  p.q = reinterpret_cast<const __nv_bfloat16*>(q); p.q_stride = q_stride;
  p.seq_lens = seq_lens; p.block_table = block_table; p.max_blocks = max_blocks; p.sequences = sequences;
  p.heads = heads; p.kv_heads = kv_heads;
  p.part_o = part_o; p.part_ml = reinterpret_cast<float2*>(part_ml); p.partials = partials;
  p.scale_log2e = scale * 1.4426950408889634f;
  p.error = nullptr;
  if (cudaGetSymbolAddress(reinterpret_cast<void**>(&p.error), g_error) != cudaSuccess) return cudaErrorInvalidValue;
  const CUtensorMap& km = *reinterpret_cast<const CUtensorMap*>(k_map);
  const CUtensorMap& vm = *reinterpret_cast<const CUtensorMap*>(v_map);
  __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(out);
  if (head_dim == 64) return launch<64>(km, vm, p, o, stream);
  if (head_dim == 128) return launch<128>(km, vm, p, o, stream);
  return cudaErrorInvalidValue;
}

SAKV_EXPORT int sakv_shared_attention_error(int* value) {
  return static_cast<int>(cudaMemcpyFromSymbol(value, g_error, sizeof(int)));
}
