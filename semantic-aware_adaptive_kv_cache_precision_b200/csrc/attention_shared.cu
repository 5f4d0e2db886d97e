// Decode attention in bfloat16 over blocks that several sequences list: one new token per sequence, and
// what sequences share (they were forked from one another) is read once for all of them.
//
//   s_j = scale q . k_j,  m = max_j s_j,  l = sum_j e^(s_j - m),  out = sum_j e^(s_j - m) v_j / l
//
// for the positions j of a sequence's length. The sum may be cut anywhere and joined: a piece with its own
// (m, l, o = sum e^(s - m) v) enters with weight e^(m - max m). The host's plan cuts the block lists into
// pieces that the same set of sequences lists (ops/shared.py); a unit of work is a piece, up to 128 rows of
// queries (sequences of the piece x query heads of one KV head) and that KV head.
//
//   grid  = units x KV heads, heaviest first; block = 6 warps, two blocks an SM
//   tile  = one cache block: 64 keys x head_dim by TMA (128-byte swizzle) into a ring of stages
// and a unit's rows of queries are worked on in one of two ways:
//   wide   (more than kNarrowRows rows, up to 128) on tcgen05: S = Q K^T with the rows on tensor memory's lanes,
//          one thread a row for the softmax, P written over S as the A operand of P V, O in tensor memory; the
//          next tile's S is computed under this tile's softmax.
//   narrow (up to kNarrowRows rows) on mma.sync: NR = groups of 16 rows (1 or 2); warp w of four takes rows
//          16 (w % NR) .. + 15 and 16 NR keys of every tile from 16 NR (w / NR) on, so that four warps have
//          work however few the rows; warps of the same rows are merged at the end.
//
// Every unit leaves a partial (m, l, o) for each of its (sequence, head); a sequence's partials lie side by
// side, in the order of its positions, and `join_kernel` merges them. Scores, maxima, exponentials and sums
// are fp32; probabilities are rounded to bf16 for the product with the values, as values are stored (an error
// of half a step, up to 2^-8 of a probability, as in the other attention kernels). Every wait on a copy is bounded.
// The reference reads a sequence's cache for every sequence (`src/core_kernels/attention.cu:754-815`).
#include "common.cuh"
#include "mma.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace {

constexpr int KT = kCacheBlock;
constexpr int kWarps = 4;
constexpr int kThreads = 192;        // 6 warps; four of them in a narrow unit and in the join
constexpr int kNarrowThreads = kWarps * 32;
constexpr int kStages = 3;           // of a narrow unit
// Rows up to which a unit is narrow. Measured, us of the kernel over 32,000 shared positions, two KV heads of 6
// query heads: 12 rows 11.5 narrow; 24 rows 14.3 narrow, 14.1 wide; 60 rows 20.2 narrow, 14.1 wide.
constexpr int kWideRows = 128, kNarrowRows = 32, kMostGroup = 16;
constexpr int kWideStages = 2;
constexpr int kMembers = kWideRows + 2;
constexpr uint32_t kTmemCols = 256;  // wide: S 2 x 64 (P over the first 32 of each), O from 128 on
constexpr uint32_t kOCol = 128;
constexpr float kLazy = 8.f;         // O is rescaled when a row's maximum has grown by 2^8
// A wide unit takes maxima before it scales them, and scales -inf: right for scales above 0 alone.
constexpr float kLeastScale = 1e-30f;

template <int D>
struct Smem {
  static constexpr int kBoxes = D / 64;
  static constexpr int kTileBytes = KT * D * 2;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kQBytes = kWideRows * D * 2;
  static constexpr int kNarrow = kStages * kStageBytes, kWide = kQBytes + kWideStages * kStageBytes;
  static constexpr int kBarriers = kNarrow > kWide ? kNarrow : kWide;     // where they lie
  static constexpr int kBytes = kBarriers + 1024 + 256;
};

// What the host's plan holds (int32 words, offsets in words): see ops/shared.py.
struct Plan {
  const int32_t* words;
  int unit_at, member_at, first_at;    // units (8 words each), members (2 each), a sequence's first partial
  int span_at;                         // the shortest and the longest length of a sequence that the plan covers
  int unit_capacity;
};

struct Params {
  Plan plan;
  const __nv_bfloat16* q;
  long long q_stride;
  int q_aligned;                       // whether its rows begin at multiples of 16 bytes
  const int32_t* seq_lens;
  const int32_t* block_table;
  int max_blocks, sequences;
  int heads, kv_heads;
  int settled;                         // whether plan, lengths and block lists may be read before the wait (see `launch`)
  float* part_o;                       // [partials][heads][D]
  float2* part_ml;                     // [partials][heads]: (maximum in base 2, sum)
  float scale_log2e;
  int* error;
};

// Words 0-1 of the plan: units, sequences. A unit's words: the sequence whose block list is read, its first
// block, blocks, first member, first row of that member, rows, whether several sequences list its blocks, 0; rows are
// (member, query head of the KV head), heads fastest. A member: (sequence, its partial). Blocks that several list are
// filled in all of them; lengths that say otherwise are outside the plan, and the unit and the join answer NaN.
struct Unit {
  int sequence, column, columns, member, row, rows, shared, pad;
};

// Row r of the unit: its query, and where its partial goes.
struct Row {
  const __nv_bfloat16* q;
  long long slot;
};
__device__ __forceinline__ Row row_at(const Params& p, const int2* member, const Unit& u, int g, int r, int d) {
  const int group = p.heads / p.kv_heads;
  const int j = (u.row + r) / group, h = g * group + u.row + r - j * group;
  return Row{p.q + (long long)member[j].x * p.q_stride + (long long)h * d, (long long)member[j].y * p.heads + h};
}

template <int D, int NR>
__device__ __forceinline__ void
attend_narrow(const Params& p, const CUtensorMap* k_map, const CUtensorMap* v_map, uint8_t* smem, uint64_t* full,
              uint64_t* empty, int* failed, const int* listed, int g, const Unit& u, int n_tiles, int kv_len,
              const int2* member) {
  using S = Smem<D>;
  constexpr int KW = 16 * NR;          // keys of a tile that a warp takes
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rg = warp % NR, kp = warp / NR;
  const int rows = u.rows, col0 = u.column;

  auto request = [&](int i) {
    const int stage = i % kStages;
    const int block = i < kThreads ? listed[i] : p.block_table[(long long)u.sequence * p.max_blocks + col0 + i];
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
      at[i] = r < rows ? row_at(p, member, u, g, r, D).q + c : nullptr;
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
  if (!alive) *failed = 1;
  asm volatile("bar.sync 1, %0;" ::"n"(kNarrowThreads) : "memory");
  if (*failed) {                  // (a copy did not come: see the others land before the memory is given back)
    if (threadIdx.x == 0)
      for (int i = max(0, n_tiles - kStages); i < n_tiles; ++i)
        tma::mbar_wait(&full[i % kStages], (i / kStages) & 1, p.error, 153);
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
  asm volatile("bar.sync 1, %0;" ::"n"(kNarrowThreads) : "memory");
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
    const long long to = row_at(p, member, u, g, r, D).slot;
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

// V tile as the B operand of P V: N (head dims) contiguous, 64 per 128-byte row, the next 64 dims one box
// further; 8 keys per 1024-byte swizzle group.
__device__ __forceinline__ uint64_t desc_values(uint32_t addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr & 0x3FFFF) >> 4);
  d |= static_cast<uint64_t>((KT * 128) >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

struct WideBarriers {
  uint64_t q_full;
  uint64_t k_full[kWideStages], k_empty[kWideStages];     // keys: free again as soon as S_j is done
  uint64_t v_full[kWideStages], v_empty[kWideStages];     // values: free once P_j V_j is done
  uint64_t s_full[2];
  uint64_t p_full;       // P_j lies in tensor memory over S_j
  uint64_t pv_done;      // P_j V_j has been added to O
};

// Up to 128 rows on tcgen05: warp 0 copies, lane 0 of warp 1 issues the products, warps 2-5 hold a row a thread.
template <int D>
__device__ __forceinline__ void
attend_wide(const Params& p, const CUtensorMap* k_map, const CUtensorMap* v_map, uint8_t* smem, WideBarriers* bar,
            uint32_t tmem, const int* listed, int g, const Unit& u, int n, int kv_len, const int2* member) {
  using S = Smem<D>;
  uint8_t* q_s = smem;
  uint8_t* kv_s = q_s + S::kQBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    if (lane == 0) {
      int j = 0, v_sent = 0;
      for (; j < n; ++j) {
        const int stage = j % kWideStages;
        const int block = j < kThreads ? listed[j]
                                       : p.block_table[(long long)u.sequence * p.max_blocks + u.column + j];
        const int row0 = (block * p.kv_heads + g) * KT;
        uint8_t* dst = kv_s + stage * S::kStageBytes;
        if (j >= kWideStages &&
            !tma::mbar_wait(&bar->k_empty[stage], ((j / kWideStages) - 1) & 1, p.error, 161))
          break;
        tma::mbar_expect_tx(&bar->k_full[stage], S::kTileBytes);
        for (int x = 0; x < S::kBoxes; ++x)
          tma::load_2d(dst + x * (KT * 128), k_map, x * 64, row0, &bar->k_full[stage]);
        if (j >= kWideStages &&
            !tma::mbar_wait(&bar->v_empty[stage], ((j / kWideStages) - 1) & 1, p.error, 162)) {
          ++j;
          break;
        }
        tma::mbar_expect_tx(&bar->v_full[stage], S::kTileBytes);
        for (int x = 0; x < S::kBoxes; ++x)
          tma::load_2d(dst + S::kTileBytes + x * (KT * 128), v_map, x * 64, row0, &bar->v_full[stage]);
        v_sent = j + 1;
      }
      // the copies in flight land before the memory is given back (they have, unless a wait ran out)
      for (int i = max(0, j - kWideStages); i < j; ++i)
        tma::mbar_wait(&bar->k_full[i % kWideStages], (i / kWideStages) & 1, p.error, 163);
      for (int i = max(0, v_sent - kWideStages); i < v_sent; ++i)
        tma::mbar_wait(&bar->v_full[i % kWideStages], (i / kWideStages) & 1, p.error, 164);
    }
  } else if (warp == 1) {
    // the whole warp walks and one lane issues, and no turn of the loop depends on what a lane saw, so that the operands
    // stay in uniform registers
    constexpr uint32_t idesc_s = tc::idesc_bf16_f32(kWideRows, KT);                   // K-major both
    constexpr uint32_t idesc_pv = tc::idesc_bf16_f32(kWideRows, D) | (1u << 16);      // B MN-major
    const uint32_t elected = tc::elect_lane();
    const int tiles = __shfl_sync(0xffffffffu, n, 0);
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t queries = tc::smem_desc_k_major_sw128(tma::smem_u32(q_s));         // (descriptors count 16 bytes)
    const uint64_t keys = tc::smem_desc_k_major_sw128(tma::smem_u32(kv_s));
    const uint64_t values = desc_values(tma::smem_u32(kv_s + S::kTileBytes));
    bool ok = tma::mbar_wait(&bar->q_full, 0, p.error, 165);
    auto issue_pv = [&](int i) {
      const int stage = i % kWideStages;
      ok = ok && tma::mbar_wait(&bar->p_full, i & 1, p.error, 166) &&
           tma::mbar_wait(&bar->v_full[stage], (i / kWideStages) & 1, p.error, 167);
      __syncwarp();
      tc::fence_after_sync();
      const uint32_t go = elected && ok;
      const uint64_t v = values + stage * (S::kStageBytes >> 4);
#pragma unroll
      for (int k = 0; k < KT / 16; ++k)
        tc::mma_ts_if(go, base + kOCol, base + (i & 1) * KT + k * 8, v + k * (2048 >> 4), idesc_pv, i > 0 || k > 0);
      tc::commit_if(go, &bar->pv_done);
      tc::commit_if(go, &bar->v_empty[stage]);
    };
    for (int j = 0; j < tiles; ++j) {
      const int stage = j % kWideStages;
      // (S_j goes where S_{j-2} and then P_{j-2} lay: P_{j-2} V_{j-2} was issued before this, and one
      // thread's products run in the order it issued them)
      ok = ok && tma::mbar_wait(&bar->k_full[stage], (j / kWideStages) & 1, p.error, 168);
      __syncwarp();
      tc::fence_after_sync();
      const uint32_t go = elected && ok;
      const uint64_t k_at = keys + stage * (S::kStageBytes >> 4);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        tc::mma_ss_if(go, base + (j & 1) * KT, queries + ((k >> 2) * (kWideRows * 128) + (k & 3) * 32) / 16,
                      k_at + ((k >> 2) * (KT * 128) + (k & 3) * 32) / 16, idesc_s, k > 0);
      tc::commit_if(go, &bar->s_full[j & 1]);
      tc::commit_if(go, &bar->k_empty[stage]);
      if (j >= 1) issue_pv(j - 1);
    }
    if (tiles > 0) issue_pv(tiles - 1);
  } else {
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;                         // row of the unit = tensor-memory lane
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    Row row{nullptr, 0};
    if (r < u.rows) row = row_at(p, member, u, g, r, D);
    // this warp's 32 queries into the swizzled tile, 16 bytes a lane, neighbouring lanes along a row (zeros for
    // rows that the unit does not have). A row a thread, 4 bytes at a time, took 5 to 8 us.
    {
      constexpr int kLanes = D / 8, kPer = 32 / kLanes;          // lanes of a row, rows at a time
      const int c = lane % kLanes;
      uint4 v[32 / kPer];
#pragma unroll
      for (int i = 0; i < 32 / kPer; ++i) {
        const int of = i * kPer + lane / kLanes;
        const uint64_t at = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(row.q), of);
        v[i] = make_uint4(0, 0, 0, 0);
        if (at) {
          const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(at) + c * 8;
          if (p.q_aligned) {
            v[i] = *reinterpret_cast<const uint4*>(src);
          } else {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(src);
            v[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 32 / kPer; ++i) {
        const int of = quarter * 32 + i * kPer + lane / kLanes;
        *reinterpret_cast<uint4*>(q_s + (c >> 3) * (kWideRows * 128) + of * 128 + (((c & 7) ^ (of & 7)) << 4)) = v[i];
      }
    }
    tma::fence_proxy_async();
    tma::mbar_arrive(&bar->q_full);
    float m_true = -INFINITY;      // running maximum of the scaled scores
    float m_ref = -INFINITY;       // what the exponentials, the row's sum and O are relative to
    float l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int bj = j & 1;
      if (!tma::mbar_wait(&bar->s_full[bj], (j >> 1) & 1, p.error, 169)) { ok = false; break; }
      tc::fence_after_sync();
      float s[KT];
      tc::ld_32x32b_x64(lane_base + bj * KT, s);
      const int valid = kv_len - (u.column + j) * KT;          // keys of the tile that exist
      if (valid < KT) {
#pragma unroll
        for (int c = 0; c < KT; ++c) s[c] = c < valid ? s[c] : -INFINITY;
      }
      float big4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < KT; c += 8) {
#pragma unroll
        for (int q = 0; q < 4; ++q) big4[q] = mma::max3(big4[q], s[c + 2 * q], s[c + 2 * q + 1]);
      }
      const float big = fmaxf(fmaxf(big4[0], big4[1]), fmaxf(big4[2], big4[3]));
      m_true = fmaxf(m_true, big * p.scale_log2e);
      bool waited = j == 0;          // whether P_{j-1} V_{j-1} is known to be done
      const bool move = m_true > m_ref + kLazy;      // (also true the first time a key is seen)
      if (__any_sync(0xffffffffu, move)) {
        const float factor = move ? mma::exp2_fast(m_ref - m_true) : 1.f;   // 0 when m_ref = -inf
        if (j >= 1) {
          if (!tma::mbar_wait(&bar->pv_done, (j - 1) & 1, p.error, 170)) { ok = false; break; }
          waited = true;
          tc::fence_after_sync();
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            float v[16];
            tc::ld_32x32b_x16(lane_base + kOCol + c, v);
#pragma unroll
            for (int i = 0; i < 16; i += 2) mma::mul2(v[i], v[i + 1], factor);
            tc::st_32x32b_x16(lane_base + kOCol + c, v);
          }
          tc::fence_before_sync();
        }
        if (move) {
          l *= factor;
          m_ref = m_true;
        }
      }
      const float minus_m = (m_ref == -INFINITY) ? 0.f : -m_ref;
      float sum4[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t packed[KT / 2];
#pragma unroll
      for (int i = 0; i < KT / 2; ++i) {
        float e0, e1;
        mma::fma2(e0, e1, s[2 * i], s[2 * i + 1], p.scale_log2e, minus_m);
        const float p0 = mma::exp2_fast(e0), p1 = mma::exp2_fast(e1);
        mma::add2(sum4[(i & 1) * 2], sum4[(i & 1) * 2 + 1], p0, p1);
        packed[i] = mma::pack_bf16(p0, p1);
      }
      tc::st_32x32b_x32(lane_base + bj * KT, packed);
      l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
      if (valid < KT) {
        // value rows behind the sequence's end are stale: zero them, so that 0 x garbage is 0
        if (!tma::mbar_wait(&bar->v_full[j % kWideStages], (j / kWideStages) & 1, p.error, 171)) { ok = false; break; }
        uint8_t* vt = kv_s + (j % kWideStages) * S::kStageBytes + S::kTileBytes;
        for (int i = r; i < (KT - valid) * (D / 8); i += kWideRows) {
          const int key = valid + i / (D / 8), c = i % (D / 8);
          *reinterpret_cast<uint4*>(vt + (c >> 3) * (KT * 128) + key * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
        }
        tma::fence_proxy_async();
      }
      // (every product is waited for once, in order: a barrier's phases are told apart by one bit)
      if (!waited && !tma::mbar_wait(&bar->pv_done, (j - 1) & 1, p.error, 172)) { ok = false; break; }
      tc::fence_before_sync();
      tma::mbar_arrive(&bar->p_full);
    }
    if (ok && tma::mbar_wait(&bar->pv_done, (n - 1) & 1, p.error, 173)) {
      tc::fence_after_sync();
      // through shared memory (every copy has landed and every product is done), so that a warp writes whole
      // rows: a row a thread took 3 us
      constexpr int kRow = D + 4;          // (padded: neighbouring rows' pieces lie in other banks)
      float* mine = reinterpret_cast<float*>(smem) + quarter * 32 * kRow;
#pragma unroll
      for (int c = 0; c < D; c += 16) {
        float v[16];
        tc::ld_32x32b_x16(lane_base + kOCol + c, v);
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4*>(mine + lane * kRow + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
      if (row.q) p.part_ml[row.slot] = make_float2(m_ref, l);
      __syncwarp();
      constexpr int kLanes = D / 4, kPer = 32 / kLanes;
      const int c = lane % kLanes * 4;
#pragma unroll 8
      for (int i = 0; i < 32; i += kPer) {
        const int of = i + lane / kLanes;
        const long long slot = __shfl_sync(0xffffffffu, row.slot, of);
        if (quarter * 32 + of < u.rows)
          *reinterpret_cast<float4*>(p.part_o + slot * D + c) = *reinterpret_cast<const float4*>(mine + of * kRow + c);
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 2)
shared_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                        const __grid_constant__ Params p) {
  using S = Smem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBarriers);       // narrow: kStages full, kStages empty
  uint64_t* empty = full + kStages;
  WideBarriers* wide = reinterpret_cast<WideBarriers*>(smem + S::kBarriers);
  __shared__ int listed[kThreads];
  __shared__ int2 member[kMembers];
  __shared__ int failed;
  __shared__ uint32_t tmem_at;

  // First of all, and in narrow units too: until a block has given up its right to tensor memory, the SM starts no
  // second block of a kernel that may ask for it (measured: the second ones started 8 to 15 us late).
  if ((threadIdx.x >> 5) == 1) tc::tmem_alloc(&tmem_at, kTmemCols);
  // (settled: the plan, the block lists and the lengths were written before the kernel before this one began; what that
  // one wrote, queries, keys and values, is read behind the wait below. Else all of it is.)
  if (!p.settled) wait_for_previous_kernel();
  const int unit = blockIdx.x / p.kv_heads, g = blockIdx.x - unit * p.kv_heads;
  const int group = p.heads / p.kv_heads;
  // (the grid is as large as the plan has room for; a unit behind its last one reads words of no meaning, and
  // nothing with them)
  const int4* words = reinterpret_cast<const int4*>(p.plan.words + p.plan.unit_at + unit * 8);
  const int4 a = words[0], b = words[1];
  const bool live = unit < p.plan.words[0];
  Unit u{};
  int n_tiles = 0, kv_len = 0;
  if (live) {
    u = Unit{a.x, a.y, a.z, a.w, b.x, b.y, b.z, 0};
    const int given = p.seq_lens[u.sequence];
    kv_len = given < 0 || given > p.max_blocks * KT ? 0 : given;
    n_tiles = min((kv_len + KT - 1) / KT - u.column, u.columns);
    if (u.shared && kv_len / KT < u.column + u.columns) n_tiles = 0;
    const int members = (u.row + u.rows + group - 1) / group;
    if (threadIdx.x < members)
      member[threadIdx.x] = *reinterpret_cast<const int2*>(p.plan.words + p.plan.member_at +
                                                           2 * (u.member + threadIdx.x));
    if (threadIdx.x < n_tiles)
      listed[threadIdx.x] = p.block_table[(long long)u.sequence * p.max_blocks + u.column + threadIdx.x];
  }
  const bool is_wide = u.rows > kNarrowRows && n_tiles > 0;
  if (threadIdx.x == 0) {
    failed = 0;
    tma::prefetch_map(&k_map);
    tma::prefetch_map(&v_map);
    if (is_wide) {
      tma::mbar_init(&wide->q_full, kWideRows);
      for (int s = 0; s < kWideStages; ++s) {
        tma::mbar_init(&wide->k_full[s], 1);
        tma::mbar_init(&wide->k_empty[s], 1);
        tma::mbar_init(&wide->v_full[s], 1);
        tma::mbar_init(&wide->v_empty[s], 1);
      }
      for (int i = 0; i < 2; ++i) tma::mbar_init(&wide->s_full[i], 1);
      tma::mbar_init(&wide->p_full, kWideRows);
      tma::mbar_init(&wide->pv_done, 1);
    } else {
      for (int s = 0; s < kStages; ++s) {
        tma::mbar_init(&full[s], 1);
        tma::mbar_init(&empty[s], kWarps);
      }
    }
    tma::fence_barrier_init();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  let_next_kernel_start();       // (with its shared and tensor memory in hand)
  wait_for_previous_kernel();
  if (n_tiles <= 0) {            // a piece that the sequence has not reached yet: it counts for nothing
    for (int r = threadIdx.x; r < u.rows; r += kThreads)
      p.part_ml[row_at(p, member, u, g, r, D).slot] = make_float2(-INFINITY, u.shared ? NAN : 0.f);
  } else if (is_wide) {
    attend_wide<D>(p, &k_map, &v_map, smem, wide, tmem_at, listed, g, u, n_tiles, kv_len, member);
  } else if (threadIdx.x < kNarrowThreads) {
#define SAKV_NARROW(NR) \
  attend_narrow<D, NR>(p, &k_map, &v_map, smem, full, empty, &failed, listed, g, u, n_tiles, kv_len, member)
    if (u.rows <= 16) SAKV_NARROW(1);
    else SAKV_NARROW(2);
#undef SAKV_NARROW
  }
  tc::fence_before_sync();
  __syncthreads();
  if ((threadIdx.x >> 5) == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem_at, kTmemCols);
  }
}

// out[b, h] = sum_s w_s o_s / sum_s w_s l_s, w_s = 2^(m_s - max m), over the sequence's partials. A block a
// (sequence, head): D / 4 threads hold four sizes each, the block's groups of them take partials s, s + groups,
// ... with kRound reads in flight, and are merged through shared memory in their order.
template <int D>
__global__ void __launch_bounds__(kNarrowThreads)
join_kernel(const Plan plan, const float* part_o, const float2* part_ml, __nv_bfloat16* __restrict__ out,
            const int32_t* seq_lens, int heads, int settled) {
  constexpr int kLanes = D / 4, kGroups = kNarrowThreads / kLanes, kRound = 4;
  let_next_kernel_start();
  if (!settled) wait_for_previous_kernel();
  const int b = blockIdx.x / heads, h = blockIdx.x - b * heads;
  const int first = plan.words[plan.first_at + b], end = plan.words[plan.first_at + b + 1];
  const int least = plan.words[plan.span_at + 2 * b], most = plan.words[plan.span_at + 2 * b + 1];
  const int len = seq_lens[b];
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
  // (no key at all: zeros; a length that the plan does not cover: not a number, rather than a part of the answer)
  const float inv = len <= 0 || total == 0.f ? 0.f : len < least || len > most ? NAN : 1.f / total;
  if (len <= 0) acc = make_float4(0.f, 0.f, 0.f, 0.f);
  *reinterpret_cast<uint2*>(out + (long long)blockIdx.x * D + c) =
      make_uint2(mma::pack_bf16(acc.x * inv, acc.y * inv), mma::pack_bf16(acc.z * inv, acc.w * inv));
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

// `p.settled`: the plan, the lengths and the block lists were written before the kernel before this one began, as a
// step's inputs are, and may be read while it runs. Else they are read behind the wait for it, which takes 1 us of 27 a
// layer (64 sequences of 32,000 positions; 5 if the kernel were launched behind all that came before).
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
  return launch_overlapped(join_kernel<D>, dim3((unsigned)(p.sequences * p.heads)), dim3(kNarrowThreads), 0, stream, 1,
                           p.plan, p.part_o, p.part_ml, out, p.seq_lens, p.heads, p.settled);
}

}  // namespace

// A plan's numbers (ops/shared.py): width of the block lists, words where units, members, the sequences' first
// partials and the lengths covered begin, units, partials that the scratch holds.
struct SakvSharedPlan {
  int width, unit_at, unit_capacity, member_at, first_at, span_at, partials, sequences, heads, kv_heads;
};

// `keys`, `values`: the cache entry [blocks][kv_heads][64][head_dim]; `plan`: int32 words on the device, laid out as the
// numbers `n` (on the host) say; `part`: scratch of partials x heads x (head_dim + 2) floats; `settled`: see `launch`.
SAKV_EXPORT int sakv_shared_attention(const void* keys, const void* values, long long blocks, const void* q,
                                      long long q_stride,
                                      const int32_t* seq_lens, const int32_t* block_table, const int32_t* plan,
                                      const SakvSharedPlan* n, void* out, float* part, int head_dim, float scale,
                                      int settled, cudaStream_t stream) {
  const int sequences = n->sequences, heads = n->heads, kv_heads = n->kv_heads, max_blocks = n->width;
  if (sequences < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads / kv_heads > kMostGroup ||
      max_blocks < 0 || max_blocks > (1 << 24) || n->unit_capacity < 0 || n->partials < 0 || (q_stride & 1) ||
      (n->unit_at & 7) || (n->member_at & 1) || (reinterpret_cast<uintptr_t>(q) & 3) ||
      (reinterpret_cast<uintptr_t>(plan) & 15) || (reinterpret_cast<uintptr_t>(part) & 15) ||
      (long long)n->unit_capacity * kv_heads > 0x7fffffffLL || (long long)sequences * heads > 0x7fffffffLL ||
      !(scale >= kLeastScale && scale <= 1.f / kLeastScale))
    return cudaErrorInvalidValue;
  if (sequences == 0) return 0;
  Params p;
  p.plan = Plan{plan, n->unit_at, n->member_at, n->first_at, n->span_at, n->unit_capacity};
  p.q = reinterpret_cast<const __nv_bfloat16*>(q); p.q_stride = q_stride;
  p.q_aligned = q_stride % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0;
  p.seq_lens = seq_lens; p.block_table = block_table; p.max_blocks = max_blocks; p.sequences = sequences;
  p.heads = heads; p.kv_heads = kv_heads; p.settled = settled != 0;
  p.part_o = part;
  p.part_ml = reinterpret_cast<float2*>(part + (long long)n->partials * heads * head_dim);
  p.scale_log2e = scale * 1.4426950408889634f;
  p.error = error_word();
  if (!p.error) return cudaErrorInvalidValue;
  const long long rows = blocks * kv_heads * KT;
  if (blocks <= 0 || rows > 0x7fffffffLL || (head_dim != 64 && head_dim != 128)) return cudaErrorInvalidValue;
  CUtensorMap km, vm;
  int bad = tma::make_map_bf16_2d(&km, keys, (uint64_t)rows, head_dim, (uint64_t)head_dim * 2, KT, 64);
  if (!bad) bad = tma::make_map_bf16_2d(&vm, values, (uint64_t)rows, head_dim, (uint64_t)head_dim * 2, KT, 64);
  if (bad) return bad;
  __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(out);
  return head_dim == 64 ? launch<64>(km, vm, p, o, stream) : launch<128>(km, vm, p, o, stream);
}

SAKV_EXPORT int sakv_shared_attention_error(int* value) {
  return static_cast<int>(cudaMemcpyFromSymbol(value, g_error, sizeof(int)));
}
