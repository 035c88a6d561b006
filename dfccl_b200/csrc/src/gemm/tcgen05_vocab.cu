// Products over a large vocabulary for the losses of a language model's head, on CTA pairs (tcgen05 cta_group::2), bf16 with fp32
// accumulators in tensor memory.  With z = x w^T, x [n, d] and the head w [v, d]:
//   VOCAB_STATS     of every row the maximum and the sum of powers of each stretch of its logits, without those of its targets
//   VOCAB_GRAD      dz = g (softmax(z) - target): the logits are computed again, what is stored is their gradient, rounded once (in the targets' places 0,
//                   or theirs: vocab.h)
//   VOCAB_POWERS    powers of the logits relative to a number known in front of the product (the largest logit of the row's list), and their
//                   sums: the logits are not computed again, for rows whose gradients are wanted with the loss
//   VOCAB_PRODUCTS  dx = dz w and dw = dz^T x, in one launch
// A logit exists in tensor memory and registers only.  What bounds them is the tensor cores: busy 91 % of the cycles in the tiles of z, 93 - 95 % in
// the gradients' products (2048 x 50257 x 1024); 8192 x 50257 x 1024 takes 527 us (statistics), 566 (powers) and 1130 (products), 1.60, 1.49 and 1.49
// PFLOP/s of the 1.64 that a library product of 8192^3 reaches, and less where such kernels run for long, by the power limit.  Widths below
// 640 are bound by the epilogue (d = 64: 92 us for statistics of 4096 x 50257, 46 of them the powers in the special function units).
//
// Tiles of 256 x 256, stages of 64 of the contraction, roles as in tcgen05_gemm_pair.cu (TMA producer, MMA issuer, eight epilogue warps,
// two accumulators).  All of n, v are any number, d a multiple of 8: the tensor maps give zeros outside, the epilogues store inside.
#include "tc_common.h"
#include "gemm.h"
#include "epilogue.h"
#include "vocab.h"
#include "../common/device_once.h"
#include "../common/log.h"
#include <algorithm>

namespace dfccl {
namespace {

using namespace tc;

constexpr int T = VOCAB_TILE, HALF = 128, BK = 64, UMMA_K = 16, STAGES = 6;
constexpr int A_BYTES = HALF * BK * 2, STAGE_BYTES = 2 * A_BYTES;                 // per CTA: 128 rows of A, 128 of B
constexpr int SMEM_BYTES = 227 * 1024;                                            // all of it: tensor memory for one CTA at a time (tcgen05_gemm_pair.cu)
enum VocabMode { VOCAB_STATS, VOCAB_GRAD, VOCAB_POWERS, VOCAB_PRODUCTS };
// Eight epilogue warps work on a tile, two (PARTS) on 32 rows of it.  Where every element is a power of two there are two groups of eight,
// one for each accumulator: the waits of one tile (for its rows' targets, tensor memory, powers) lie beside the other's.
constexpr int PARTS = 2, EPI_WARPS = 4 * PARTS;
__host__ __device__ constexpr int groupsOf(int mode) { return mode == VOCAB_PRODUCTS ? 1 : 2; }
// Columns at a time.  (Powers that are stored and summed: with 32 the registers of 576 threads do not do; 4096 x 50257 x 256 with both gradients 386 us
// instead of 350.  Statistics with 16 are 2 - 6 % slower.  Loading the next columns ahead, the registers allowing it, gains nothing: the other warps do.)
__host__ __device__ constexpr int unitOf(int mode) { return mode == VOCAB_POWERS ? 16 : 32; }
__host__ __device__ constexpr int threadsOf(int mode) { return 64 + 32 * EPI_WARPS * groupsOf(mode); }
constexpr int JOIN_BYTES = 4 * HALF * 8;                                          // what one part of a tile's rows leaves for the other, of four tiles in turn
constexpr uint64_t WAIT_NS = 4000000000ull;                                       // nothing here waits on another GPU
static_assert(STAGES * STAGE_BYTES + JOIN_BYTES + 1024 + 512 <= SMEM_BYTES, "stages");

// One product: result [M, N], `kBlocks` blocks of 64 of the contraction cut into slices of `perSlice`.
struct Product {
  int M, N, mTiles, nTiles, kBlocks, slices, perSlice, items, groupM;
  int tn, stageBytes;               // columns of a tile (a multiple of 32, 128 to 256); bytes that a stage of a CTA is loaded with
  int aMn, bMn, bLoose;             // operand stored with the contraction index slow; loose: its blocks of 64 columns are loaded one by one
  __nv_bfloat16* out;               // direct results, ld N
  float* part;                      // or slices [slice][M][N]
  int add, wide;
  int exact;                        // what VocabExact adds to a direct result: 1 of dx, 2 of dw, 0 nothing
};
struct VocabArgs {
  Product p[2];                     // items of the first, then of the second (items = 0: none)
  int kStep, stages, stride;        // of the products: blocks of 64 of the contraction in a stage (1 or 2), stages, their bytes per CTA
  int headStart;                    // rounds of the second product's items that pairs with one item less of the first take alone
  VocabRows rows;
  float2* parts;
  VocabGrad grad;
  const float* base;                // of the powers
  VocabFactor factor;
  VocabExact exact;
  const int* only;                  // null, or a word without which there is nothing to do
  int early;                        // the kernel in front is nothing to this one: it is waited for at the end
  __nv_bfloat16* dz;
  int ld, first;                    // of dz; first column of the vocabulary
  uint32_t* err;
  uint32_t* errHost;
};

// The items of a pair.  Those of the first product go round; pairs that get one less of them (their time is several items' of the
// second) start on the second product while the others finish, then its items go round too.  What a pair gets is a matter of time, not of results.
struct Items {
  int pair, pairs, r, k0, t1, t2, n1, n2, early;
  __device__ Items(const VocabArgs& g, int pair_, int pairs_) : pair(pair_), pairs(pairs_) {
    t1 = g.p[0].items; t2 = g.p[1].items;
    r = t1 % pairs;
    early = r && pair >= r ? 1 : 0;
    k0 = r ? g.headStart : 0;
    n1 = t1 > pair ? (t1 - pair + pairs - 1) / pairs : 0;
    const int e = pairs - r, alone = k0 * e;
    n2 = t2 - alone > pair ? (t2 - alone - pair + pairs - 1) / pairs : 0;
    if (early) n2 += min(k0, t2 > pair - r ? (t2 - (pair - r) + e - 1) / e : 0);
  }
  __device__ int count() const { return n1 + n2; }
  // Which product, and its item.
  __device__ int at(int j, int& item) const {
    if (j < n1) { item = pair + j * pairs; return 0; }
    j -= n1;
    const int e = pairs - r;
    if (!early) item = k0 * e + pair + j * pairs;
    else item = j < k0 ? j * e + pair - r : k0 * e + pair + (j - k0) * pairs;
    return 1;
  }
};

struct Tile { int mt, nt, slice, k0, k1; };
__device__ __forceinline__ Tile tileOf(const Product& p, int item) {
  Tile t;
  const int tiles = p.mTiles * p.nTiles;
  t.slice = item / tiles;
  raster_tile(item - t.slice * tiles, p.mTiles, p.nTiles, p.groupM, t.mt, t.nt);
  t.k0 = t.slice * p.perSlice;
  t.k1 = min(p.kBlocks, t.k0 + p.perSlice);
  return t;
}

// A row's list from the first entry at or behind a column on.  The entry behind the present one is on its way too: a step does not wait
// for memory (without it 32 entries a row cost 60 us of the 640 that dz of 8192 x 50257 x 1024 took).
struct List {
  const int* tokens;
  const float* rest;
  int k, behind, next, next2;
  float q, q2;
  __device__ __forceinline__ void load(int at, int& token, float& q) {
    token = at < k ? tokens[at] : VOCAB_NO_TOKEN;
    q = at < k && rest ? rest[at] : 0.f;
  }
  __device__ __forceinline__ void none() { tokens = nullptr; rest = nullptr; k = behind = 0; next = next2 = VOCAB_NO_TOKEN; q = q2 = 0.f; }
  __device__ __forceinline__ void seek(const VocabRows& r, const float* allRest, int row, int token, int col) {
    none();
    if (r.targets) { if (token >= col) next = token; if (allRest) q = allRest[row]; return; }
    k = r.k; tokens = r.tokens + (size_t)row * k; rest = allRest ? allRest + (size_t)row * k : nullptr;
    int lo = 0, hi = k;
    while (lo < hi) { const int mid = (lo + hi) >> 1; if (tokens[mid] < col) lo = mid + 1; else hi = mid; }
    load(lo, next, q);
    load(lo + 1, next2, q2);
    behind = lo + 2;
  }
  __device__ __forceinline__ void step() { next = next2; q = q2; load(behind++, next2, q2); }
};

__device__ __forceinline__ void tmemLoad(uint32_t at, uint32_t (&r)[16]) { tmem_ld16(at, r); }
__device__ __forceinline__ void tmemLoad(uint32_t at, uint32_t (&r)[32]) { tmem_ld32(at, r); }

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(threadsOf(MODE), 1)
dfcclVocabKernel(const __grid_constant__ CUtensorMap mapA0, const __grid_constant__ CUtensorMap mapB0, const __grid_constant__ CUtensorMap mapA1,
                 const __grid_constant__ CUtensorMap mapB1, const __grid_constant__ VocabArgs g) {
  extern __shared__ uint8_t smemRaw[];
  constexpr int GROUPS = groupsOf(MODE), UNIT = unitOf(MODE);
  uint8_t* smem = (uint8_t*)(((uintptr_t)smemRaw + 1023) & ~(uintptr_t)1023);       // the same offset in both CTAs
  float2* joinBuf = (float2*)(smem + STAGES * STAGE_BYTES);          // [4 tiles][HALF rows]
  uint64_t* fullBar = (uint64_t*)(smem + STAGES * STAGE_BYTES + JOIN_BYTES);      // used in the leader only
  uint64_t* emptyBar = fullBar + STAGES;                             // in both CTAs (commit to both)
  uint64_t* accFull = emptyBar + STAGES;                             // [2] in both CTAs
  uint64_t* accEmpty = accFull + 2;                                  // [2] used in the leader only
  uint64_t* joinBar = accEmpty + 2;                                  // [4 quarters][4 tiles] the other part of 32 rows is in place
  uint32_t* tmemBaseSlot = (uint32_t*)(joinBar + 16);
  volatile uint32_t* giveUp = tmemBaseSlot + 1;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t cr = cluster_ctarank();             // 0 = leader
  const Items items(g, blockIdx.x >> 1, gridDim.x >> 1);
  int count = items.count();
  const int kStep = MODE == VOCAB_PRODUCTS ? g.kStep : 1, stages = MODE == VOCAB_PRODUCTS ? g.stages : STAGES;
  const int stride = MODE == VOCAB_PRODUCTS ? g.stride : STAGE_BYTES, aBytes = A_BYTES * kStep, mnBlock = 64 * BK * 2 * kStep;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&fullBar[s], 1); mbar_init(&emptyBar[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&accFull[a], 1); mbar_init(&accEmpty[a], 2 * EPI_WARPS); }
    for (int a = 0; a < 16; ++a) mbar_init(&joinBar[a], 1);
    *giveUp = 0;
    mbar_fence_init();
    tma_prefetch_desc(&mapA0);
    tma_prefetch_desc(&mapB0);
  }
  if (warp == 1) tmem_alloc_pair(tmemBaseSlot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                // the partner's barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t tmemBase = *tmemBaseSlot;
  if (!g.early) grid_dependency_wait();
  grid_launch_dependents();
  if ((MODE == VOCAB_STATS || MODE == VOCAB_POWERS) && g.only && *g.only == 0) count = 0;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs; bytes counted in the leader)
    if (elect_one()) {
      const uint32_t bar0 = mapa_u32(smem_u32(fullBar), 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int j = 0; j < count && ok; ++j) {
        int item;
        const int which = MODE == VOCAB_PRODUCTS ? items.at(j, item) : (items.at(j, item), 0);
        const Product& p = g.p[which];
        const CUtensorMap* ma = which ? &mapA1 : &mapA0;
        const CUtensorMap* mb = which ? &mapB1 : &mapB0;
        const Tile t = tileOf(p, item);
        const int bHalf = MODE == VOCAB_PRODUCTS ? p.tn / 2 : HALF;
        const int rowA = t.mt * T + (int)cr * HALF, rowB = t.nt * 2 * bHalf + (int)cr * bHalf;
        for (int k = t.k0; k < t.k1; k += kStep) {       // (the second half of a slice's last stage may be another's, or outside: it is not multiplied)
          if (!mbar_wait(&emptyBar[stage], phase ^ 1, giveUp, WAIT_NS)) { ok = false; break; }
          if (cr == 0) mbar_expect_tx(&fullBar[stage], 2 * (MODE == VOCAB_PRODUCTS ? p.stageBytes : STAGE_BYTES));       // my bytes and the partner's
          uint8_t* sa = smem + stage * stride;
          uint8_t* sb = sa + aBytes;
          const uint32_t bar = bar0 + stage * 8;
          // K-major: boxes of 64 of the contraction x 128 rows.  MN-major: blocks of 64 columns x 64 kStep of the contraction, in one load
          // where the matrix and the tile are cut into whole blocks, else block by block from any multiple of 16 columns.
          if (MODE != VOCAB_PRODUCTS) {
            tma_load_2d_pair(sa, ma, k * BK, rowA, bar);
            tma_load_2d_pair(sb, mb, k * BK, rowB, bar);
          } else {
            tma_load_3d_pair(sa, ma, p.aMn ? k * BK : rowA, p.aMn ? rowA / 64 : k, bar);
            if (!p.bLoose) tma_load_3d_pair(sb, mb, k * BK, rowB / 64, bar);
            else for (int i = 0; i * 64 < bHalf; ++i) tma_load_2d_pair(sb + i * mnBlock, mb, rowB + 64 * i, k * BK, bar);
          }
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) for (int i = 0; i < 20000; ++i) __nanosleep(200);     // copies already issued land before the CTA goes away
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (cr == 0 && elect_one()) {
      int stage = 0, blocks = 0;
      uint32_t phase = 0;
      for (int j = 0; j < count; ++j) {                // stages that are loaded again need their release
        int item;
        const Product& p = g.p[items.at(j, item)];
        const Tile t = tileOf(p, item);
        blocks += (t.k1 - t.k0 + kStep - 1) / kStep;
      }
      int loads = blocks - stages;
      bool ok = true;
      for (int j = 0; j < count && ok; ++j) {
        int item;
        const int which = MODE == VOCAB_PRODUCTS ? items.at(j, item) : (items.at(j, item), 0);
        const Product& p = g.p[which];
        const Tile t = tileOf(p, item);
        const bool aMn = MODE == VOCAB_PRODUCTS && p.aMn, bMn = MODE == VOCAB_PRODUCTS && p.bMn;
        const uint32_t idesc = umma_idesc_bf16(T, MODE == VOCAB_PRODUCTS ? p.tn : T, aMn, bMn);
        // per instruction (16 of the contraction): 32 bytes along a K-major row, two groups of 8 rows of an MN-major block.  Per 64: the next
        // box, or further down the same blocks.
        const uint32_t stepA = aMn ? 128u : 2u, stepB = bMn ? 128u : 2u, hopA = aMn ? 512u : A_BYTES / 16, hopB = 512u;
        const int ab = j & 1;
        if (!mbar_wait(&accEmpty[ab], ((j >> 1) & 1) ^ 1, giveUp, WAIT_NS)) break;
        tc_fence_after();
        const uint32_t d = tmemBase + ab * T;
        for (int k = t.k0; k < t.k1; k += kStep) {
          if (!mbar_wait(&fullBar[stage], phase, giveUp, WAIT_NS)) { ok = false; break; }
          tc_fence_after();
          const uint8_t* pa = smem + stage * stride;
          const uint64_t da = aMn ? umma_smem_desc_mn_sw128(pa, mnBlock) : umma_smem_desc_sw128(pa);
          const uint64_t db = bMn ? umma_smem_desc_mn_sw128(pa + aBytes, mnBlock) : umma_smem_desc_sw128(pa + aBytes);
#pragma unroll
          for (int h = 0; h < (MODE == VOCAB_PRODUCTS ? 2 : 1); ++h) {
            if (h == 1 && (kStep == 1 || k + 1 == t.k1)) break;
#pragma unroll
            for (int i = 0; i < BK / UMMA_K; ++i) umma_bf16_pair(d, da + hopA * h + stepA * i, db + hopB * h + stepB * i, idesc, k != t.k0 || (h | i) != 0);
          }
          if (loads-- > 0) umma_commit_pair(&emptyBar[stage]);      // both CTAs' stage is free once these MMAs have read it
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
        if (ok) umma_commit_pair(&accFull[ab]);       // both halves of the accumulator complete
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue: a row of my 128 per lane, 32 columns at a time
    const int quarter = warp & 3, part = (warp - 2) >> 2 & 1, group = (warp - 2) >> 3;
    const uint32_t accEmptyLeader0 = mapa_u32(smem_u32(&accEmpty[0]), 0), accEmptyLeader1 = mapa_u32(smem_u32(&accEmpty[1]), 0);
    const float factor = MODE == VOCAB_PRODUCTS ? vocabFactor(g.factor) : 1.f;
    // an accumulator goes back to the item after the next: every arrival is waited for
    auto release = [&](int j) {
      if (j + 2 >= count) return;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(j & 1 ? accEmptyLeader1 : accEmptyLeader0);
    };
    for (int j = group; j < count; j += GROUPS) {
      int item;
      const int which = MODE == VOCAB_PRODUCTS ? items.at(j, item) : (items.at(j, item), 0);
      const Product& p = g.p[which];
      const Tile t = tileOf(p, item);
      const int ab = j & 1;
      const int row0 = t.mt * T + (int)cr * HALF + quarter * 32, row = row0 + lane, tn = MODE == VOCAB_PRODUCTS ? p.tn : T, col0 = t.nt * tn;
      const bool mine = row0 < p.M, here = row < p.M;
      const uint32_t acc = tmemBase + ((uint32_t)(quarter * 32) << 16) + ab * T;
      if (MODE != VOCAB_PRODUCTS) {
        List list;
        list.none();
        const float scale = g.rows.scale;
        float lse = 0.f, coef = 0.f;
        if (here) {                                    // on its way while the accumulator is computed
          int token;
          const int state = rowState(g.rows, row, token);
          if (MODE == VOCAB_POWERS) {
            lse = g.base[row];
            coef = state == ROW_LIST ? 1.f : 0.f;
          }
          if (MODE == VOCAB_GRAD) {
            lse = g.grad.lse[row];
            coef = g.grad.gout ? g.grad.gout[(size_t)row * g.grad.goutStride] : 1.f;
            if (state != ROW_LIST) coef = state == ROW_BAD ? __int_as_float(0x7fffffff) : 0.f;
          }
          list.seek(g.rows, MODE == VOCAB_GRAD ? g.grad.rest : nullptr, row, token, g.first + col0);
        }
        if (!mbar_wait(&accFull[ab], (j >> 1) & 1, giveUp, WAIT_NS)) break;
        tc_fence_after();
        float top = -INFINITY, sum = 0.f;
        const int cols = MODE == VOCAB_STATS ? p.N : g.ld, units = (min(T, cols - col0) + UNIT - 1) / UNIT;
        uint32_t r[UNIT];
#pragma unroll 1
        for (int i = part; i < units; i += PARTS) {
          if (!mine) break;
          const int c = col0 + i * UNIT;
          __syncwarp();
          tmemLoad(acc + i * UNIT, r);
          tmem_ld_wait();
          if (MODE != VOCAB_GRAD) {
            if (c + UNIT > p.N) {
#pragma unroll
              for (int e = 0; e < UNIT; ++e) if (c + e >= p.N) r[e] = 0xff800000u;          // -inf
            }
            while (list.next < c + UNIT) {               // the list's entries: no power
              if (list.next >= c) {
                const int at = list.next - c;
#pragma unroll
                for (int e = 0; e < UNIT; ++e) if (e == at) r[e] = 0xff800000u;
              }
              list.step();
            }
            float m[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) m[e] = __uint_as_float(r[e]);
#pragma unroll
            for (int e = 4; e < UNIT; ++e) m[e & 3] = fmaxf(m[e & 3], __uint_as_float(r[e]));
            const float most = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            float base = lse;
            if (MODE == VOCAB_STATS) {
              // running maximum and sum over the row's columns
              const float now = fmaxf(top, most * scale);
              base = now == -INFINITY ? 0.f : now;
              sum *= exp2Approx(top - base);
              top = now;
            } else {
              top = fmaxf(top, fmaf(most, scale, -base));
            }
            float s[4] = {sum, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < UNIT; ++e) {
              const float v = exp2Approx(fmaf(__uint_as_float(r[e]), scale, -base));
              s[e & 3] += v;
              if (MODE == VOCAB_POWERS) r[e] = __float_as_uint(v);
            }
            sum = (s[0] + s[1]) + (s[2] + s[3]);
          } else {
#pragma unroll
            for (int e = 0; e < UNIT; ++e) r[e] = __float_as_uint(exp2Approx(fmaf(__uint_as_float(r[e]), scale, -lse)));
            int before = -1;
            while (list.next < g.first + c + UNIT) {
              if (list.next >= g.first + c) {
                const int at = list.next - g.first - c;
                if (at != before) {                      // (the first entry of a token has all of it)
#pragma unroll
                  for (int e = 0; e < UNIT; ++e) if (e == at) r[e] = __float_as_uint(-list.q);
                }
                before = at;
              }
              list.step();
            }
            if (c + UNIT > p.N) {
#pragma unroll
              for (int e = 0; e < UNIT; ++e) if (c + e >= p.N) r[e] = 0u;
            }
          }
          // (a row without a gradient may hold anything, infinities and NaN among it)
          if (MODE != VOCAB_STATS && here) {
            uint4 o[UNIT / 8];
#pragma unroll
            for (int v = 0; v < UNIT / 8; ++v) {
              uint32_t* ow = (uint32_t*)&o[v];
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                float lo = __uint_as_float(r[8 * v + 2 * w]), hi = __uint_as_float(r[8 * v + 2 * w + 1]);
                if (MODE == VOCAB_GRAD) { lo *= coef; hi *= coef; }
                ow[w] = coef == 0.f ? 0u : pack_bf16x2(lo, hi);
              }
            }
            __nv_bfloat16* dst = g.dz + (size_t)row * g.ld + c;
#pragma unroll
            for (int v = 0; v < UNIT / 8; v += 2) st_global32(dst + 8 * v, o + v, true);
          }
        }
        release(j);
        if (MODE != VOCAB_GRAD) {
          // The parts of a row meet in the first one's warp.  (The other comes back to this place four tiles on, when the first has released
          // the tile in between.)
          uint64_t* bar = joinBar + quarter * 4 + (j & 3);
          float2* at = joinBuf + (j & 3) * HALF + quarter * 32 + lane;
          if (part) {
            *at = make_float2(top, sum);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
          } else {
            if (!mbar_wait(bar, (j >> 2) & 1, giveUp, WAIT_NS)) break;
            const float2 q = *at;
            const float m = fmaxf(top, q.x), base = m == -INFINITY ? 0.f : m;
            sum = MODE == VOCAB_POWERS ? sum + q.y : sum * exp2Approx(top - base) + q.y * exp2Approx(q.x - base);
            if (here) g.parts[(size_t)t.nt * p.M + row] = make_float2(m, sum);
          }
        }
      } else {
        const float* sums = here && p.exact == 2 ? vocabSumsOf(g.exact, g.exact.first + row, p.N) : nullptr;      // (while the accumulator is computed)
        if (!mbar_wait(&accFull[ab], (j >> 1) & 1, giveUp, WAIT_NS)) break;
        tc_fence_after();
        const int steps = (min(tn, p.N - col0) + 31) / 32;
#pragma unroll 1
        for (int i = part; i < steps; i += PARTS) {
          if (!mine) break;
          const int c = col0 + i * 32, packs = min(4, (p.N - c) / 8);
          uint32_t r[32];
          __syncwarp();
          tmem_ld32(acc + i * 32, r);
          tmem_ld_wait();
          if (!here) continue;
          if (p.part) {
            float4* dst = (float4*)(p.part + ((size_t)t.slice * p.M + row) * p.N + c);
#pragma unroll
            for (int v = 0; v < 8; ++v) {
              if (v / 2 >= packs) break;
              float4 o = make_float4(__uint_as_float(r[4 * v]), __uint_as_float(r[4 * v + 1]), __uint_as_float(r[4 * v + 2]), __uint_as_float(r[4 * v + 3]));
              if (p.add) { const float4 q = dst[v]; o.x += q.x; o.y += q.y; o.z += q.z; o.w += q.w; }
              dst[v] = o;
            }
          } else {
            float f[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] = __uint_as_float(r[e]);
            if (p.exact == 1) vocabExactX<4>(f, g.exact, row, p.N, c, packs);
            else if (sums) {
#pragma unroll
              for (int v = 0; v < 8; ++v) {
                if (v / 2 >= packs) break;
                const float4 q = *((const float4*)(sums + c) + v);
                f[4 * v] -= q.x; f[4 * v + 1] -= q.y; f[4 * v + 2] -= q.z; f[4 * v + 3] -= q.w;
              }
            }
            uint4 o[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t* ow = (uint32_t*)&o[v];
#pragma unroll
              for (int w = 0; w < 4; ++w) ow[w] = pack_bf16x2(f[8 * v + 2 * w] * factor, f[8 * v + 2 * w + 1] * factor);
            }
            __nv_bfloat16* dst = p.out + (size_t)row * p.N + c;
            if (packs == 4) { st_global32(dst, o, p.wide); st_global32(dst + 16, o + 2, p.wide); }
            else {
#pragma unroll
              for (int v = 0; v < 4; ++v) if (v < packs) ((uint4*)dst)[v] = o[v];
            }
          }
        }
      }
      if (MODE == VOCAB_PRODUCTS) release(j);
    }
  }

  if (g.early) grid_dependency_wait();               // what comes behind this kernel comes behind the one in front too
  // ---------------------------------------------------------------- leave: nothing of the pair may still use my shared or tensor memory
  tc_fence_before();
  __syncthreads();
  cluster_sync_relaxed();
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmemBase, 512);
  if (threadIdx.x == 0 && *giveUp) { atomicExch(g.err, 1u); *(volatile uint32_t*)g.errHost = 1u; __threadfence_system(); }
}

// A tile's way out of tensor memory, in blocks of the contraction: no item takes less (3950 clocks and 512).  With items of one block counted as
// that, few pairs got nearly all of dw of 32 rows: 50257 x 1024 with both gradients took 257 us instead of 129.
constexpr int STORE = 8;

template <int MODE>
ncclResult_t launchVocab(const CUtensorMap& a0, const CUtensorMap& b0, const CUtensorMap& a1, const CUtensorMap& b1, VocabArgs& g, cudaStream_t stream) {
  CUDACHECK(oncePerDevice([] { return allowSharedMemory(dfcclVocabKernel<MODE>, SMEM_BYTES); }));
  DFCHECK(gemmErrorWords(&g.err, &g.errHost));
  cudaLaunchConfig_t cfg = {};
  const int pairs = std::min(g.p[0].items + g.p[1].items, gemmPairResident());
  cfg.gridDim = dim3(2 * pairs); cfg.blockDim = dim3(threadsOf(MODE)); cfg.dynamicSmemBytes = SMEM_BYTES; cfg.stream = stream;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization; at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at; cfg.numAttrs = 1;
  // the head start of pairs with one item less of the first product: as many items of the second as that one takes
  const int64_t c1 = std::max(g.p[0].perSlice, STORE), c2 = std::max(g.p[1].perSlice, STORE);
  g.headStart = g.p[1].items ? (int)((c1 + c2 / 2) / c2) : 0;
  CUDACHECK(cudaLaunchKernelEx(&cfg, dfcclVocabKernel<MODE>, a0, b0, a1, b1, g));
  return ncclSuccess;
}

Product productOf(int M, int N, int K, int per, int tn) {
  Product p = {};
  p.M = M; p.N = N; p.mTiles = (M + T - 1) / T; p.nTiles = (N + tn - 1) / tn;
  p.tn = tn; p.stageBytes = STAGE_BYTES;
  p.kBlocks = (K + BK - 1) / BK;
  p.perSlice = per;
  p.slices = vocabSlices(K, per);
  p.items = p.mTiles * p.nTiles * p.slices;
  p.groupM = 8;
  return p;
}

// The tiles of z: x and w both K-major.
ncclResult_t logits(CUtensorMap* a, CUtensorMap* b, VocabArgs* g, const void* x, const void* w, int n, int v, int d, const VocabRows& rows) {
  *g = VocabArgs{};
  DFCHECK(gemmEncodeMap(a, x, (uint64_t)n, (uint64_t)d, HALF));
  DFCHECK(gemmEncodeMap(b, w, (uint64_t)v, (uint64_t)d, HALF));
  g->p[0] = productOf(n, v, d, (d + BK - 1) / BK, T);
  g->rows = rows;
  return ncclSuccess;
}

}  // namespace

ncclResult_t vocabStats(const void* x, const void* w, int n, int v, int d, const VocabRows& rows, float2* parts, const int* only, bool early, cudaStream_t stream) {
  CUtensorMap a, b;
  VocabArgs g;
  DFCHECK(logits(&a, &b, &g, x, w, n, v, d, rows));
  g.parts = parts; g.only = only; g.early = early;
  return launchVocab<VOCAB_STATS>(a, b, a, b, g, stream);
}

ncclResult_t vocabPowers(const void* x, const void* w, int n, int v, int d, const VocabRows& rows, const float* base, float2* parts, void* powers, const int* only,
                         cudaStream_t stream) {
  CUtensorMap a, b;
  VocabArgs g;
  DFCHECK(logits(&a, &b, &g, x, w, n, v, d, rows));
  g.parts = parts; g.base = base; g.dz = (__nv_bfloat16*)powers; g.ld = (v + 63) / 64 * 64; g.only = only;
  return launchVocab<VOCAB_POWERS>(a, b, a, b, g, stream);
}

ncclResult_t vocabGrad(const void* x, const void* w, int n, int v, int first, int d, const VocabRows& rows, const VocabGrad& grad, void* dz, bool early,
                       cudaStream_t stream) {
  CUtensorMap a, b;
  VocabArgs g;
  DFCHECK(logits(&a, &b, &g, x, w, n, v, d, rows));
  g.grad = grad; g.early = early; g.dz = (__nv_bfloat16*)dz; g.ld = (v + 63) / 64 * 64; g.first = first;
  return launchVocab<VOCAB_GRAD>(a, b, a, b, g, stream);
}

// Columns of a tile of dx and dw: as few tiles as 256 columns make them, no wider than they need be (d = 640:
// 3 x 224; dx and dw of 4096 x 50257 in 355 us, in tiles of 256 387; d = 384 237 and 266, d = 128 130 and 149).
static int productWidth(int d) {
  const int tiles = (d + T - 1) / T;
  return std::max(128, ((d + tiles - 1) / tiles + 31) / 32 * 32);
}

// How long the pair with most to do is busy with `i1` items of `c1` blocks and `i2` of `c2`, handed out as Items does.
static int64_t longest(int64_t i1, int64_t c1, int64_t i2, int64_t c2, int64_t pairs) {
  const int64_t whole = i1 / pairs, r = i1 % pairs, e = pairs - r;
  if (!i2) return (whole + (r != 0)) * c1;
  const int64_t ahead = r ? (c1 + c2 / 2) / c2 : 0, left = std::max<int64_t>(0, i2 - ahead * e), each = (left + pairs - 1) / pairs;
  const int64_t alone = whole * c1 + (std::min(ahead, (i2 + e - 1) / e) + each) * c2;
  return r ? std::max(alone, (whole + 1) * c1 + each * c2) : alone;
}

// A product is cut into slices of its contraction where its tiles alone would keep pairs waiting: of some numbers of slices - none, as many as
// fill the pairs once, twice ..., or as give each item no more than a pair's share of all the work - those that by this estimate are
// through first.  A slice costs its sums a way to memory and back and the launch that joins them 3 us; none is cut below 16 blocks.
// 512 x 50257 x 1024, dx alone: 9 slices of 8 tiles on 74 pairs instead of 10, 136 us instead of 152.
VocabPlan vocabProductPlan(int n, int v, int d, bool wantX, bool wantW, int pairs) {
  constexpr double BLOCK_US = 0.27, BYTES_US = 6.5e6;              // a block under a tile of 256 columns; of memory
  const int tn = productWidth(d);
  const int64_t td = (d + tn - 1) / tn;
  struct Side { int64_t tiles, k, area; int64_t slices[6]; };
  Side x{(n + T - 1) / T * td, (v + BK - 1) / BK, (int64_t)n * d, {}}, w{(v + T - 1) / T * td, (n + BK - 1) / BK, (int64_t)v * d, {}};
  if (!wantX) x.tiles = 0;
  if (!wantW) w.tiles = 0;
  const int64_t share = std::max<int64_t>(1, (x.tiles * std::max<int64_t>(x.k, STORE) + w.tiles * std::max<int64_t>(w.k, STORE)) / pairs);
  for (Side* s : {&x, &w}) {
    const int64_t most = std::max<int64_t>(1, s->k / 16);
    for (int i = 0; i < 6; ++i)
      s->slices[i] = std::min(most, i == 0 || !s->tiles || s->tiles >= 4 * pairs ? 1 : i == 5 ? (s->k + share - 1) / share : std::max<int64_t>(1, i * pairs / s->tiles));
  }
  VocabPlan best{(int)x.k, (int)w.k};
  double least = 0.0;
  for (int i = 0; i < 6; ++i)
    for (int j = 0; j < 6; ++j) {
      if ((i && x.slices[i] == x.slices[0]) || (j && w.slices[j] == w.slices[0])) continue;
      const int64_t perX = (x.k + x.slices[i] - 1) / x.slices[i], perW = (w.k + w.slices[j] - 1) / w.slices[j];
      const int64_t sx = (x.k + perX - 1) / perX, sw = (w.k + perW - 1) / perW;
      const int64_t cx = std::max<int64_t>(perX, STORE), cw = std::max<int64_t>(perW, STORE);
      const int64_t blocks = x.tiles ? longest(x.tiles * sx, cx, w.tiles * sw, cw, pairs) : longest(w.tiles * sw, cw, 0, 0, pairs);
      auto join = [&](const Side& s, int64_t slices) { return s.tiles && slices > 1 ? 3.0 + (double)(slices * s.area * 8) / BYTES_US : 0.0; };
      const double us = blocks * BLOCK_US * tn / T + join(x, sx) + join(w, sw);
      if ((i | j) == 0 || us < least) { least = us; best = VocabPlan{(int)perX, (int)perW}; }
    }
  return best;
}

ncclResult_t vocabProducts(const void* dz, const void* x, const void* w, int n, int v, int d, const VocabPlan& plan, const VocabFactor& factor, const VocabExact* exact,
                           const VocabResult& dx, const VocabResult& dw, cudaStream_t stream) {
  const int ld = (v + 63) / 64 * 64;
  CUtensorMap a[2], b[2];
  VocabArgs g = {};
  g.factor = factor;
  if (exact) g.exact = *exact;
  int k = 0;
  // Stages of 128 of the contraction under narrower tiles: the tensor cores are through with one of 64 before its loads are issued.
  const int tn = productWidth(d), kStep = tn < T ? 2 : 1, box = BK * kStep;
  const bool loose = d % 64 != 0 || tn % 128 != 0;
  g.kStep = kStep;
  g.stride = A_BYTES * kStep + (tn / 2 + 63) / 64 * 64 * BK * 2 * kStep;
  g.stages = std::min(STAGES, STAGES * STAGE_BYTES / g.stride);
  auto narrow = [&](CUtensorMap* m, const void* base, int rows) {      // [rows of the contraction][d columns]
    return loose ? gemmEncodeMap(m, base, (uint64_t)rows, (uint64_t)d, box) : gemmEncodeMap3(m, base, (uint64_t)d, (uint64_t)rows, 1, tn / 2, box);
  };
  auto result = [&](const VocabResult& r, int which) {
    Product& p = g.p[k++];
    p.bMn = 1; p.bLoose = loose;
    p.stageBytes = g.stride;
    p.out = (__nv_bfloat16*)r.out; p.part = r.part; p.add = r.add;
    p.exact = exact && r.out ? which : 0;
    p.wide = d % 16 == 0 && ((uintptr_t)r.out & 31) == 0;
  };
  if (dx.out || dx.part) {
    DFCHECK(gemmEncodeMap3(&a[k], dz, (uint64_t)n, (uint64_t)ld, 0, HALF, box));
    DFCHECK(narrow(&b[k], w, v));
    g.p[k] = productOf(n, d, v, plan.perX, tn);
    result(dx, 1);
  }
  if (dw.out || dw.part) {
    DFCHECK(gemmEncodeMap3(&a[k], dz, (uint64_t)ld, (uint64_t)n, 1, HALF, box));
    DFCHECK(narrow(&b[k], x, n));
    g.p[k] = productOf(v, d, n, plan.perW, tn);
    g.p[k].aMn = 1;
    result(dw, 2);
  }
  if (!k) return ncclInvalidArgument;
  if (k == 1) { a[1] = a[0]; b[1] = b[0]; }
  return launchVocab<VOCAB_PRODUCTS>(a[0], b[0], a[1], b[1], g, stream);
}

}  // namespace dfccl
