// Expert products for many rows: out[r] = residual[r] + mul[r] * act(x[r] . W[e(r)]^T + bias[e(r)]) for rows sorted by
// expert, on the 5th-generation tensor cores from the packed 12-bit weights (no counterpart in the reference).
//
// One persistent CTA per SM walks the tiles t = blockIdx.x, + gridDim.x, ... of a list that exists only as arithmetic:
// tile t is row block t % nblk of token tile t / nblk, and the token tiles are counted expert by expert (at most 128
// rows each) from the experts' borders, which stay on the device.  Each CTA scans the borders once into shared
// memory; a tile's expert is then a binary search.  Row blocks of one token tile run side by side on neighbouring
// SMs and share its x rows in L2; token tiles of one expert follow one another and share its weights there.
//
// Inside a tile the roles are those of the projection GEMM (weights by TMA into a packed ring, x by TMA into an
// operand ring, 16 decoder warps writing decoded tiles to TMEM as the MMA's A operand, a scheduler warp handing
// stages to the issuing thread); what differs:
//   * every ring and its phases run on across the tiles, so the next tile's weights and x are on their way while
//     this one ends; the epilogue has four warps of its own (one per TMEM lane quadrant) and the accumulator is
//     double-buffered, so the decoders and the MMAs go on meanwhile;
//   * the MMA's N and the x boxes (32 rows each) follow the tile's own row count;
//   * the weights are packed in the tensor cores' pair order (mbp_expert_order), so decoded registers go to TMEM
//     without the quad transpose.
// Bound: the chain of a stage, not a unit.  12 experts of 1536 x 6144 (one round of tiles), 8 / 128 rows each: 44 / 59 us,
// DRAM 3.9 / 3.2 TB/s, ALU pipe 51 / 42 % of its cycles (the decode), tensor pipe 4 / 25 %, L2 to SM 15 / 20 %; warps wait for
// loads and barriers.  A stage of 24.5 KB of weights is a load, a decode, a store to TMEM, a hand-over, eight MMAs and a
// commit; with 128 rows its 32 KB of x, which every row block reads again, have to arrive as well.  64 experts (906 MB; 5.2
// rounds of tiles take 6): 195 us at 8 rows each, 216 at 64, 262 at 128, 399 at 160 (two token tiles: the weights decoded
// twice).  ptxas spills 24 bytes of the 80 registers that 768 threads leave each.
// All waits are bounded; TMEM is always released.
#include <cstdlib>
#include <map>
#include <mutex>

#include "common.cuh"
#include "epilogue.cuh"
#include "escape.cuh"
#include "tc.cuh"

using namespace mbp;

namespace {

constexpr int kDecWarps = 16;              // 8 row tiles x 2 chunks per stage
constexpr int kXWarp = 2 + kDecWarps;      // the x producer
constexpr int kSchedWarp = 3 + kDecWarps;  // waits for each stage's operands on behalf of the MMA issuer
constexpr int kEpiWarp = 4 + kDecWarps;    // four epilogue warps, warp kEpiWarp + q of TMEM lane quadrant q
constexpr int kThreads = 32 * (8 + kDecWarps);
static_assert(kEpiWarp % 4 == 0, "an epilogue warp reads the lane quadrant warp % 4");
constexpr int kHandBar = 1;   // named barrier of the scheduler -> issuer hand-over (64 threads)
constexpr int kPS = 3;        // packed ring depth (stages)
constexpr int kSub = MBP_C12_UNIT_BYTES;
constexpr int kStage = 16 * kSub;
constexpr int kBox = 32;      // rows of an x box
constexpr int kMaxExperts = 1024;
constexpr int kMaxSmem = 227 * 1024;

constexpr int kBN = 128;      // rows of a token tile.  (Tiles of 256, which decode a well-filled expert's weights once
                              // but leave room for two operand stages and one accumulator only, measured 5-25 % slower
                              // up to 128 rows per expert and even at 256.)
constexpr int kOS = 4;        // operand ring depth: x in shared memory and decoded A in TMEM (64 columns a stage)
constexpr int kAcc = 2;       // accumulators
constexpr int kXTile = kBN * 128;  // bytes of one chunk's x tile
constexpr int kTmemCols = kAcc * kBN + kOS * 64;
static_assert(kTmemCols == 512, "a power of two, and no more than TMEM has");

// Shared memory, bytes from the 1024-aligned base: packed ring, x ring, escape masks, barriers, words (TMEM base, abort),
// scan scratch, 1 KB per epilogue warp, first token tile of each expert [E + 1].
constexpr int kX = kPS * kStage;
constexpr int kMask = kX + kOS * 2 * kXTile;
constexpr int kBars = kMask + kDecWarps * kMaskUnitBytes;
constexpr int kWords = kBars + 8 * (2 * kPS + 3 * kOS + 2 * kAcc + 2);  // (one barrier more than there are: 16-byte pieces)
constexpr int kScan = kWords + 16;
constexpr int kTurn = kScan + 128;
constexpr int kTable = kTurn + 4096;
int smem_bytes(int experts) { return kTable + 4 * (experts + 1) + 1024; }
static_assert(kTable + 4 * (kMaxExperts + 1) + 1024 <= kMaxSmem, "fits for every expert count");

struct __align__(64) ExpertParams {
  CUtensorMap wmap;  // units [experts * R][C][192 x u64], box {192, 2, 8}
  CUtensorMap xmap;  // x [rows, k] bf16, box {64 columns, 32 rows}, 128-byte swizzle
  const uint8_t* bases;
  const int32_t* esc_off;
  const uint32_t* esc;
  void* out;
  int C, R, ldo;
  int wsubs;  // chunks per weight box: 2 (1 for a matrix of a single chunk)
  EpiArgs epi;
  GroupArgs group;
  unsigned long long wait_ns;  // limit of every bounded wait
};

// mbar_wait by a whole warp with one answer for all its lanes: what follows is warp-collective, and lanes that gave up
// at different times must not part.
MBP_DEV bool warp_wait(uint32_t bar, uint32_t parity, int code, uint64_t limit) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, code, limit)) != 0;
}

struct Tile {
  int expert, tok0, tend, rb0, rvalid;
};

__global__ void __launch_bounds__(kThreads, 1) k_experts(const __grid_constant__ ExpertParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* sm = smem_raw + (base - raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bars = base + kBars;
  const uint32_t pfull = bars, pempty = pfull + 8 * kPS;
  const uint32_t afull = pempty + 8 * kPS, xfull = afull + 8 * kOS, oempty = xfull + 8 * kOS;
  const uint32_t accfull = oempty + 8 * kOS, accfree = accfull + 8 * kAcc;
  const uint32_t done = accfree + 8 * kAcc;
  volatile uint32_t* words = reinterpret_cast<volatile uint32_t*>(sm + kWords);
  volatile uint32_t* abort_word = words + 1;  // set by the scheduler when a wait gave up
  int* scan = reinterpret_cast<int*>(sm + kScan);
  const int E = p.group.experts, C = p.C, R = p.R;
  int* first = reinterpret_cast<int*>(sm + kTable);  // first token tile of each expert
  const int nst = (C + 1) / 2;                       // stages of a tile (the last may hold one chunk)

  if (tid == 0) {
    for (int i = 0; i < kPS; ++i) {
      mbar_init(pfull + 8 * i, 1);
      mbar_init(pempty + 8 * i, kDecWarps * 32);
    }
    for (int i = 0; i < kOS; ++i) {
      mbar_init(afull + 8 * i, kDecWarps * 32);
      mbar_init(xfull + 8 * i, 1);
      mbar_init(oempty + 8 * i, 1);
    }
    for (int i = 0; i < kAcc; ++i) {
      mbar_init(accfull + 8 * i, 1);
      mbar_init(accfree + 8 * i, 4);
    }
    mbar_init(done, 1);
    *abort_word = 0u;
    fence_mbar_init();
    prefetch_tmap(&p.wmap);
    prefetch_tmap(&p.xmap);
  }
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + kWords),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  grid_dep_wait();
  grid_dep_launch();

  // ---- the token tiles before each expert (thread i takes experts 2i, 2i + 1); borders are clamped to the rows ----
  const auto border = [&](int e) { return min(max(p.group.offsets[e], 0), p.group.rows); };
  const auto rows_of = [&](int e) { return max(border(e + 1) - border(e), 0); };
  {
    const int e0 = 2 * tid;
    const int a = e0 < E ? (rows_of(e0) + kBN - 1) / kBN : 0, b = e0 + 1 < E ? (rows_of(e0 + 1) + kBN - 1) / kBN : 0;
    int inc = a + b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) scan[warp] = inc;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += scan[w];
    before += inc - a - b;
    if (e0 < E) first[e0] = before;
    if (e0 + 1 < E) first[e0 + 1] = before + a;
    if (e0 + 1 == E || e0 + 2 == E) first[E] = before + a + b;
    __syncthreads();
  }
  const uint32_t tmem = words[0];
  // Row blocks per token tile: blocks of up to 8 row tiles, smaller where that evens out the last round.  A block of b
  // row tiles costs about b + kBlockCost: the weight box and the decoders' chain of waits are as long for fewer tiles,
  // so smaller blocks pay only while SMs would hold none (3 experts of 1536 x 6144: 37 us in 36 blocks, 31 us in 144).
  constexpr int kBlockCost = 12;
  const int ttiles = first[E], G = gridDim.x;
  int nblk = (R + 7) / 8;
  {
    int best = 0x7fffffff;
    for (int b = 8; b >= 1; --b) {
      const int n = (R + b - 1) / b;
      const int cost = (int)(((long long)ttiles * n + G - 1) / G) * ((R + n - 1) / n + kBlockCost);
      if (cost < best) best = cost, nblk = n;
    }
  }
  const int tiles = ttiles * nblk;
  const auto tile_at = [&](int t) {
    const int tt = t / nblk, rb = t - tt * nblk;
    int l = 0, h = E - 1;  // the last expert whose first token tile is at or before tt (it has rows: tt < first[e + 1])
    while (l < h) {
      const int mid = (l + h + 1) >> 1;
      if (first[mid] <= tt)
        l = mid;
      else
        h = mid - 1;
    }
    Tile r;
    r.expert = l;
    const int lo = border(l);
    // an expert's token tiles alike, in whole x boxes: 128 rows and a few wait for x and then for the MMAs' fixed cost, two
    // halves for neither (64 experts of 1536 x 6144, 160 rows each on average: 414 -> 395 us)
    const int rows = rows_of(l);
    int per = kBN;
    if (rows > kBN) {
      const int parts = (rows + kBN - 1) / kBN;
      per = ((rows + parts - 1) / parts + kBox - 1) / kBox * kBox;
    }
    r.tok0 = lo + (tt - first[l]) * per;
    r.tend = min(r.tok0 + per, lo + rows);
    r.rb0 = (int)((long long)rb * R / nblk);
    r.rvalid = (int)((long long)(rb + 1) * R / nblk) - r.rb0;
    return r;
  };
  const auto width = [](const Tile& t) { return (t.tend - t.tok0 + 15) & ~15; };  // the MMA's N

  if (p.group.zero_tail) zero_tail(p.group, p.epi, p.out, p.ldo, 0, R * 16, blockIdx.x, G, tid, kThreads);

  if (warp == 0) {
    // ---------------- weight producer ----------------
    if (lane == 0) {
      Ring r{0, 1};
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += G) {
        const Tile tl = tile_at(t);
        const int row = tl.expert * R + tl.rb0;
        for (int i = 0; i < nst && ok; ++i, r.next(kPS)) {
          ok = mbar_wait(pempty + 8 * r.i, r.ph, MBP_DEV_TIMEOUT_EMPTY, p.wait_ns);
          if (!ok) break;
          mbar_arrive_expect_tx(pfull + 8 * r.i, (uint32_t)(p.wsubs * 8 * kSub));
          tma_load_3d(base + r.i * kStage, &p.wmap, 0, 2 * i, row, pfull + 8 * r.i);
        }
      }
      drain_ring(pfull, r, kPS, MBP_DEV_TIMEOUT_FULL);
    }
    __syncwarp();
  } else if (warp == kXWarp) {
    // ---------------- x producer ----------------
    if (lane == 0) {
      Ring r{0, 1};
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += G) {
        const Tile tl = tile_at(t);
        const int nb = (width(tl) + kBox - 1) / kBox;
        for (int i = 0; i < nst && ok; ++i, r.next(kOS)) {
          const int nt = min(2, C - 2 * i);
          ok = mbar_wait(oempty + 8 * r.i, r.ph, MBP_DEV_TIMEOUT_EMPTY, p.wait_ns);
          if (!ok) break;
          mbar_arrive_expect_tx(xfull + 8 * r.i, (uint32_t)(nt * nb * kBox * 128));
          for (int c = 0; c < nt; ++c)
            for (int b = 0; b < nb; ++b)
              tma_load_2d(base + kX + (r.i * 2 + c) * kXTile + b * kBox * 128, &p.xmap, (2 * i + c) * 64,
                          tl.tok0 + b * kBox, xfull + 8 * r.i);
        }
      }
      drain_ring(xfull, r, kOS, MBP_DEV_TIMEOUT_FULL);
    }
    __syncwarp();
  } else if (warp == kSchedWarp) {
    // ---------------- MMA scheduler: every round is always met, a timed-out wait ends both warps' work ----------------
    Ring r{0, 0}, acc{0, 1};
    bool ok = true;
    for (int t = blockIdx.x; t < tiles; t += G, acc.next(kAcc)) {
      for (int i = 0; i < nst; ++i, r.next(kOS)) {
        if (lane == 0 && ok) {
          if (i == 0) ok = mbar_wait(accfree + 8 * acc.i, acc.ph, MBP_DEV_TIMEOUT_MMA, p.wait_ns);
          ok = ok && mbar_wait(afull + 8 * r.i, r.ph, MBP_DEV_TIMEOUT_FULL, p.wait_ns) &&
               mbar_wait(xfull + 8 * r.i, r.ph, MBP_DEV_TIMEOUT_FULL, p.wait_ns);
          if (!ok) *abort_word = 1u;
        }
        named_bar_sync(kHandBar, 64);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    const uint64_t db0 = smem_desc_sw128(base + kX);
    int o = 0, acc = 0;
    for (int t = blockIdx.x; t < tiles; t += G) {
      const uint32_t idesc = idesc_bf16(width(tile_at(t))), d = tmem + (uint32_t)(acc * kBN);
      for (int i = 0; i < nst; ++i) {
        const uint32_t ta = tmem + (uint32_t)(kAcc * kBN + o * 64);
        const uint64_t db = db0 + (uint64_t)(o * (2 * kXTile >> 4));
        named_bar_sync(kHandBar, 64);
        if (lane == 0 && *abort_word == 0u) {
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_ts(d, ta + 8 * k, db + 2 * k, idesc, (i | k) != 0);
          if (2 * i + 1 < C) {
#pragma unroll
            for (int k = 0; k < 4; ++k) tc_mma_ts(d, ta + 32 + 8 * k, db + (kXTile >> 4) + 2 * k, idesc, 1u);
          }
          tc_commit(oempty + 8 * o);
          if (i + 1 == nst) tc_commit(accfull + 8 * acc);
        }
        __syncwarp();
        o = (o + 1) & (kOS - 1);
      }
      acc ^= 1;
    }
    // every issued MMA has completed before TMEM is given back, also where the epilogue gave up
    if (lane == 0) {
      tc_commit(done);
      mbar_wait(done, 0, MBP_DEV_TIMEOUT_MMA, kDefaultWaitLimitNs);
    }
    __syncwarp();
  } else if (warp < kXWarp) {
    // ---------------- decoders: warp (d, j) = row tile d, chunk j of every stage ----------------
    // A warp may only write its TMEM lane quadrant (warp % 4): the four warps of quadrant q take row tiles 2q and
    // 2q + 1, both chunks.
    const int dw = warp - 2, q = warp & 3, qi = dw >> 2;
    const int d = 2 * q + (qi & 1), j = qi >> 1;
    const uint32_t ta0 = tmem + ((uint32_t)(16 * d) << 16) + (uint32_t)(kAcc * kBN) + 32u * (uint32_t)j;
    const uint32_t xr = base + kMask + dw * kMaskUnitBytes;
    mask_clear(xr, kMaskUnitBytes, lane);
    Ring pr{0, 0}, orr{0, 1};
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += G) {
      const Tile tl = tile_at(t);
      const int rt = tl.expert * R + tl.rb0 + d;
      const bool valid = d < tl.rvalid;  // the box's other rows belong to the next block or lie past the matrix
      uint32_t T0 = 0, T1 = 0;
      EscCursor cur;
      if (valid) {
        const uint32_t b = p.bases[rt];
        T0 = table_lo(b);
        T1 = table_hi(b);
        cur.init(p.esc, p.esc_off[(size_t)rt * C], p.esc_off[(size_t)(rt + 1) * C], lane);
      } else {
        cur.init(p.esc, 0, 0, lane);
      }
      for (int c = j; c < 2 * nst; c += 2) {
        ok = warp_wait(pfull + 8 * pr.i, pr.ph, MBP_DEV_TIMEOUT_FULL, p.wait_ns);
        if (!ok) break;
        const bool live = valid && c < C;
        uint32_t A[16], dep = 0;
        if (live) {
          const unsigned char* u = sm + pr.i * kStage + (p.wsubs * d + j) * kSub + lane * 16;
          const uint4 p0 = *reinterpret_cast<const uint4*>(u);
          const uint4 p1 = *reinterpret_cast<const uint4*>(u + 512);
          const uint4 p2 = *reinterpret_cast<const uint4*>(u + 1024);
          cur.seek((uint32_t)c, lane);
          if (cur.next_chunk == (uint32_t)c) {
            uint32_t tgt[1] = {0u};
            cur.scatter<1>((uint32_t)c, (uint32_t)c + 1, xr, kMaskUnitBytes, lane, tgt);
            __syncwarp();
            uint4 m0, m1;
            take_mask(xr, tgt[0], lane, m0, m1);
            decode_unit_m(p0, p1, p2, T0, T1, m0, m1, A);
          } else {
            decode_unit(p0, p1, p2, T0, T1, A);
          }
          dep = A[0] ^ A[8];  // A[0] depends on p0 and p2, A[8] on p1: every load has returned before the hand-back
        }
        mbar_arrive_dep(pempty + 8 * pr.i, dep);
        pr.next(kPS);
        ok = warp_wait(oempty + 8 * orr.i, orr.ph, MBP_DEV_TIMEOUT_EMPTY, p.wait_ns);
        if (!ok) break;
        tc_fence_after();  // the stores come after the MMAs whose commit freed the stage
        if (live) tc_st_a<false>(ta0 + (uint32_t)(orr.i * 64), A, lane & 3);
        tc_fence_before();  // the stores are complete (wait::st) and ordered before the arrive
        mbar_arrive(afull + 8 * orr.i);
        orr.next(kOS);
      }
    }
  } else {
    // ---------------- epilogue: warp q = the tile's rows 32q .. 32q + 31 ----------------
    const int q = warp - kEpiWarp, r8 = (lane & 3) * 8;
    uint16_t* sm_m = reinterpret_cast<uint16_t*>(sm + kTurn + q * 1024);  // [8 tokens][32 rows]
    uint16_t* sm_r = sm_m + 256;                                             // the residual, then the results
    const auto bf = [](uint16_t u) { return __uint_as_float((uint32_t)u << 16); };
    Ring acc{0, 0};
    for (int t = blockIdx.x; t < tiles; t += G, acc.next(kAcc)) {
      const Tile tl = tile_at(t);
      const int row0 = tl.rb0 * 16 + q * 32, wrows = min(32, tl.rvalid * 16 - q * 32), nt = tl.tend - tl.tok0;
      const float bias = lane < wrows ? epi_bias(p.epi, (long long)tl.expert * R * 16 + row0 + lane) : 0.f;
      epi_prefetch(p.epi, tl.rb0 * 16, (tl.rb0 + tl.rvalid) * 16, tl.tok0, tl.tend, tid - 32 * kEpiWarp, 128);
      // Wide form: 8 tokens x 32 rows at a time turn between "lane = eight rows of a token" (one 16-byte access, lane
      // l: token l / 4, rows 8(l % 4)) and "lane = row" through 1 KB of shared memory.
      uint4 m4 = {}, r4 = {};
      const auto fetch = [&](int c) {
        const long long tk = tl.tok0 + c + (lane >> 2);
        if (r8 < wrows && tk < tl.tend) {
          if (p.epi.mul)
            m4 = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.epi.mul) + tk * p.epi.ld_mul + row0 + r8);
          if (p.epi.residual)
            r4 = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.epi.residual) + tk * p.epi.ld_res + row0 +
                                                 r8);
        }
      };
      if (p.epi.wide) fetch(0);
      if (!warp_wait(accfull + 8 * acc.i, acc.ph, MBP_DEV_TIMEOUT_MMA, p.wait_ns)) break;
      tc_fence_after();
      const uint32_t ta = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc.i * kBN);
#pragma unroll 1
      for (int g = 0; g < nt; g += 8) {
        float y[8];
        tc_ld8(ta + (uint32_t)g, y);
        if (p.epi.wide) {
          if (p.epi.mul) reinterpret_cast<uint4*>(sm_m)[lane] = m4;
          if (p.epi.residual) reinterpret_cast<uint4*>(sm_r)[lane] = r4;
          __syncwarp();
          fetch(g + 8);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] += bias;
          epi_act<8>(y, p.epi.act);
          if (p.epi.mul) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] *= bf(sm_m[i * 32 + lane]);
          }
          if (p.epi.residual) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] += bf(sm_r[i * 32 + lane]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) sm_r[i * 32 + lane] = __bfloat16_as_ushort(__float2bfloat16_rn(y[i]));
          __syncwarp();
          const long long tk = tl.tok0 + g + (lane >> 2);
          if (r8 < wrows && tk < tl.tend)
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + tk * p.ldo + row0 + r8) =
                reinterpret_cast<const uint4*>(sm_r)[lane];
          __syncwarp();
        } else if (lane < wrows) {
          epi_column<8>(p.epi, p.out, p.ldo, y, bias, row0 + lane, tl.tok0 + g, nt - g);
        }
      }
      __syncwarp();
      tc_fence_before();  // the accumulator has been read
      if (lane == 0) mbar_arrive(accfree + 8 * acc.i);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

std::mutex g_mu;
std::map<int, int> g_sms;  // device -> SM count, once the kernel's attributes are set there

int launch(const ExpertParams& p, long long max_tok_tiles, cudaStream_t stream) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return MBP_ERR_LAUNCH;
  {
    std::lock_guard<std::mutex> lk(g_mu);
    auto it = g_sms.find(dev);
    if (it != g_sms.end()) {
      sms = it->second;
    } else {
      if (cudaFuncSetAttribute(k_experts, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) != cudaSuccess)
        return MBP_ERR_SMEM;
      if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return MBP_ERR_LAUNCH;
      g_sms[dev] = sms;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(max_tok_tiles * p.R < sms ? max_tok_tiles * p.R : sms));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_bytes(p.group.experts);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  static const bool pdl = getenv("MBP_NO_PDL") == nullptr;  // MBP_NO_PDL set: plain stream serialisation
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, k_experts, p) == cudaSuccess ? MBP_OK : MBP_ERR_LAUNCH;
}

}  // namespace

extern "C" int mbp_gemm_c12_experts(const mbp_c12* w, int experts, const uint16_t* x, int rows, const int32_t* offsets,
                                    const mbp_epilogue* epi, int zero_tail, void* out, int ldo,
                                    cudaStream_t stream) {
  if (!w || !w->units || !w->bases || !w->esc_off || !x || !offsets || !out) return MBP_ERR_ARG;
  if (w->n_esc > 0 && !w->esc) return MBP_ERR_ARG;
  if (zero_tail != 0 && zero_tail != 1) return MBP_ERR_ARG;
  if (experts < 1 || experts > kMaxExperts || w->n % (16 * experts) || w->k % 64 || w->k / 64 > 32766)
    return MBP_ERR_SHAPE;
  if (rows < 1) return MBP_ERR_M;
  const int n = w->n / experts;
  if (n < 16 || w->k < 64 || ldo < n) return MBP_ERR_SHAPE;
  if (((uintptr_t)x & 15u) || ((uintptr_t)w->units & 15u) || ((uintptr_t)offsets & 3u)) return MBP_ERR_ALIGN;
  ExpertParams p;
  int rc = check_epilogue(epi, n, out, ldo, &p.epi);
  if (rc) return rc;
  const long long tt = max_tiles(experts, rows, kBN);
  p.C = w->k / 64;
  p.R = n / 16;
  if (tt * p.R > 0x7fffffffLL) return MBP_ERR_SHAPE;
  const int R = experts * p.R;
  const TmapKey wkey{w->units, (uint64_t)R, (uint64_t)p.C, 0, 0, 0, 0x202u};
  if (!cached_map(&p.wmap, wkey, [&](CUtensorMap* mp) { return encode_units_3d(mp, w->units, R, p.C, false); }))
    return MBP_ERR_TMAP;
  if (!encode_bf16_2d_cached(&p.xmap, x, (uint64_t)rows, (uint64_t)w->k, (uint64_t)w->k, kBox, 64u,
                             CU_TENSOR_MAP_SWIZZLE_128B))
    return MBP_ERR_TMAP;
  p.bases = w->bases;
  p.esc_off = w->esc_off;
  p.esc = w->esc;
  p.out = out;
  p.ldo = ldo;
  p.wsubs = p.C >= 2 ? 2 : 1;
  p.group = GroupArgs{offsets, experts, rows, zero_tail};
  p.wait_ns = wait_limit_ns();
  return launch(p, tt, stream);
}

int mbp_status_expert_gemm(int* v, int clear) { return read_status_here(v, clear); }
