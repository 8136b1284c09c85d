// Expert products for few rows: out[r] = residual[r] + mul[r] * act(x[r] . W[e(r)]^T + bias[e(r)]) for rows sorted by
// expert, streaming each used expert's packed 12-bit weights once (no counterpart in the reference).
//
// The GEMV's mathematics (gemv.cu: 16 weight rows decoded in registers are the A operand of mma.sync m16n8k16, up to 8
// tokens of one expert an 8-column B operand) on a persistent grid: how many experts a batch uses is known on the
// device only, and a grid of one block per (expert, rows) made for a guess leaves SMs idle in its last round.  The work
// is the list of (token tile, 16-row weight tile) pairs, token tiles counted expert by expert from the borders; CTA b of
// G takes the b-th of G equal parts, so every SM streams the same bytes, in chunks of up to one weight tile per warp out
// of at most two token tiles.  With fewer tiles than warps the warps of a tile split every stage's columns and slice 0
// adds their sums in order.  The producer warp's ring runs on across the chunks, so HBM keeps busy through an epilogue.
// The weights are packed in the tensor cores' pair order (mbp_expert_order), so the B fragments are ldmatrix loads of x
// as it is.
// Bound: HBM.  64 experts of 1536 x 6144, 8 of them per token, 1 / 8 / 30 tokens: 24 / 86 / 139 us (floors of the used
// experts' bytes at the measured copy rate 17 / 78 / 115).  Few tiles leave SMs idle: one token of 2 experts gives a third of
// them two tiles and the rest one, 13.2 us; two experts of 512 x 1024 take 6.3 us, mostly the way to the first load and the
// partial sums' way through shared memory.
// All waits are bounded and reported through the device status word.
#include <cstdlib>
#include <map>
#include <mutex>

#include "common.cuh"
#include "epilogue.cuh"
#include "escape.cuh"
#include "tmap.h"

using namespace mbp;

namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxSmem = 227 * 1024;
constexpr int kWarps = 14;  // consumer warps: 128 registers a thread with the producer
constexpr int kSub = MBP_C12_UNIT_BYTES;

struct __align__(64) Params {
  CUtensorMap xmap;  // x [rows, k] bf16, box 64 columns x 8*MT rows, 128-byte swizzle
  const uint8_t* units;
  const uint8_t* bases;
  const int32_t* esc_off;
  const uint32_t* esc;
  void* out;
  int C, R, ldo, most;  // most: upper bound of the (token tile, weight tile) pairs
  int stage, stages;    // bytes of a stage, ring depth
  int has_esc;
  EpiArgs epi;
  GroupArgs group;
  unsigned long long wait_ns;  // limit of every bounded wait
};

// A stage has room for this many units and x boxes.
constexpr int kUnits = 2 * kWarps;
__host__ __device__ constexpr int boxes_of(int mt) { return mt == 4 ? 4 : 8; }

// Units without escapes decoded per pass (their loads in flight together: 0.6 us of 13 for 2 experts of 1536 x 6144 on
// 8 tokens; wider token tiles have no registers for a second) and independent accumulators per 8 tokens.
__host__ __device__ constexpr int pass_of(int mt) { return mt == 1 ? 2 : 1; }
__host__ __device__ constexpr int accs_of(int mt) { return mt == 1 ? 4 : mt == 2 ? 2 : 1; }

// A chunk of n weight tiles out of nx token tiles: each stage holds kci 64-column chunks of all of them, and slices warps
// share a tile, each taking kci / slices (at most 2, so that a pass has two units' loads in flight).  The fewer the tiles,
// the more warps per tile: 1, 2, 4 or 8 (14 warps on a single tile: 7.6 us instead of 6.6 for 2 experts of 512 x 1024,
// the sums' way through shared memory outweighs the shorter slices).
struct Split {
  int slices, kci;
};

__host__ __device__ inline Split split_of(int n, int nx, int mt) {
  Split s{1, 1};
  while (2 * s.kci * n <= kUnits && 2 * s.kci * nx <= boxes_of(mt)) s.kci *= 2;
  while (2 * s.slices <= s.kci && 2 * s.slices * n <= kWarps) s.slices *= 2;
  return s;
}

struct Layout {
  int masks, mask, part, bars, table, total;
};

// Bytes from the 1024-aligned base: `stages` stages (a stage: its x boxes, then its units), one escape mask per warp, the
// slices' partial sums, barriers, scan scratch (one int per warp) and the first token tile and border of each expert.
__host__ __device__ inline Layout layout(int mt, int stage, int stages, bool esc, int experts) {
  Layout L;
  L.masks = stages * stage;
  L.mask = esc ? kMaskUnitBytes : 0;
  L.part = L.masks + kWarps * L.mask;
  L.bars = L.part + kWarps * mt * 512;
  L.table = L.bars + 16 * (stages + kWarps) + 64;
  L.total = L.table + 8 * (experts + 1);
  return L;
}

MBP_DEV void prefetch_line(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

MBP_DEV void add4(float4& a, const float4 b) {
  a.x += b.x;
  a.y += b.y;
  a.z += b.z;
  a.w += b.w;
}

MBP_DEV bool warp_wait(uint32_t bar, uint32_t parity, int code, uint64_t limit) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, code, limit)) != 0;  // one answer for the whole warp
}

struct Chunk {
  int tt, n, nx, kci, slices;
};

struct TokenTile {
  int expert, tok0, tend;  // tokens [tok0, tend)
};

template <int MT>
__global__ void __launch_bounds__(32 * (kWarps + 1), 1) k_expert_gemv(const __grid_constant__ Params p) {
  constexpr int TOK = 8 * MT, KC = pass_of(MT), NA = accs_of(MT);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char* sm = smem_raw + (base - raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nt = blockDim.x;
  const int E = p.group.experts, C = p.C, R = p.R;
  const Layout L = layout(MT, p.stage, p.stages, p.has_esc != 0, E);
  const uint32_t full = base + L.bars, empty = full + 8 * p.stages;
  const uint32_t psum = empty + 8 * p.stages, pfree = psum + 8 * kWarps;  // a warp's partial sums: written, read
  int* scan = reinterpret_cast<int*>(sm + L.bars + 16 * (p.stages + kWarps));
  int* first = reinterpret_cast<int*>(sm + L.table);  // first token tile of each expert
  int* lo = first + E + 1;                            // its first row
  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, kWarps);
    }
    for (int i = 0; i < kWarps; ++i) {
      mbar_init(psum + 8 * i, 1);
      mbar_init(pfree + 8 * i, 1);
    }
    fence_mbar_init();
    prefetch_tmap(&p.xmap);
  }
  grid_dep_wait();
  grid_dep_launch();

  // ---- the token tiles before each expert (thread i takes the experts [i*q, (i+1)*q)); borders clamped to the rows ----
  const auto border = [&](int e) { return min(max(p.group.offsets[e], 0), p.group.rows); };
  {
    const int q = (E + nt - 1) / nt, e0 = min(E, tid * q), e1 = min(E, e0 + q);
    int sum = 0, at = border(e0);
    for (int e = e0; e < e1; ++e) {
      const int to = border(e + 1);
      first[e] = sum;
      lo[e] = at;
      sum += (max(to - at, 0) + TOK - 1) / TOK;
      at = to;
    }
    if (tid == nt - 1) lo[E] = border(E);
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    int before = inc - sum;
    for (int w = 0; w < warp; ++w) before += scan[w];
    for (int e = e0; e < e1; ++e) first[e] += before;
    if (tid == nt - 1) first[E] = before + sum;
    __syncthreads();
  }

  // ---- this CTA's part of the (token tile, weight tile) list ----
  const long long total = min((long long)first[E] * R, (long long)p.most);
  const int beg = (int)(total * blockIdx.x / gridDim.x), end = (int)(total * (blockIdx.x + 1) / gridDim.x);
  // the expert and rows of a token tile, and how many tiles the chunk at `pos` takes: at most two token tiles' worth
  const auto tile_at = [&](int tt) {
    int l = 0, h = E - 1;  // the last expert whose first token tile is at or before tt (it has rows)
    while (l < h) {
      const int mid = (l + h + 1) >> 1;
      if (first[mid] <= tt)
        l = mid;
      else
        h = mid - 1;
    }
    TokenTile t;
    t.expert = l;
    t.tok0 = lo[l] + (tt - first[l]) * TOK;
    t.tend = min(t.tok0 + TOK, lo[l + 1]);
    return t;
  };
  const auto chunk_at = [&](int pos) {  // at most one weight tile per warp, out of at most two token tiles
    const int left = end - pos, r0 = pos % R;
    Chunk c;
    c.tt = pos / R;
    c.n = min(min(left, kWarps), 2 * R - r0);
    // 8 to 10 tiles would leave a third of the warps idle: 7 with two warps each, then the rest (12 experts of 1536 x 6144,
    // 8 tiles a CTA: 38 -> 36 us), where the columns are long enough for the extra chunk's start (at K = 1536 27.0 -> 28.5)
    if (c.n > kWarps / 2 && c.n <= kWarps - 4 && C >= 64) c.n = kWarps / 2;
    c.nx = r0 + c.n > R ? 2 : 1;
    const Split sp = split_of(c.n, c.nx, MT);
    c.kci = sp.kci;
    c.slices = sp.slices;
    return c;
  };

  if (warp == kWarps) {
    // ---------------- producer ----------------
    const uint64_t pol = policy_evict_first();
    Ring r{0, 1};
    bool ok = true;
    for (int pos = beg; pos < end && ok;) {
      const Chunk c = chunk_at(pos);
      const int n = c.n, nx = c.nx, kci = c.kci, r0 = pos - c.tt * R, nit = (C + kci - 1) / kci;
      // lane l < n copies units of the chunk's tile l; lane 16 + i the x boxes i (of nx * kci, token tile by token tile)
      const int slot = lane < 16 ? (r0 + lane >= R ? 1 : 0) : (lane - 16 >= kci ? 1 : 0), xc = lane - 16 - slot * kci;
      const TokenTile t = tile_at(c.tt + min(slot, nx - 1));
      const uint8_t* src = p.units + ((size_t)t.expert * R + (size_t)max(r0 + lane - slot * R, 0)) * C * kSub;
      if (lane < n) {  // what the consumers read at the chunk's start, a ring's length ahead of them
        const int rt = t.expert * R + r0 + lane - slot * R;
        prefetch_line(p.bases + rt);
        if (p.epi.bias) prefetch_line(static_cast<const char*>(p.epi.bias) + (size_t)rt * (p.epi.bias_f32 ? 64 : 32));
        if (p.has_esc) {
          prefetch_line(p.esc_off + (size_t)rt * C);
          prefetch_line(p.esc_off + (size_t)(rt + 1) * C);
        }
      }
      for (int it = 0; it < nit; ++it, r.next(p.stages)) {
        ok = warp_wait(empty + 8 * r.i, r.ph, MBP_DEV_TIMEOUT_EMPTY, p.wait_ns);
        if (!ok) break;
        const int c0 = it * kci, nk = min(kci, C - c0);
        const uint32_t stage = base + r.i * p.stage, fb = full + 8 * r.i;
        if (lane == 0) mbar_arrive_expect_tx(fb, (uint32_t)nk * (uint32_t)(n * kSub + nx * TOK * 128));
        __syncwarp();
        if (lane < n)
          bulk_g2s_hint(stage + (uint32_t)(nx * kci * TOK * 128 + lane * kci * kSub), src + (size_t)c0 * kSub, (uint32_t)nk * kSub, fb,
                        pol);
        else if (lane >= 16 && slot < nx && xc < nk)
          tma_load_2d(stage + (uint32_t)((lane - 16) * TOK * 128), &p.xmap, (c0 + xc) * 64, t.tok0, fb);
      }
      pos += n;
    }
    drain_ring(full, r, p.stages, MBP_DEV_TIMEOUT_FULL);
  } else {
    // ---------------- consumers: warp sl * n + wt = tile wt of a chunk's n, sl-th part of every stage's columns ----------------
    const uint32_t xr = base + L.masks + warp * L.mask;
    if (L.mask) mask_clear(xr, L.mask, lane);
    float* part = reinterpret_cast<float*>(sm + L.part) + lane * 4;
    uint32_t phases = 0;  // of every warp's partial-sum barriers
    // lane l addresses token l % 8, 16-byte piece l / 8 of a chunk's x rows (0-3; 4-7 are 64 bytes on)
    const uint32_t lm = (uint32_t)((lane & 7) * 128 + (((lane >> 3) ^ (lane & 7)) << 4));
    Ring r{0, 0};
    bool ok = true;
    for (int pos = beg; pos < end && ok;) {
      const Chunk c = chunk_at(pos);
      const int n = c.n, S = c.slices, kci = c.kci, kps = kci / S, nit = (C + kci - 1) / kci, sl = warp / n,
                wt = warp - sl * n;
      const bool mine = sl < S;
      const int tt = (pos + wt) / R, row0 = pos + wt - tt * R;
      const uint32_t xo = tt != c.tt ? (uint32_t)(kci * TOK * 128) : 0u;
      const uint32_t uoff = (uint32_t)(c.nx * kci * TOK * 128 + wt * kci * kSub + lane * 16);
      TokenTile t{0, 0, 0};
      if (mine) t = tile_at(tt);
      const int rt = t.expert * R + row0;
      uint32_t T0 = 0, T1 = 0;
      float2 bias = make_float2(0.f, 0.f);
      EscCursor cur;
      cur.init(p.esc, 0, 0, lane);
      if (mine) {
        const uint32_t b = p.bases[rt];
        T0 = table_lo(b);
        T1 = table_hi(b);
        if (p.has_esc) cur.init(p.esc, p.esc_off[(size_t)rt * C], p.esc_off[(size_t)(rt + 1) * C], lane);
        if (sl == 0) {
          bias = epi_fragment_bias(p.epi, (long long)rt * 16 + (lane >> 2));
          epi_prefetch(p.epi, row0 * 16, row0 * 16 + 16, t.tok0, t.tend, lane, 32);
        }
      }
      float acc[NA][MT][4];
#pragma unroll
      for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int n = 0; n < MT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[a][n][i] = 0.f;

      // J chunks from k0 of a stage on, straight-line code.  ESC (J = 1): escapes restored from this warp's mask.
      const auto pass = [&](uint32_t stage, int k0, uint32_t tgt, auto esc_tag, auto j_tag) {
        constexpr bool ESC = decltype(esc_tag)::value;
        constexpr int J = decltype(j_tag)::value;
        uint4 u[J][3], m0, m1;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int l = 0; l < 3; ++l) u[j][l] = lds128(stage + uoff + (uint32_t)((k0 + j) * kSub + l * 512));
        if constexpr (ESC) {
          take_mask(xr, tgt, lane, m0, m1);
          __syncwarp();  // a branch per lane, and ldmatrix and mma.sync are .sync.aligned
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          uint32_t bx[MT][8];
#pragma unroll
          for (int n = 0; n < MT; ++n) {
            const uint32_t a = stage + xo + lm + (uint32_t)((k0 + j) * TOK * 128 + n * 1024);
            ldmatrix_x4(a, bx[n][0], bx[n][1], bx[n][2], bx[n][3]);
            ldmatrix_x4(a ^ 64u, bx[n][4], bx[n][5], bx[n][6], bx[n][7]);
          }
          uint32_t A[16];
          if constexpr (ESC)
            decode_unit_m(u[j][0], u[j][1], u[j][2], T0, T1, m0, m1, A);
          else
            decode_unit(u[j][0], u[j][1], u[j][2], T0, T1, A);
#pragma unroll
          for (int n = 0; n < MT; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              mma_bf16_16816(acc[(j * 4 + q) % NA][n], A[4 * q], A[4 * q + 1], A[4 * q + 2], A[4 * q + 3], bx[n][2 * q],
                             bx[n][2 * q + 1]);
        }
      };
      for (int it = 0; it < nit; ++it, r.next(p.stages)) {
        ok = warp_wait(full + 8 * r.i, r.ph, MBP_DEV_TIMEOUT_FULL, p.wait_ns);
        if (!ok) break;
        const uint32_t stage = base + r.i * p.stage;
        const int c0 = it * kci;  // a warp without a tile only hands stages back
        const int nk = mine ? min((sl + 1) * kps, C - c0) : 0;
        for (int k0 = sl * kps; k0 < nk;) {
          const int at = c0 + k0;
          if ((int)cur.next_chunk < at) cur.seek((uint32_t)at, lane);  // the other slices'
          if ((int)cur.next_chunk == at) {
            uint32_t tgt[1] = {0u};
            cur.template scatter<1>((uint32_t)at, (uint32_t)(at + 1), xr, kMaskUnitBytes, lane, tgt);
            __syncwarp();
            pass(stage, k0, tgt[0], std::true_type{}, std::integral_constant<int, 1>{});
            k0 += 1;
          } else if (k0 + KC <= nk && (int)cur.next_chunk >= at + KC) {
            pass(stage, k0, 0u, std::false_type{}, std::integral_constant<int, KC>{});
            k0 += KC;
          } else {
            pass(stage, k0, 0u, std::false_type{}, std::integral_constant<int, 1>{});
            k0 += 1;
          }
        }
        // every lane's shared loads of the stage have returned (the accumulators depend on all of them) before lane 0
        // hands it back
        uint32_t dep = 0;
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int n = 0; n < MT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) dep ^= __float_as_uint(acc[a][n][i]);
        dep = __any_sync(0xffffffffu, dep == 0x7FC00001u);
        if (lane == 0) mbar_arrive_dep(empty + 8 * r.i, dep);
      }
      if (ok && mine) {
        // ---- slices 1.. leave their sums in shared memory; slice 0 adds them in order and runs the epilogue ----
        float4 v[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          v[i] = make_float4(acc[0][i][0], acc[0][i][1], acc[0][i][2], acc[0][i][3]);
#pragma unroll
          for (int a = 1; a < NA; ++a) add4(v[i], make_float4(acc[a][i][0], acc[a][i][1], acc[a][i][2], acc[a][i][3]));
        }
        if (sl) {
          ok = warp_wait(pfree + 8 * warp, (phases >> warp & 1u) ^ 1u, MBP_DEV_TIMEOUT_EMPTY, p.wait_ns);
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < MT; ++i) *reinterpret_cast<float4*>(part + (warp * MT + i) * 128) = v[i];
          __syncwarp();
          if (lane == 0) mbar_arrive(psum + 8 * warp);
        } else {
          for (int w = warp + n; w < n * S; w += n) {
            ok = warp_wait(psum + 8 * w, phases >> w & 1u, MBP_DEV_TIMEOUT_FULL, p.wait_ns);
            if (!ok) break;
#pragma unroll
            for (int i = 0; i < MT; ++i) add4(v[i], *reinterpret_cast<const float4*>(part + (w * MT + i) * 128));
            __syncwarp();
            if (lane == 0) mbar_arrive(pfree + 8 * w);
          }
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const int row = row0 * 16 + (lane >> 2), tk = t.tok0 + i * 8 + 2 * (lane & 3);
            if (tk < t.tend) epi_fragment(p.epi, p.out, p.ldo, v[i], bias, row, tk, t.tend - tk);
          }
        }
      }
      phases ^= (1u << n * S) - (1u << n);  // warps n .. n * S - 1 handed their sums on
      pos += n;
    }
    if (p.group.zero_tail)
      zero_tail(p.group, p.epi, p.out, p.ldo, 0, R * 16, blockIdx.x, gridDim.x, tid, 32 * kWarps);
  }
}

using Kernel = void (*)(Params);
Kernel kernel_of(int mt) { return mt == 1 ? k_expert_gemv<1> : mt == 2 ? k_expert_gemv<2> : k_expert_gemv<4>; }

std::mutex g_mu;
std::map<std::pair<int, int>, int> g_sms;  // (device, token tile) -> SM count, once the kernel's attributes are set

}  // namespace

extern "C" int mbp_gemv_c12_experts(const mbp_c12* w, int experts, const uint16_t* x, int rows, const int32_t* offsets,
                                    const mbp_epilogue* epi, int zero_tail, void* out, int ldo, int tile,
                                    cudaStream_t stream) {
  if (!w || !w->units || !w->bases || !w->esc_off || !x || !offsets || !out) return MBP_ERR_ARG;
  if (w->n_esc > 0 && !w->esc) return MBP_ERR_ARG;
  if (zero_tail != 0 && zero_tail != 1) return MBP_ERR_ARG;
  if (experts < 1 || experts > kMaxExperts || w->n % (16 * experts) || w->k % 64 || w->k / 64 > 32766)
    return MBP_ERR_SHAPE;
  if (tile != 0 && tile != 8 && tile != 16 && tile != 32) return MBP_ERR_SPLIT;
  if (rows < 1) return MBP_ERR_M;
  const int n = w->n / experts;
  if (n < 16 || w->k < 64 || ldo < n) return MBP_ERR_SHAPE;
  if (((uintptr_t)x & 15u) || ((uintptr_t)w->units & 15u) || ((uintptr_t)offsets & 3u)) return MBP_ERR_ALIGN;
  Params p;
  int rc = check_epilogue(epi, n, out, ldo, &p.epi);
  if (rc) return rc;
  const int used = experts < rows ? experts : rows;
  // rows per expert, 64 experts of 1536 x 6144, tiles of 8 / 16 / 32: 133 / 139 / 168 us at 3, 168 / 148 / 170 at 6,
  // 274 / 195 / 176 at 12
  if (!tile) tile = rows <= 4LL * used ? 8 : rows <= 10LL * used ? 16 : 32;
  const int mt = tile / 8;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return MBP_ERR_LAUNCH;
  {
    std::lock_guard<std::mutex> lk(g_mu);
    auto it = g_sms.find({dev, mt});
    if (it != g_sms.end()) {
      sms = it->second;
    } else {
      if (cudaFuncSetAttribute(kernel_of(mt), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) != cudaSuccess)
        return MBP_ERR_SMEM;
      if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return MBP_ERR_LAUNCH;
      g_sms[{dev, mt}] = sms;
    }
  }
  p.C = w->k / 64;
  p.R = n / 16;
  p.has_esc = w->n_esc > 0 ? 1 : 0;
  const long long most = max_tiles(experts, rows, tile) * p.R;
  // list positions, and the tiles that any borders can name, stay within 31 bits
  if (most > (1LL << 30) || (long long)experts * (rows / tile + 1) > INT32_MAX) return MBP_ERR_M;
  p.most = (int)most;
  const int grid = (int)(most < sms ? most : sms);
  // No more shared memory than the largest part of the list needs: the next kernel's blocks start beside small ones.
  const int part = (int)((most + grid - 1) / grid), few = p.R < kWarps / 2 ? p.R + 1 : kWarps / 2;
  const int chunks = (part + few - 1) / few;
  p.stage = 0;
  int kmin = p.C;
  for (int i = 1; i <= part && i <= kWarps; ++i)
    for (int nx = 1; nx <= 2 && nx <= i; ++nx) {
      const Split sp = split_of(i, nx, mt);
      const int bytes = (sp.kci * (nx * mt * 1024 + i * kSub) + 1023) & ~1023;
      if (bytes > p.stage) p.stage = bytes;
      if (sp.kci < kmin) kmin = sp.kci;
    }
  const long long need = (long long)chunks * ((p.C + kmin - 1) / kmin);
  p.stages = 2;
  while (p.stages < 8 && p.stages < need && layout(mt, p.stage, p.stages + 1, p.has_esc != 0, experts).total + 1024 <= kMaxSmem)
    ++p.stages;
  const int smem = layout(mt, p.stage, p.stages, p.has_esc != 0, experts).total + 1024;
  if (smem > kMaxSmem) return MBP_ERR_SMEM;
  if (!encode_bf16_2d_cached(&p.xmap, x, (uint64_t)rows, (uint64_t)w->k, (uint64_t)w->k, (uint32_t)tile, 64u,
                             CU_TENSOR_MAP_SWIZZLE_128B))
    return MBP_ERR_TMAP;
  p.units = w->units;
  p.bases = w->bases;
  p.esc_off = w->esc_off;
  p.esc = w->esc;
  p.out = out;
  p.ldo = ldo;
  p.group = GroupArgs{offsets, experts, rows, zero_tail};
  p.wait_ns = wait_limit_ns();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(32 * (kWarps + 1));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  static const bool pdl = getenv("MBP_NO_PDL") == nullptr;  // MBP_NO_PDL set: plain stream serialisation
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel_of(mt), p) == cudaSuccess ? MBP_OK : MBP_ERR_LAUNCH;
}

int mbp_status_expert_gemv(int* v, int clear) { return read_status_here(v, clear); }
