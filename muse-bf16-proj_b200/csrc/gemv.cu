// Weight-streaming GEMV for small token counts: out[m, n] = x[m, k] . W[n, k]^T, FP32 accumulation.
//
// Replaces the reference's family of M <= 32 GEMVs (submission.py: sm_gemv S:46<177-477>, m32_gemv S:416,
// cpstage S:1649/S:1920, smallm2 S:2696, smtrace S:3844, v18d/v18s S:6586/S:6886, router rr_small S:943).
// Same math (swap-AB mma.sync m16n8k16: 16 weight rows are the A operand decoded in registers, 8 tokens are B),
// re-designed for B200:
//
//   * one CTA = one producer warp + `nwc` consumer warps; the CTA tile is rb 16-row tiles x a K range;
//   * per pipeline stage the producer issues, through the TMA engine, one 1-D bulk copy per row tile of `kci`
//     consecutive packed units (>= 6 KB each; the packed matrix is row-tile-major, so no per-geometry
//     re-ordering of the weights is needed) with an L2 evict-first policy, plus one 2-D tensor copy per 64-column
//     chunk of x (128-byte swizzle, so the fragment loads below are bank-conflict free).  Stages are large
//     (tens of KB): B200's TMA engine only reaches HBM bandwidth with large slots and copies;
//   * consumer warp (wr, wk) owns rtw row tiles and the wk-th K slice; per stage it loads its units with plain
//     shared loads first (instruction-level parallelism across units), decodes each 1536-byte unit in registers
//     (3 prmt per 8 weights), patches escapes through an unbounded per-tile list (escape.cuh) and issues 4*MT
//     mma.sync per unit into several independent accumulators;
//   * split-K: the wki K slices reduce through shared memory, the `split` CTAs of a thread-block cluster push
//     their partials into the owning CTA through distributed shared memory, each rank summing and storing
//     1/split of the tile; without a K split every warp stores its sums straight from registers;
//   * tensor-parallel exchange (output kinds MBP_OUT_TAGGED_*): the results go to every rank's exchange buffer as
//     epoch-tagged 64-bit words over NVLink, and with a fused receive each CTA then gathers (or sums, in rank
//     order) its tiles from every rank into the output, the grid's last CTA advancing the epoch;
//   * epilogue instances (kOutEpi): bias, activation, multiplier and residual on the FP32 sums before the store;
//   * every wait is bounded and reports through the device status word (no trap).
//
// The same kernel serves the FP32 router (S:854, S:941, S:943, S:5377, S:5424) with hi/lo BF16 units: two
// mma.sync per k-step into one FP32 accumulator.
#include <cstdlib>
#include <map>
#include <mutex>
#include <tuple>
#include <type_traits>

#include "common.cuh"
#include "epilogue.cuh"
#include "escape.cuh"
#include "tmap.h"

using namespace mbp;

namespace {

enum { FMT_C12 = 0, FMT_HILO = 1 };
enum { kOutEpi = 4 };  // output kind past MBP_OUT_*: one output through the epilogue, BF16 or FP32

constexpr int kMaxThreads = 384;  // 11 consumer warps + 1 producer (up to 168 registers per thread)
constexpr int kMaxSmem = 227 * 1024;
constexpr int kMaxConsumerWarps = 11;
constexpr int kMaxOuts = 8;  // local output + up to 7 peers

struct __align__(64) GemvParams {
  CUtensorMap xmap;  // x [m, k] bf16, box 64 columns x 8*MT rows, 128-byte swizzle
  const uint8_t* units;
  const uint8_t* bases;
  const int32_t* esc_off;
  const uint32_t* esc;
  void* outs[kMaxOuts];  // outs[0] local; the others peers' buffers (tensor-parallel peer stores), same layout
  // Tensor-parallel exchange (the tagged output kinds): outputs are epoch-tagged 64-bit words (ldo in words), this
  // call's epoch is *epoch + 1 and every output pointer moves by parity_stride bytes when it is odd:
  // MBP_OUT_TAGGED_BF16X2 word (tk, 8*tile + g) = rows 16*tile + g and + 8 as two bf16; MBP_OUT_TAGGED_F32 word
  // (tk, row) = one f32.  A word and its tag travel in one 64-bit store, so a reader needs no fence.
  const int* epoch;
  long long parity_stride;
  // Fused receive (tagged kinds with `rout` set): this rank's exchange buffer, the projection output [m][rn], the
  // rank count, and the epoch counter (MBP_TP_COUNTER_SLOTS slots + ticket) the grid's last CTA advances.
  const uint8_t* rbuf;
  void* rout;
  int* ctr;
  int rn, rP;
  // Row-parallel reduce-scatter + gather (MBP_TP_RSAG, tagged f32 words with `rout` set): CTA (x, z)'s tiles are
  // owned by rank (x + z) % rP; partials go to the owner only, the owner sums them and sends the BF16 result as
  // bf16x2 words into every rank's gather region (byte offset goff of each buffer half; peer o's region is
  // outs[o] + gdelta).
  int rsag, rrank;
  long long goff, gdelta;
  EpiArgs epi;  // kOutEpi
  int nout;
  int C;     // 64-column chunks (k / 64)
  int Rout;  // 16-row tiles computed (n_out / 16)
  int m;     // tokens
  int ldo;   // leading dimension of out (elements)
  int rb, split, wki, kci, stages;
  int nblk;     // row blocks: block b owns row tiles [b*Rout/nblk, (b+1)*Rout/nblk), at most rb of them
  int has_esc;  // the matrix has escapes: consumer warps get escape masks
  int pre_stages;  // pipeline stages whose weights are prefetched into L2 before the dependency wait
  unsigned long long wait_ns;  // limit of every bounded wait
};

// Chunks per unrolled consumer pass and independent accumulators per (row tile, token tile), sized so that a
// pass's unit loads, B fragments and accumulators fit in 128 registers without spills.
__host__ __device__ constexpr int kc_for(int fmt, int mt, int rtw) {
  return rtw == 2 ? (fmt == FMT_C12 && mt == 1 ? 2 : 1)
                  : fmt == FMT_C12 ? (mt <= 2 ? 4 : 1) : (mt == 1 ? 2 : 1);
}
__host__ __device__ constexpr int na_for(int fmt, int mt, int rtw) {
  return rtw == 2 ? (mt == 1 ? 2 : 1) : mt == 4 ? 1 : 2 + 2 * (fmt == FMT_C12 && mt == 1);
}
// Chunks per escape mask group (a multiple of the pass): the pass itself for one row tile per warp, two chunks
// (4 unit masks) for two row tiles per warp, whose passes are a single chunk.
__host__ __device__ constexpr int mg_for(int fmt, int mt, int rtw) {
  return rtw == 2 && kc_for(fmt, mt, rtw) < 2 ? 2 : kc_for(fmt, mt, rtw);
}

template <int I, int N, class F>
MBP_DEV void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<I + 1, N>(f);
  }
}

struct Layout {
  int xplane;   // bytes of one staged x chunk: 8*MT rows x 128 bytes
  int xbytes;   // x bytes per stage
  int sbytes;   // stage bytes (multiple of 1024)
  int ring;     // ring bytes (also holds the split-K reduction after the main loop)
  int mask;     // escape mask bytes per consumer warp: one 1 KB mask per unit of a mask group (0 without escapes)
  int xr_off;   // per-warp escape masks
  int bar_off;  // full[stages], empty[stages]
  int total;    // bytes from the 1024-aligned base
};

__host__ __device__ inline Layout make_layout(int fmt, int mt, int rb, int rtw, int wki, int kci, int stages,
                                              bool esc) {
  const int ub = fmt == FMT_C12 ? MBP_C12_UNIT_BYTES : 2 * MBP_RAW_UNIT_BYTES;
  Layout L;
  L.xplane = 8 * mt * 128;
  L.xbytes = wki * kci * L.xplane;
  const int wbytes = rb * wki * kci * ub;
  L.sbytes = (L.xbytes + wbytes + 1023) & ~1023;
  int ring = stages * L.sbytes;
  const int red = (wki + 1) * rb * mt * 32 * 16 + 256;  // + the split-K slots' rounding (< 16 items)
  if (red > ring) ring = red;
  L.ring = (ring + 127) & ~127;
  L.mask = (fmt == FMT_C12 && esc) ? mg_for(fmt, mt, rtw) * rtw * kMaskUnitBytes : 0;
  L.xr_off = L.ring;
  L.bar_off = L.xr_off + (rb / rtw) * wki * L.mask;
  L.total = L.bar_off + 2 * stages * 8;
  return L;
}

inline int smem_request(const Layout& L) { return L.total + 1024; }  // + alignment slack

template <int FMT>
struct Fmt;
template <>
struct Fmt<FMT_C12> {
  static constexpr int UB = MBP_C12_UNIT_BYTES;
};
template <>
struct Fmt<FMT_HILO> {
  static constexpr int UB = 2 * MBP_RAW_UNIT_BYTES;
};

// Fills i0 .. i1 - 1 of the ring have landed, under the default limit: a wait gave up, and the block must not end (nor use
// the ring for its sums) while the copy engine still writes to its shared memory.  Off the normal path, where waiting for
// the last copies in the producer held up the block's reduction (0.15 us a call).
__device__ __noinline__ void await_copies(uint32_t full0, int stages, int i0, int i1) {
  for (int i = i0; i < i1; ++i)
    mbar_wait(full0 + 8 * (i % stages), (uint32_t)(i / stages) & 1u, MBP_DEV_TIMEOUT_FULL, kDefaultWaitLimitNs);
}

MBP_DEV void store_out(uint16_t* o, float v) { *o = __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
MBP_DEV void store_out(float* o, float v) { *o = v; }
MBP_DEV uint32_t bf16x2_bits(float lo, float hi) {
  return __bfloat16_as_ushort(__float2bfloat16_rn(lo)) | (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(hi)) << 16;
}

// The four results (row, tk), (row + 8, tk), (row, tk + 1), (row + 8, tk + 1) of one accumulator as words tagged
// with `epoch` into every output (the buffer of the epoch's parity).
template <int OUTK>
MBP_DEV void emit_tagged(const GemvParams& p, float4 v, int row, int tk, uint32_t epoch, int owner) {
  const uint64_t tag = (uint64_t)epoch << 32;
  const long long par = (long long)(epoch & 1u) * p.parity_stride;
  for (int o = 0; o < p.nout; ++o) {
    if (p.rsag && o != owner) continue;  // reduce-scatter: the partials go to the tiles' owner only
    uint64_t* out = reinterpret_cast<uint64_t*>(static_cast<char*>(p.outs[o]) + par);
    if constexpr (OUTK == MBP_OUT_TAGGED_BF16X2) {
      const int j = (row >> 4) * 8 + (row & 7);  // word of rows (16*tile + g, 16*tile + g + 8), g = row % 8
      if (tk < p.m) st_relaxed_sys_u64(out + (size_t)tk * p.ldo + j, tag | bf16x2_bits(v.x, v.z));
      if (tk + 1 < p.m) st_relaxed_sys_u64(out + (size_t)(tk + 1) * p.ldo + j, tag | bf16x2_bits(v.y, v.w));
    } else {
      if (tk < p.m) {
        st_relaxed_sys_u64(out + (size_t)tk * p.ldo + row, tag | __float_as_uint(v.x));
        st_relaxed_sys_u64(out + (size_t)tk * p.ldo + row + 8, tag | __float_as_uint(v.z));
      }
      if (tk + 1 < p.m) {
        st_relaxed_sys_u64(out + (size_t)(tk + 1) * p.ldo + row, tag | __float_as_uint(v.y));
        st_relaxed_sys_u64(out + (size_t)(tk + 1) * p.ldo + row + 8, tag | __float_as_uint(v.w));
      }
    }
  }
}

// Eight consecutive tagged words: all eight loads are issued before any is checked (one round trip when they
// have arrived), then each word not yet carrying the epoch is waited for (bounded).
MBP_DEV void wait_tags8(const uint64_t* w, uint32_t (&d)[8], uint32_t epoch, uint64_t& t0, bool& dead,
                        uint64_t limit) {
  uint64_t v[8];
#pragma unroll
  for (int g = 0; g < 8; ++g) v[g] = ld_relaxed_sys_u64(w + g);
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    if ((uint32_t)(v[g] >> 32) != epoch) v[g] = wait_tag(w + g, epoch, t0, dead, limit);
    d[g] = (uint32_t)v[g];
  }
}

// Fused receive of one CTA: the tiles this CTA computed (row tiles r0 .. r0+rvalid-1, tokens tok0 .. of this
// token block), as every rank computed them, from this rank's exchange buffer into the output.  Items are split
// over i0, i0 + istride, ... (the cluster's CTAs share them).
//   gather (column-parallel): item (q, rr, t) = 8 words of rank q's shard -> 16 BF16 of out row t, columns
//                             q*ns + (r0+rr)*16 .. +15 (ns = this shard's rows);
//   sum (row-parallel):       item (rr, t, quad) = 4 consecutive rows, the P ranks' FP32 partials added in rank
//                             order -> 4 BF16.
template <int OUTK, int TOK>
MBP_DEV void tp_receive(const GemvParams& p, uint32_t epoch, int r0, int rvalid, int tok0, int i0, int istride) {
  const uint64_t* words = reinterpret_cast<const uint64_t*>(p.rbuf + (long long)(epoch & 1u) * p.parity_stride);
  const int ntok = min(TOK, p.m - tok0);
  if (ntok <= 0 || rvalid <= 0) return;
  uint64_t t0 = 0;
  bool dead = false;
  if constexpr (OUTK == MBP_OUT_TAGGED_BF16X2) {
    const int ns = p.Rout * 16, half = p.rn / 2, per_q = rvalid * ntok;
    for (int it = i0; it < p.rP * per_q; it += istride) {
      const int q = it / per_q, rest = it - q * per_q, rr = rest / ntok, t = tok0 + rest - rr * ntok;
      const uint64_t* w = words + (size_t)t * half + q * (ns / 2) + (r0 + rr) * 8;
      uint32_t d[8];
      wait_tags8(w, d, epoch, t0, dead, p.wait_ns);
      uint4 lo, hi;
      lo.x = (d[0] & 0xffffu) | d[1] << 16;
      lo.y = (d[2] & 0xffffu) | d[3] << 16;
      lo.z = (d[4] & 0xffffu) | d[5] << 16;
      lo.w = (d[6] & 0xffffu) | d[7] << 16;
      hi.x = (d[0] >> 16) | (d[1] & 0xffff0000u);
      hi.y = (d[2] >> 16) | (d[3] & 0xffff0000u);
      hi.z = (d[4] >> 16) | (d[5] & 0xffff0000u);
      hi.w = (d[6] >> 16) | (d[7] & 0xffff0000u);
      uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.rout) + (size_t)t * p.rn + q * ns + (r0 + rr) * 16);
      o[0] = lo;
      o[1] = hi;
    }
  } else {
    const int per_r = ntok * 4;
    for (int it = i0; it < rvalid * per_r; it += istride) {
      const int rr = it / per_r, rest = it - rr * per_r, t = tok0 + (rest >> 2), row = (r0 + rr) * 16 + (rest & 3) * 4;
      float a[4];
      for (int q = 0; q < p.rP; ++q) {
        const uint64_t* w = words + ((size_t)q * p.m + t) * p.rn + row;
        uint64_t v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = ld_relaxed_sys_u64(w + j);  // one round trip for the four
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if ((uint32_t)(v[j] >> 32) != epoch) v[j] = wait_tag(w + j, epoch, t0, dead, p.wait_ns);
          const float f = __uint_as_float((uint32_t)v[j]);
          a[j] = q == 0 ? f : a[j] + f;
        }
      }
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.rout) + (size_t)t * p.rn + row) =
          make_uint2(bf16x2_bits(a[0], a[1]), bf16x2_bits(a[2], a[3]));
    }
  }
}

// Fused receive of the row-parallel reduce-scatter + gather (MBP_TP_RSAG) for one CTA's tiles (rows
// (r0 .. r0+rvalid-1) x 16, tokens tok0 ..).  On the tiles' owner: item (rr, t, g) = rows 16(r0+rr) + g and + 8 of
// token t, the P ranks' partials added in rank order (the same sum the all-to-all form makes), rounded to BF16,
// written to the output and sent as one bf16x2 word to every other rank's gather region.  On the other ranks:
// item (rr, t) = the owner's 8 words of that tile row -> 16 BF16 of the output.
template <int TOK>
MBP_DEV void tp_receive_rsag(const GemvParams& p, uint32_t epoch, int r0, int rvalid, int tok0, int i0, int istride,
                             int owner) {
  const long long par = (long long)(epoch & 1u) * p.parity_stride;
  const uint64_t* words = reinterpret_cast<const uint64_t*>(p.rbuf + par);
  const int ntok = min(TOK, p.m - tok0);
  if (ntok <= 0 || rvalid <= 0) return;
  const int half = p.rn / 2;
  uint64_t t0 = 0;
  bool dead = false;
  if (p.rrank == owner) {
    const uint64_t tag = (uint64_t)epoch << 32;
    const int per_r = ntok * 8;
    for (int it = i0; it < rvalid * per_r; it += istride) {
      const int rr = it / per_r, rest = it - rr * per_r, t = tok0 + (rest >> 3), g = rest & 7;
      const int row = (r0 + rr) * 16 + g;
      // every rank's two words loaded before any is checked: one round trip once they have all arrived
      const size_t qs = (size_t)p.m * p.rn;
      const uint64_t* w0 = words + (size_t)t * p.rn + row;
      uint64_t v[2 * kMaxOuts];
#pragma unroll
      for (int q = 0; q < kMaxOuts; ++q)
        if (q < p.rP) {
          v[2 * q] = ld_relaxed_sys_u64(w0 + q * qs);
          v[2 * q + 1] = ld_relaxed_sys_u64(w0 + q * qs + 8);
        }
      float a0 = 0.f, a1 = 0.f;
#pragma unroll
      for (int q = 0; q < kMaxOuts; ++q)
        if (q < p.rP) {
          if ((uint32_t)(v[2 * q] >> 32) != epoch) v[2 * q] = wait_tag(w0 + q * qs, epoch, t0, dead, p.wait_ns);
          if ((uint32_t)(v[2 * q + 1] >> 32) != epoch)
            v[2 * q + 1] = wait_tag(w0 + q * qs + 8, epoch, t0, dead, p.wait_ns);
          const float f0 = __uint_as_float((uint32_t)v[2 * q]), f1 = __uint_as_float((uint32_t)v[2 * q + 1]);
          a0 = q == 0 ? f0 : a0 + f0;
          a1 = q == 0 ? f1 : a1 + f1;
        }
      const uint32_t b2 = bf16x2_bits(a0, a1);
      uint16_t* o = static_cast<uint16_t*>(p.rout) + (size_t)t * p.rn + row;
      o[0] = (uint16_t)(b2 & 0xffffu);
      o[8] = (uint16_t)(b2 >> 16);
      const size_t wi = (size_t)t * half + (r0 + rr) * 8 + g;
      for (int q = 0; q < p.rP; ++q) {
        if (q == p.rrank) continue;
        uint64_t* gq = reinterpret_cast<uint64_t*>(static_cast<char*>(p.outs[q]) + p.gdelta + par);
        st_relaxed_sys_u64(gq + wi, tag | b2);
      }
    }
  } else {
    const uint64_t* gw = reinterpret_cast<const uint64_t*>(p.rbuf + p.goff + par);
    for (int it = i0; it < rvalid * ntok; it += istride) {
      const int rr = it / ntok, t = tok0 + it - rr * ntok;
      const uint64_t* w = gw + (size_t)t * half + (r0 + rr) * 8;
      uint32_t d[8];
      wait_tags8(w, d, epoch, t0, dead, p.wait_ns);
      uint4 lo, hi;
      lo.x = (d[0] & 0xffffu) | d[1] << 16;
      lo.y = (d[2] & 0xffffu) | d[3] << 16;
      lo.z = (d[4] & 0xffffu) | d[5] << 16;
      lo.w = (d[6] & 0xffffu) | d[7] << 16;
      hi.x = (d[0] >> 16) | (d[1] & 0xffff0000u);
      hi.y = (d[2] >> 16) | (d[3] & 0xffff0000u);
      hi.z = (d[4] >> 16) | (d[5] & 0xffff0000u);
      hi.w = (d[6] >> 16) | (d[7] & 0xffff0000u);
      uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.rout) + (size_t)t * p.rn + (r0 + rr) * 16);
      o[0] = lo;
      o[1] = hi;
    }
  }
}

// The grid's last CTA (ticket = grid size - 1) advances the exchange epoch: every CTA read it before taking its
// ticket, and the next kernel reads it only after this grid has completed.
// (No static shared memory: the kernels take the whole dynamic allowance; a barrier with predicate broadcasts.)
MBP_DEV void tp_advance_epoch(int* ctr, int tid) {
  __syncthreads();
  int mine = 0;
  if (tid == 0) {
    const unsigned total = gridDim.x * gridDim.y * gridDim.z;
    mine = atomicAdd(reinterpret_cast<unsigned*>(ctr + MBP_TP_COUNTER_SLOTS), 1u) == total - 1;
  }
  if (__syncthreads_or(mine)) {
    if (tid < MBP_TP_COUNTER_SLOTS) ctr[tid] += 1;
    if (tid == 0) ctr[MBP_TP_COUNTER_SLOTS] = 0;
  }
}

// OUTK: MBP_OUT_BF16 / MBP_OUT_F32 plain outputs, MBP_OUT_TAGGED_BF16X2 / MBP_OUT_TAGGED_F32 exchange words.
template <int FMT, int MT, int RTW, int OUTK>
__global__ void __launch_bounds__(kMaxThreads, 1) k_gemv(const __grid_constant__ GemvParams p) {
  constexpr bool F32OUT = OUTK == MBP_OUT_F32 || OUTK == MBP_OUT_TAGGED_F32;
  using OutT = typename std::conditional<F32OUT, float, uint16_t>::type;
  constexpr int UB = Fmt<FMT>::UB;
  constexpr int TOK = 8 * MT;
  constexpr int KC = kc_for(FMT, MT, RTW);  // chunks per unrolled pass
  constexpr int NA = na_for(FMT, MT, RTW);  // independent accumulators per (row tile, token tile)
  constexpr int MG = mg_for(FMT, MT, RTW);  // chunks per escape mask group
  static_assert(MG % KC == 0, "a mask group is a whole number of passes");
  constexpr int NL = FMT == FMT_C12 ? 3 : 8;         // 16-byte loads per lane per unit
  extern __shared__ __align__(128) unsigned char smem_raw[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows_w = p.rb / RTW;
  const int nwc = rows_w * p.wki;
  const Layout L = make_layout(FMT, MT, p.rb, RTW, p.wki, p.kci, p.stages, p.has_esc != 0);
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t sbase = (raw_base + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (sbase - raw_base);
  const uint32_t full0 = sbase + L.bar_off, empty0 = full0 + 8 * p.stages;

  const int r0 = (int)((long long)blockIdx.x * p.Rout / p.nblk);
  const int rvalid = (int)((long long)(blockIdx.x + 1) * p.Rout / p.nblk) - r0;  // <= rb
  const int tok0 = blockIdx.z * TOK;
  const int s = blockIdx.y;
  const int cs = (int)((long long)s * p.C / p.split), ce = (int)((long long)(s + 1) * p.C / p.split);
  const int Lk = (ce - cs + p.wki - 1) / p.wki;  // chunks per K slice
  const int nit = (Lk + p.kci - 1) / p.kci;

  // Launched as a programmatic dependent of the previous kernel in the stream: the packed weights never depend
  // on it, so the producer warp starts pulling the first stages' weights into L2 while that kernel drains; every
  // thread then waits for it to complete (x, the output and the exchange epoch may be its output / input) before
  // any other access.  (Filling the shared-memory ring itself before the wait measured no faster.)
  // The ring barriers and the x tensor map do not depend on it either.
  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, nwc);
    }
    fence_mbar_init();
  }
  if (warp == nwc) {
    if (lane == 0) prefetch_tmap(&p.xmap);
    const int per_it = rvalid * p.wki, npre = min(p.pre_stages, nit) * per_it;
    for (int i = lane; i < npre; i += 32) {
      const int it = i / per_it, rr = (i - it * per_it) / p.wki, q = i - it * per_it - rr * p.wki;
      const int c0 = cs + q * Lk + it * p.kci, e = min(cs + (q + 1) * Lk, ce);
      const int nk = min(p.kci, e - c0);
      if (nk > 0) prefetch_l2(p.units + ((size_t)(r0 + rr) * p.C + c0) * UB, (uint32_t)nk * UB);
    }
  }
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch();
  if constexpr (OUTK == kOutEpi) {
    if (s == 0) epi_prefetch(p.epi, r0 * 16, (r0 + rvalid) * 16, tok0, min(tok0 + TOK, p.m), tid, blockDim.x);
  }

  float acc[RTW][NA][MT][4];
#pragma unroll
  for (int j = 0; j < RTW; ++j)
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int n = 0; n < MT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[j][a][n][c] = 0.f;

  const int wr = warp % rows_w, wk = warp / rows_w;
  if (warp == nwc) {
    // ---------------- producer ----------------
    const uint64_t pol = policy_evict_first();
    for (int it = 0; it < nit; ++it) {
      const int st = it % p.stages;
      const uint32_t ph = (uint32_t)(it / p.stages) & 1u;
      if (it >= p.stages && !mbar_wait(empty0 + 8 * st, ph ^ 1u, MBP_DEV_TIMEOUT_EMPTY, p.wait_ns)) {
        await_copies(full0, p.stages, it - p.stages, it);
        break;
      }
      uint32_t bytes = 0;
      for (int q = 0; q < p.wki; ++q) {
        const int c0 = cs + q * Lk + it * p.kci, e = min(cs + (q + 1) * Lk, ce);
        const int nk = max(0, min(p.kci, e - c0));
        bytes += (uint32_t)nk * (uint32_t)(rvalid * UB + L.xplane);
      }
      const uint32_t stage = sbase + st * L.sbytes, fb = full0 + 8 * st;
      if (lane == 0) mbar_arrive_expect_tx(fb, bytes);
      __syncwarp();
      for (int i = lane; i < rvalid * p.wki; i += 32) {
        const int rr = i / p.wki, q = i - rr * p.wki;
        const int c0 = cs + q * Lk + it * p.kci, e = min(cs + (q + 1) * Lk, ce);
        const int nk = min(p.kci, e - c0);
        if (nk > 0)
          bulk_g2s_hint(stage + L.xbytes + (uint32_t)((rr * p.wki + q) * p.kci) * UB,
                        p.units + ((size_t)(r0 + rr) * p.C + c0) * UB, (uint32_t)nk * UB, fb, pol);
      }
      for (int i = lane; i < p.wki * p.kci; i += 32) {
        const int q = i / p.kci, jc = i - q * p.kci;
        const int c0 = cs + q * Lk + it * p.kci, e = min(cs + (q + 1) * Lk, ce);
        if (c0 + jc < e) tma_load_2d(stage + (uint32_t)(i * L.xplane), &p.xmap, (c0 + jc) * 64, tok0, fb);
      }
    }
  } else {
    // ---------------- consumers ----------------
    const int b = cs + wk * Lk, e = min(cs + (wk + 1) * Lk, ce);
    bool rvalid_j[RTW];
#pragma unroll
    for (int j = 0; j < RTW; ++j) rvalid_j[j] = wr * RTW + j < rvalid;
    uint32_t T0[RTW], T1[RTW];
    EscCursor cur[RTW];
    const uint32_t xr = sbase + L.xr_off + warp * L.mask;  // mask of (group chunk s, tile j): xr + (s*RTW + j) KB
    if constexpr (FMT == FMT_C12) {
      if (L.mask) mask_clear(xr, L.mask, lane);
#pragma unroll
      for (int j = 0; j < RTW; ++j) {
        const int rt = r0 + wr * RTW + j;
        T0[j] = T1[j] = 0;
        if (rvalid_j[j] && b < e) {
          const uint32_t base = p.bases[rt];
          T0[j] = table_lo(base);
          T1[j] = table_hi(base);
        }
        if (rvalid_j[j] && b < e && p.has_esc)
          cur[j].init(p.esc, p.esc_off[(size_t)rt * p.C + b], p.esc_off[(size_t)rt * p.C + e], lane);
        else
          cur[j].init(p.esc, 0, 0, lane);
      }
    }
    const int g = lane >> 2, t = lane & 3;
    // byte offsets inside a stage, fixed for this warp
    uint32_t uoff[RTW];
#pragma unroll
    for (int j = 0; j < RTW; ++j)
      uoff[j] = (uint32_t)L.xbytes + (uint32_t)((min(wr * RTW + j, p.rb - 1) * p.wki + wk) * p.kci) * UB + lane * 16;
    const uint32_t xoff = (uint32_t)(wk * p.kci * L.xplane + g * 128);
    const uint32_t swz0 = ((2 * t) ^ g) << 4, swz1 = ((2 * t + 1) ^ g) << 4;

    // One pass of KC chunks [c0 + cl0, c0 + min(cl0 + KC, nk)), pass PI of its mask group.  ESC selects the
    // variant that restores escapes from the group's masks; a group whose chunks hold none of this warp's
    // escapes runs the variant without any escape code.  FULL passes (all KC chunks present, the common case)
    // are straight-line code, so the compiler interleaves the decode of one unit with the mma of another.
    // A second tile past the block's valid rows (RTW = 2) is decoded from zero tables and never stored.
    auto pass_fn = [&](const unsigned char* stage, int cl0, int nk, const uint32_t(&tgt)[RTW][MG], auto esc_tag,
                       auto full_tag, auto pi_tag) {
      constexpr bool ESC = decltype(esc_tag)::value;
      constexpr bool FULL = decltype(full_tag)::value;
      constexpr int S0 = decltype(pi_tag)::value * KC;  // first mask slot of this pass
      uint4 u[KC][RTW][NL];  // all units of the pass first: independent shared loads in flight together
#pragma unroll
      for (int jc = 0; jc < KC; ++jc)
#pragma unroll
        for (int j = 0; j < RTW; ++j) {
          const uint4* src = reinterpret_cast<const uint4*>(stage + uoff[j] + (cl0 + jc) * UB);
#pragma unroll
          for (int l = 0; l < NL; ++l) u[jc][j][l] = src[l * 32];
        }
      uint4 mk[ESC ? KC : 1][RTW][2];
      if constexpr (ESC) {
#pragma unroll
        for (int jc = 0; jc < KC; ++jc)
#pragma unroll
          for (int j = 0; j < RTW; ++j)
            take_mask(xr + (uint32_t)((S0 + jc) * RTW + j) * kMaskUnitBytes, tgt[j][S0 + jc], lane, mk[jc][j][0],
                      mk[jc][j][1]);
      }
#pragma unroll
      for (int jc = 0; jc < KC; ++jc) {
        const int cl = cl0 + jc;  // chunk within the stage
        if constexpr (!FULL) {
          if (cl >= nk) break;
        }
        const unsigned char* xrow = stage + xoff + cl * L.xplane;
        uint32_t bx[MT][8];
#pragma unroll
        for (int n = 0; n < MT; ++n) {
          const uint4 v0 = *reinterpret_cast<const uint4*>(xrow + n * 1024 + swz0);
          const uint4 v1 = *reinterpret_cast<const uint4*>(xrow + n * 1024 + swz1);
          bx[n][0] = v0.x; bx[n][1] = v0.y; bx[n][2] = v0.z; bx[n][3] = v0.w;
          bx[n][4] = v1.x; bx[n][5] = v1.y; bx[n][6] = v1.z; bx[n][7] = v1.w;
        }
#pragma unroll
        for (int j = 0; j < RTW; ++j) {
          uint32_t A[16];
          if constexpr (FMT == FMT_C12) {
            if constexpr (ESC)
              decode_unit_m(u[jc][j][0], u[jc][j][1], u[jc][j][2], T0[j], T1[j], mk[jc][j][0], mk[jc][j][1], A);
            else
              decode_unit(u[jc][j][0], u[jc][j][1], u[jc][j][2], T0[j], T1[j], A);
#pragma unroll
            for (int n = 0; n < MT; ++n)
#pragma unroll
              for (int q = 0; q < 4; ++q)
                mma_bf16_16816(acc[j][(jc * 4 + q) % NA][n], A[4 * q], A[4 * q + 1], A[4 * q + 2], A[4 * q + 3],
                               bx[n][2 * q], bx[n][2 * q + 1]);
          } else {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const uint4 v = u[jc][j][4 * h + q];
                  A[4 * q] = v.x; A[4 * q + 1] = v.y; A[4 * q + 2] = v.z; A[4 * q + 3] = v.w;
                }
#pragma unroll
                for (int n = 0; n < MT; ++n)
#pragma unroll
                  for (int q = 0; q < 4; ++q)
                    mma_bf16_16816(acc[j][(jc * 4 + q) % NA][n], A[4 * q], A[4 * q + 1], A[4 * q + 2],
                                   A[4 * q + 3], bx[n][2 * q], bx[n][2 * q + 1]);
              }
            }
          }
        }
    };

    for (int it = 0; it < nit; ++it) {
      const int st = it % p.stages;
      const uint32_t ph = (uint32_t)(it / p.stages) & 1u;
      if (!mbar_wait(full0 + 8 * st, ph, MBP_DEV_TIMEOUT_FULL, p.wait_ns)) {
        await_copies(full0, p.stages, it, min(it + p.stages, nit));  // the producer may have ended: its last ring of copies
        break;
      }
      const unsigned char* stage = smem + st * L.sbytes;
      const int c0 = b + it * p.kci;
      const int nk = rvalid_j[0] ? max(0, min(p.kci, e - c0)) : 0;  // a warp without valid rows only drains
      // Mask groups of MG chunks: one escape scatter and one __syncwarp per group, then MG / KC passes.
      for (int g0 = 0; g0 < nk; g0 += MG) {
        const int gend = min(g0 + MG, nk);
        uint32_t tgt[RTW][MG];  // lanes holding escape bytes, per (tile, chunk) of the group
        bool esc_here = false;
        if constexpr (FMT == FMT_C12) {
#pragma unroll
          for (int j = 0; j < RTW; ++j) esc_here |= (int)cur[j].next_chunk < c0 + gend;
          if (esc_here) {
#pragma unroll
            for (int j = 0; j < RTW; ++j) {
#pragma unroll
              for (int s = 0; s < MG; ++s) tgt[j][s] = 0u;
              if ((int)cur[j].next_chunk < c0 + gend)
                cur[j].template scatter<MG>((uint32_t)(c0 + g0), (uint32_t)(c0 + gend),
                                            xr + (uint32_t)j * kMaskUnitBytes, RTW * kMaskUnitBytes, lane, tgt[j]);
            }
            __syncwarp();
          }
        }
        static_for<0, MG / KC>([&](auto pi) {
          const int cl0 = g0 + decltype(pi)::value * KC;
          if (cl0 >= nk) return;
          const bool full = cl0 + KC <= nk;
          if constexpr (FMT == FMT_C12) {
            if (esc_here) {
              if (full)
                pass_fn(stage, cl0, nk, tgt, std::true_type{}, std::true_type{}, pi);
              else
                pass_fn(stage, cl0, nk, tgt, std::true_type{}, std::false_type{}, pi);
              return;
            }
          }
          if (full)
            pass_fn(stage, cl0, nk, tgt, std::false_type{}, std::true_type{}, pi);
          else
            pass_fn(stage, cl0, nk, tgt, std::false_type{}, std::false_type{}, pi);
        });
      }
      // Hand the stage back only once every lane's shared loads of it have returned: fold the accumulators (which
      // depend on all of them) into one word per lane, and let a warp vote gather the lanes before lane 0's arrive.
      uint32_t dep = 0;
#pragma unroll
      for (int j = 0; j < RTW; ++j)
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int n = 0; n < MT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) dep ^= __float_as_uint(acc[j][a][n][c]);
      dep = __any_sync(0xffffffffu, dep == 0x7FC00001u);
      if (lane == 0) mbar_arrive_dep(empty0 + 8 * st, dep);
    }
  }

  // ---------------- split-K reduction ----------------
  __syncthreads();  // ring is free: every stage has been consumed
  // Reduction.  Accumulator (j, n) of consumer warp (wr, wk) is item ((wr*RTW + j)*MT + n)*32 + lane of the CTA
  // tile (NI items of 4 results).  wki > 1: the K-slice warps add up through shared memory (`red`).  split > 1:
  // after a cluster barrier (every CTA is past its main loop, so its ring area is free) each CTA pushes its
  // partial items with distributed-shared-memory stores into the CTA that owns them (1/split of the tile each,
  // slot = pusher's cluster rank), and after a second barrier every owner adds its slots in rank order from its
  // own shared memory and stores.  (Pulling the partials with remote loads measured 1-2 us slower per call.)
  const int NI = p.rb * MT * 32;
  float4* red = reinterpret_cast<float4*>(smem);
  auto acc_item = [&](int j, int n) {
    float4 v = make_float4(acc[j][0][n][0], acc[j][0][n][1], acc[j][0][n][2], acc[j][0][n][3]);
#pragma unroll
    for (int a = 1; a < NA; ++a) {
      v.x += acc[j][a][n][0];
      v.y += acc[j][a][n][1];
      v.z += acc[j][a][n][2];
      v.w += acc[j][a][n][3];
    }
    return v;
  };
  if (p.wki > 1) {
    if (warp < nwc) {
#pragma unroll
      for (int j = 0; j < RTW; ++j)
#pragma unroll
        for (int n = 0; n < MT; ++n) red[(size_t)wk * NI + ((wr * RTW + j) * MT + n) * 32 + lane] = acc_item(j, n);
    }
    __syncthreads();
  }
  auto red_item = [&](int idx) {
    float4 v = red[idx];
    for (int q = 1; q < p.wki; ++q) {
      const float4 w = red[(size_t)q * NI + idx];
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    return v;
  };
  // The exchange epoch is read after this grid's dependency wait: the exchange's receive kernel, this grid's
  // dependent, advances the counter only after this grid has completed.
  uint32_t epoch = 0;
  constexpr bool TAGGED = OUTK == MBP_OUT_TAGGED_BF16X2 || OUTK == MBP_OUT_TAGGED_F32;
  if constexpr (TAGGED) epoch = (uint32_t)__ldcg(p.epoch) + 1u;
  const int owner = p.rsag ? (int)((blockIdx.x + blockIdx.z) % (unsigned)p.rP) : -1;
  auto emit = [&](int idx, float4 v) {
    const int ln = idx & 31, rest = idx >> 5, n = rest % MT, rr = rest / MT;
    if (rr >= rvalid) return;
    const int row = (r0 + rr) * 16 + (ln >> 2);
    const int tk = tok0 + n * 8 + 2 * (ln & 3);
    if constexpr (TAGGED) {
      emit_tagged<OUTK>(p, v, row, tk, epoch, owner);
    } else if constexpr (OUTK == kOutEpi) {
      if (tk < p.m) epi_fragment(p.epi, p.outs[0], p.ldo, v, epi_fragment_bias(p.epi, row), row, tk, p.m - tk);
    } else {
      for (int o = 0; o < p.nout; ++o) {
        OutT* out = reinterpret_cast<OutT*>(p.outs[o]);
        if (tk < p.m) {
          store_out(out + (size_t)tk * p.ldo + row, v.x);
          store_out(out + (size_t)tk * p.ldo + row + 8, v.z);
        }
        if (tk + 1 < p.m) {
          store_out(out + (size_t)(tk + 1) * p.ldo + row, v.y);
          store_out(out + (size_t)(tk + 1) * p.ldo + row + 8, v.w);
        }
      }
    }
  };
  const int nthr = blockDim.x;
  if (p.split == 1) {
    if (p.wki == 1) {
      if (warp < nwc) {  // every warp holds complete sums: store straight from registers
#pragma unroll
        for (int j = 0; j < RTW; ++j)
#pragma unroll
          for (int n = 0; n < MT; ++n) emit(((wr * RTW + j) * MT + n) * 32 + lane, acc_item(j, n));
      }
    } else {
      for (int idx = tid; idx < NI; idx += nthr) emit(idx, red_item(idx));
    }
  } else {
    const uint32_t rank = cluster_rank();
    const int per = (NI + p.split - 1) / p.split;
    float4* recv = red + (size_t)(p.wki > 1 ? p.wki : 0) * NI;  // [split][per]: this CTA's slots, after `red`
    const uint32_t recv_u32 = smem_u32(recv);
    auto push = [&](int idx, float4 v) {
      const int o = idx / per;
      st_dsmem_f4(mapa(recv_u32 + (uint32_t)((int)rank * per + idx - o * per) * 16u, (uint32_t)o), v);
    };
    cluster_sync();  // every CTA of the cluster is past its main loop: the slots may be written
    if (p.wki == 1) {
      if (warp < nwc) {
#pragma unroll
        for (int j = 0; j < RTW; ++j)
#pragma unroll
          for (int n = 0; n < MT; ++n) push(((wr * RTW + j) * MT + n) * 32 + lane, acc_item(j, n));
      }
    } else {
      for (int idx = tid; idx < NI; idx += nthr) push(idx, red_item(idx));
    }
    cluster_sync();  // every push has landed (release / acquire at cluster scope)
    const int i0 = (int)rank * per, i1 = min(NI, i0 + per);
    for (int idx = i0 + tid; idx < i1; idx += nthr) {
      float4 v = recv[idx - i0];
      for (int q = 1; q < p.split; ++q) {
        const float4 w = recv[(size_t)q * per + idx - i0];
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
      emit(idx, v);
    }
  }
  if constexpr (TAGGED) {
    if (p.rout) {  // fused receive: this CTA's tiles from every rank, then the epoch ticket
      const int crank = p.split > 1 ? (int)cluster_rank() : 0;
      if (OUTK == MBP_OUT_TAGGED_F32 && p.rsag)
        tp_receive_rsag<TOK>(p, epoch, r0, rvalid, tok0, crank * nthr + tid, nthr * p.split, owner);
      else
        tp_receive<OUTK, TOK>(p, epoch, r0, rvalid, tok0, crank * nthr + tid, nthr * p.split);
      tp_advance_epoch(p.ctr, tid);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------------------
using KernelFn = void (*)(GemvParams);

template <int FMT, int MT, int RTW, int OUTK>
KernelFn kernel_ptr() {
  return reinterpret_cast<KernelFn>(&k_gemv<FMT, MT, RTW, OUTK>);
}

template <int MT, int RTW>
KernelFn pick_c12(int outk) {
  switch (outk) {
    case MBP_OUT_F32: return kernel_ptr<FMT_C12, MT, RTW, MBP_OUT_F32>();
    case MBP_OUT_TAGGED_BF16X2: return kernel_ptr<FMT_C12, MT, RTW, MBP_OUT_TAGGED_BF16X2>();
    case MBP_OUT_TAGGED_F32: return kernel_ptr<FMT_C12, MT, RTW, MBP_OUT_TAGGED_F32>();
    case kOutEpi: return kernel_ptr<FMT_C12, MT, RTW, kOutEpi>();
    default: return kernel_ptr<FMT_C12, MT, RTW, MBP_OUT_BF16>();
  }
}

// outk: MBP_OUT_* or kOutEpi (the router format always writes plain FP32)
KernelFn pick(int fmt, int mt, int rtw, int outk) {
  if (fmt == FMT_C12) {
    if (mt == 1 && rtw == 1) return pick_c12<1, 1>(outk);
    if (mt == 1) return pick_c12<1, 2>(outk);
    if (mt == 2 && rtw == 1) return pick_c12<2, 1>(outk);
    if (mt == 2) return pick_c12<2, 2>(outk);
    return pick_c12<4, 2>(outk);
  }
  if (mt == 1) return kernel_ptr<FMT_HILO, 1, 1, MBP_OUT_F32>();
  if (mt == 2) return kernel_ptr<FMT_HILO, 2, 1, MBP_OUT_F32>();
  return kernel_ptr<FMT_HILO, 4, 2, MBP_OUT_F32>();
}

int mt_of(int m) { return m <= 8 ? 1 : m <= 16 ? 2 : 4; }
int rtw_of(int mt) { return mt == 4 ? 2 : 1; }
// register-tile widths that have an instance for this format and token tile
bool rtw_ok(int fmt, int mt, int rtw) { return rtw == 2 ? (fmt == FMT_C12 || mt == 4) : mt != 4; }
int ub_of(int fmt) { return fmt == FMT_C12 ? MBP_C12_UNIT_BYTES : 2 * MBP_RAW_UNIT_BYTES; }

// Per-device one-time function attributes (max dynamic shared memory, non-portable cluster sizes).
std::mutex g_attr_mu;
std::map<std::pair<int, KernelFn>, bool> g_attr_done;

int ensure_attrs(KernelFn fn) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return MBP_ERR_LAUNCH;
  std::lock_guard<std::mutex> lk(g_attr_mu);
  auto key = std::make_pair(dev, fn);
  if (g_attr_done.count(key)) return MBP_OK;
  if (cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) !=
      cudaSuccess)
    return MBP_ERR_SMEM;
  if (cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeNonPortableClusterSizeAllowed, 1) !=
      cudaSuccess)
    return MBP_ERR_CLUSTER;
  g_attr_done[key] = true;
  return MBP_OK;
}

int sm_count() {
  int dev = 0, n = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

// Co-resident CTAs (clusters of `split` CTAs) for this kernel/config, cached.
std::mutex g_occ_mu;
std::map<std::tuple<int, KernelFn, int, int, int>, int> g_occ;

int max_ctas(KernelFn fn, int split, int threads, int smem) {
  int dev = 0;
  cudaGetDevice(&dev);
  auto key = std::make_tuple(dev, fn, split, threads, smem);
  {
    std::lock_guard<std::mutex> lk(g_occ_mu);
    auto it = g_occ.find(key);
    if (it != g_occ.end()) return it->second;
  }
  int ctas = 0;
  if (ensure_attrs(fn) == MBP_OK) {
    if (split == 1) {
      int per_sm = 0;
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, reinterpret_cast<const void*>(fn), threads, smem) ==
          cudaSuccess)
        ctas = per_sm * sm_count();
    } else {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1, split, 1);
      cfg.blockDim = dim3(threads);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = 1;
      attr.val.clusterDim.y = split;
      attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, reinterpret_cast<const void*>(fn), &cfg) == cudaSuccess)
        ctas = clusters * split;
    }
  }
  cudaGetLastError();
  std::lock_guard<std::mutex> lk(g_occ_mu);
  g_occ[key] = ctas;
  return ctas;
}

// Geometry search over a bandwidth model fit to measurements on B200:
//   * the device streams at most ~6.0 TB/s and one SM at most ~45 GB/s, so a launch takes at least
//     max(all bytes / 6.0 TB/s, bytes of the busiest SM / 45 GB/s);
//   * the TMA engine only reaches that with stages of ~48-96 KB made of copies of >= 6 KB (kci units per row
//     tile), 2-4 stages deep;
//   * each level of cluster split-K costs a fixed reduction / synchronisation overhead;
//   * ~8 consumer warps per SM (fewer, fatter CTAs when the token tile is large and 2 CTAs fit an SM).
// Only single-wave launches are considered.
// zb: token blocks (grid z); outk: MBP_OUT_BF16 or MBP_OUT_F32 (an epilogue runs in the geometry of its output type).
int plan_search(int fmt, int Rout, int C, int mt, int zb, int outk, bool esc, mbp_gemv_geom* g) {
  constexpr double kHbmBw = 6.0e12, kSmBw = 45.0e9, kSplitCost = 1.2e-6;
  const int ub = ub_of(fmt);
  const int rtw = rtw_of(mt), tok = 8 * mt, kc = kc_for(fmt, mt, rtw);
  const KernelFn fn = pick(fmt, mt, rtw, outk);
  const int sms = sm_count();
  const double total = (double)Rout * C * ub * zb;
  double best = 1e30;
  mbp_gemv_geom bg = {};
  const int rb_max = ((Rout + rtw - 1) / rtw) * rtw;
  // cluster sizes that pack evenly into the GPCs (sizes like 5 or 7 strand SMs and measured far slower)
  for (const int split : {1, 2, 3, 4, 6, 8}) {
    if (split > C) break;
    const int cpc = (C + split - 1) / split;
    for (int rb = rtw; rb <= kMaxConsumerWarps * rtw && rb <= rb_max; rb += rtw) {
      const int rows_w = rb / rtw;
      const int nblk = (Rout + rb - 1) / rb;
      const long long G = (long long)nblk * split * zb;
      // consumer warps: ~8 per CTA, never more than the slice count
      int wki = (8 + rows_w / 2) / rows_w;
      if (wki < 1) wki = 1;
      while (rows_w * wki > kMaxConsumerWarps) --wki;
      if (wki > cpc) wki = cpc;
      const int per_slice = (cpc + wki - 1) / wki;
      // largest copy whose stage stays <= 96 KB and whose 2-stage ring fits; 3-4 stages when they fit
      int kci = kc;
      while (kci + kc <= 16 && kci < per_slice && rb * wki * (kci + kc) * ub <= 96 * 1024) kci += kc;
      while (kci > kc && smem_request(make_layout(fmt, mt, rb, rtw, wki, kci, 2, esc)) > kMaxSmem) kci -= kc;
      const int slot_w = rb * wki * kci * ub;
      int st = 2;
      while (st < 4 && (st + 1) * slot_w <= 192 * 1024 &&
             smem_request(make_layout(fmt, mt, rb, rtw, wki, kci, st + 1, esc)) <= kMaxSmem)
        ++st;
      const Layout L = make_layout(fmt, mt, rb, rtw, wki, kci, st, esc);
      if (smem_request(L) > kMaxSmem) continue;
      const int threads = 32 * (rows_w * wki + 1);
      const int cap = max_ctas(fn, split, threads, smem_request(L));
      if (cap <= 0) continue;
      const long long waves = (G + cap - 1) / cap;
      const double per_cta = (double)(rb < Rout ? rb : Rout) * cpc * ub + (double)cpc * tok * 128;
      const long long per_sm = (G + sms - 1) / sms;
      double t = total / kHbmBw;
      const double t_sm = per_cta * per_sm / kSmBw;
      if (t_sm > t) t = t_sm;
      if (waves > 1) t *= 1.0 + 0.15 * (waves - 1);  // wave tails
      if (split > 1) t += kSplitCost * (1.0 + 0.1 * split);
      if (kci * ub < 6144 && kci < per_slice) t *= 1.3;  // small copies starve the TMA engine
      if (st * slot_w < 96 * 1024) t *= 1.0 + (96.0 * 1024 - st * slot_w) / (192.0 * 1024);
      if (t < best) {
        best = t;
        bg.rb = rb;
        bg.rtw = rtw;
        bg.split = split;
        bg.wki = wki;
        bg.kci = kci;
        bg.stages = st;
        bg.nblk = nblk;
      }
    }
  }
  if (best >= 1e30) return MBP_ERR_SPLIT;
  *g = bg;
  return MBP_OK;
}

// Escape density classes of a 12-bit matrix: none, sparse (< 1 escape per 1000 weights: N(0, s) weights, whose
// 16-binade exponent window misses only the far tail near zero), dense (heavy-tailed matrices such as the
// reference's 1%-scaled stress variant).
enum { ESC_NONE = 0, ESC_SPARSE = 1, ESC_DENSE = 2 };

int esc_class(int64_t n_esc, int n, int k) {
  return n_esc <= 0 ? ESC_NONE : n_esc * 1000 >= (int64_t)n * k ? ESC_DENSE : ESC_SPARSE;
}

// Geometries measured fastest on B200 for the reference's decode shapes (fused QKV+gate 14336 x 6144 and output
// projection 6144 x 6144; one token block; CUDA-graph replay over weight copies larger than L2, programmatic
// launch on), by an exhaustive sweep of the single-wave geometries that fit shared memory.  Shapes not listed
// use the model search below.
struct Tuned {
  int Rout, C, mt, dense;
  mbp_gemv_geom g;
  int zb = 1;  // token blocks of 8*mt (grid z): m > 32 launches one wave of CTAs per block
};
constexpr Tuned kTuned[] = {
    {896, 96, 1, 0, {7, 1, 1, 1, 8, 2, 128}},  {896, 96, 1, 1, {7, 1, 1, 1, 8, 2, 128}},
    {896, 96, 2, 0, {7, 1, 1, 1, 4, 3, 128}},  {896, 96, 2, 1, {7, 1, 1, 1, 4, 3, 128}},
    {896, 96, 4, 0, {14, 2, 2, 1, 3, 2, 64}},  {896, 96, 4, 1, {22, 2, 3, 1, 2, 2, 41}},
    {384, 96, 1, 0, {3, 1, 1, 2, 8, 2, 128}},  {384, 96, 1, 1, {3, 1, 1, 3, 4, 2, 128}},
    {384, 96, 2, 0, {3, 1, 1, 3, 4, 2, 128}},  {384, 96, 2, 1, {3, 1, 1, 3, 4, 2, 128}},
    {384, 96, 4, 0, {12, 2, 4, 1, 4, 2, 32}},  {384, 96, 4, 1, {6, 2, 2, 3, 2, 2, 64}},
    // tensor-parallel shards of the same projections (column-parallel qkv_gate: n/P rows; row-parallel o: k/P
    // columns, FP32 partials), P = 2, 4, 8; only where the measured best beat the planner by more than 3%
    {448, 96, 1, 0, {7, 1, 2, 1, 8, 2, 64}},   {448, 96, 2, 0, {14, 2, 4, 1, 4, 2, 32}},
    {448, 96, 4, 0, {14, 2, 4, 1, 3, 2, 32}},  {448, 96, 1, 1, {11, 1, 3, 1, 4, 2, 41}},
    {448, 96, 2, 1, {11, 1, 3, 1, 4, 2, 41}},  {448, 96, 4, 1, {22, 2, 6, 1, 2, 2, 21}},
    {384, 48, 1, 0, {3, 1, 1, 2, 8, 2, 148}},  {384, 48, 4, 0, {6, 2, 2, 2, 3, 2, 64}},
    {384, 48, 4, 1, {6, 2, 2, 3, 2, 2, 64}},   {224, 96, 1, 0, {2, 1, 1, 3, 8, 2, 112}},
    {224, 96, 2, 0, {11, 1, 6, 1, 4, 2, 21}},  {224, 96, 4, 0, {8, 2, 4, 2, 3, 2, 28}},
    {224, 96, 1, 1, {11, 1, 6, 1, 4, 2, 21}},  {224, 96, 2, 1, {2, 1, 1, 4, 4, 2, 112}},
    {224, 96, 4, 1, {2, 2, 1, 7, 2, 2, 112}},  {384, 24, 4, 0, {4, 2, 1, 4, 2, 2, 96}},
    {384, 24, 4, 1, {4, 2, 1, 4, 2, 2, 96}},   {112, 96, 1, 0, {2, 1, 2, 3, 8, 2, 56}},
    {112, 96, 2, 0, {4, 1, 4, 2, 4, 2, 28}},   {112, 96, 4, 0, {4, 2, 4, 3, 3, 2, 28}},
    {112, 96, 1, 1, {4, 1, 4, 2, 4, 2, 28}},   {112, 96, 2, 1, {4, 1, 4, 2, 4, 2, 28}},
    {112, 96, 4, 1, {4, 2, 4, 4, 2, 2, 28}},   {384, 12, 4, 0, {4, 2, 1, 3, 2, 3, 96}},
    {384, 12, 4, 1, {4, 2, 1, 4, 2, 2, 96}},
    // the reference's own layer shapes (qkv_gate 2304x8192, o 8192x1024, pooler 4096x8192, unpooler 8192x4096 and
    // its first 1024 rows), where the measured best beat the planner by more than 3%
    {144, 128, 1, 0, {2, 1, 2, 3, 8, 2, 72}},  {144, 128, 2, 0, {2, 1, 2, 2, 8, 2, 72}},
    {144, 128, 4, 0, {2, 2, 2, 7, 2, 2, 72}},  {512, 16, 1, 0, {4, 1, 1, 1, 8, 2, 128}},
    {512, 16, 4, 0, {4, 2, 1, 4, 2, 2, 128}},  {256, 128, 1, 0, {2, 1, 1, 3, 8, 2, 148}},
    {256, 128, 4, 0, {8, 2, 4, 2, 3, 2, 32}},  {512, 64, 4, 0, {4, 2, 1, 3, 3, 2, 128}},
    {64, 64, 1, 0, {4, 1, 8, 1, 4, 2, 16}},    {64, 64, 2, 0, {4, 1, 8, 1, 4, 2, 16}},
    {64, 64, 4, 0, {4, 2, 8, 2, 2, 2, 16}},
};
// hi/lo router (256 x 8192), M tiles 8 / 16 / 32: 4.95 / 5.23 / 6.56 us against the planner's 9.6 / 10.1 / 7.5 us;
// M = 64 / 128 / 256 (2 / 4 / 8 token blocks of 32): 8.05 / 9.62 / 13.77 us against 14.5 / 11.3 / 16.1 us
constexpr Tuned kTunedHilo[] = {
    {16, 128, 1, 0, {1, 1, 8, 2, 4, 2, 16}},    {16, 128, 2, 0, {1, 1, 8, 3, 3, 2, 16}},
    {16, 128, 4, 0, {2, 2, 16, 4, 1, 2, 9}},    {16, 128, 4, 0, {2, 2, 6, 3, 3, 2, 8}, 2},
    {16, 128, 4, 0, {2, 2, 4, 4, 2, 2, 8}, 4},  {16, 128, 4, 0, {4, 2, 4, 2, 2, 2, 4}, 8},
    // the BASELINE router (256 x 6144), M = 1-8 / 9-16 / 17-32 and 64 / 128 / 256 tokens: 4.51 / 4.89 / 5.79 and
    // 6.91 / 8.38 / 10.82 us against the planner's 9.06 / 9.50 / 6.94 and 13.6 / 9.73 / 13.5 us (exhaustive sweep;
    // only geometries within half the 1e-5 tolerance against FP64: a warp that alone accumulates all 6144 columns
    // of a row in FP32 can exceed it)
    {16, 96, 1, 0, {1, 1, 8, 2, 4, 2, 16}},     {16, 96, 2, 0, {1, 1, 8, 2, 4, 2, 16}},
    {16, 96, 4, 0, {2, 2, 16, 3, 1, 2, 8}},     {16, 96, 4, 0, {2, 2, 6, 4, 2, 2, 8}, 2},
    {16, 96, 4, 0, {2, 2, 4, 4, 2, 2, 8}, 4},   {16, 96, 4, 0, {2, 2, 8, 2, 1, 2, 8}, 8},
};

std::mutex g_plan_mu;
std::map<std::tuple<int, int, int, int, int, int, int, int>, mbp_gemv_geom> g_plans;

// Planned geometries are cached per (device, format, shape, token tile count, output type, escape class).
int plan_impl(int fmt, int Rout, int C, int m, bool f32, int esc, mbp_gemv_geom* g) {
  int dev = 0;
  cudaGetDevice(&dev);
  const int mt = mt_of(m);
  const int zb = (m + 8 * mt - 1) / (8 * mt);
  const int outk = f32 ? MBP_OUT_F32 : MBP_OUT_BF16;
  const auto key = std::make_tuple(dev, fmt, Rout, C, mt, zb, outk, esc);
  {
    std::lock_guard<std::mutex> lk(g_plan_mu);
    auto it = g_plans.find(key);
    if (it != g_plans.end()) {
      *g = it->second;
      return MBP_OK;
    }
  }
  {
    const bool c12 = fmt == FMT_C12;
    const Tuned* tab = c12 ? kTuned : kTunedHilo;
    const size_t nt = c12 ? sizeof(kTuned) / sizeof(Tuned) : sizeof(kTunedHilo) / sizeof(Tuned);
    for (size_t i = 0; i < nt; ++i) {
      const Tuned& t = tab[i];
      if (t.Rout == Rout && t.C == C && t.mt == mt && t.zb == zb && t.dense == (esc == ESC_DENSE)) {
        *g = t.g;
        std::lock_guard<std::mutex> lk(g_plan_mu);
        g_plans[key] = *g;
        return MBP_OK;
      }
    }
  }
  const int rc = plan_search(fmt, Rout, C, mt, zb, outk, esc != ESC_NONE, g);
  if (rc == MBP_OK) {
    std::lock_guard<std::mutex> lk(g_plan_mu);
    g_plans[key] = *g;
  }
  return rc;
}

struct RecvArgs {  // fused receive of a tensor-parallel exchange (mbp_gemv_c12_tp)
  const uint8_t* buf;
  void* out;
  int* ctr;
  int n, P;
  int rsag, rank;  // row-parallel reduce-scatter + gather: this rank, and the gather region's offsets
  long long goff, gdelta;
};

int launch(int fmt, const uint8_t* units, const uint8_t* bases, const int32_t* esc_off, const uint32_t* esc,
           int esc_cls, int C, int K, int n_out, const uint16_t* x, int ldx, int m, void* const* outs, int nout,
           int ldo, bool f32, const mbp_gemv_geom* geom, cudaStream_t stream, const int* epoch = nullptr,
           long long parity_stride = 0, int tagged = 0, const RecvArgs* recv = nullptr,
           const EpiArgs* epi = nullptr) {
  if (m < 1) return MBP_ERR_M;
  if (!outs || nout < 1 || nout > kMaxOuts) return MBP_ERR_ARG;
  if (parity_stride < 0 || (parity_stride & 15)) return MBP_ERR_ALIGN;
  if (tagged && !epoch) return MBP_ERR_ARG;
  for (int o = 0; o < nout; ++o) {
    if (!outs[o]) return MBP_ERR_ARG;
    if (tagged && ((uintptr_t)outs[o] & 7u)) return MBP_ERR_ALIGN;
  }
  if (n_out <= 0 || n_out % 16) return MBP_ERR_SHAPE;
  if (ldo < (tagged == MBP_OUT_TAGGED_BF16X2 ? n_out / 2 : n_out)) return MBP_ERR_SHAPE;
  if (((uintptr_t)x & 15u) || ((uintptr_t)units & 15u) || ldx < K || ldx % 8) return MBP_ERR_ALIGN;
  const int mt = mt_of(m), tok = 8 * mt;
  const int Rout = n_out / 16;
  const bool with_esc = fmt == FMT_C12 && esc_cls != ESC_NONE;
  mbp_gemv_geom g;
  if (geom) {
    g = *geom;
  } else {
    const int rc = plan_impl(fmt, Rout, C, m, f32, esc_cls, &g);
    if (rc) return rc;
  }
  const int rtw = g.rtw, kc = kc_for(fmt, mt, rtw);
  if (!rtw_ok(fmt, mt, rtw) || g.rb < rtw || g.rb % rtw || g.rb / rtw > kMaxConsumerWarps) return MBP_ERR_SPLIT;
  if (g.split < 1 || g.split > 16 || g.split > C || g.wki < 1 || g.kci < kc || g.kci % kc || g.stages < 1)
    return MBP_ERR_SPLIT;
  const int rows_w = g.rb / rtw;
  if (rows_w * g.wki > kMaxConsumerWarps) return MBP_ERR_SPLIT;
  const int nblk = g.nblk > 0 ? g.nblk : (Rout + g.rb - 1) / g.rb;
  if (nblk > Rout || (Rout + nblk - 1) / nblk > g.rb) return MBP_ERR_SPLIT;  // a block holds at most rb tiles
  const Layout L = make_layout(fmt, mt, g.rb, rtw, g.wki, g.kci, g.stages, with_esc);
  if (smem_request(L) > kMaxSmem) return MBP_ERR_SMEM;
  const KernelFn fn = pick(fmt, mt, rtw, epi ? (int)kOutEpi : tagged ? tagged : f32 ? MBP_OUT_F32 : MBP_OUT_BF16);
  int rc = ensure_attrs(fn);
  if (rc) return rc;
  // A fused receive waits for other ranks' CTAs of the same index: the whole grid must be resident at once.
  if (recv && (long long)nblk * g.split * ((m + tok - 1) / tok) >
                  max_ctas(fn, g.split, 32 * (rows_w * g.wki + 1), smem_request(L)))
    return MBP_ERR_SPLIT;
  GemvParams p;
  if (!encode_bf16_2d_cached(&p.xmap, x, (uint64_t)m, (uint64_t)K, (uint64_t)ldx, (uint32_t)tok, 64u,
                             CU_TENSOR_MAP_SWIZZLE_128B))
    return MBP_ERR_TMAP;
  p.units = units;
  p.bases = bases;
  p.esc_off = esc_off;
  p.esc = esc;
  for (int o = 0; o < kMaxOuts; ++o) p.outs[o] = o < nout ? outs[o] : nullptr;
  p.epoch = epoch;
  p.parity_stride = epoch ? parity_stride : 0;
  p.rbuf = recv ? recv->buf : nullptr;
  p.rout = recv ? recv->out : nullptr;
  p.ctr = recv ? recv->ctr : nullptr;
  p.rn = recv ? recv->n : 0;
  p.rP = recv ? recv->P : 0;
  p.rsag = recv ? recv->rsag : 0;
  p.rrank = recv ? recv->rank : 0;
  p.goff = recv ? recv->goff : 0;
  p.gdelta = recv ? recv->gdelta : 0;
  p.epi = epi ? *epi : EpiArgs{};
  p.nout = nout;
  p.C = C;
  p.Rout = Rout;
  p.m = m;
  p.ldo = ldo;
  p.rb = g.rb;
  p.split = g.split;
  p.wki = g.wki;
  p.kci = g.kci;
  p.stages = g.stages;
  p.nblk = nblk;
  p.has_esc = with_esc ? 1 : 0;
  p.wait_ns = wait_limit_ns();
  static const int pre_env = getenv("MBP_GEMV_PREFETCH") ? atoi(getenv("MBP_GEMV_PREFETCH")) : 0;
  p.pre_stages = pre_env > 0 ? pre_env : g.stages;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(nblk, g.split, (m + tok - 1) / tok);
  cfg.blockDim = dim3(32 * (rows_w * g.wki + 1));
  cfg.dynamicSmemBytes = smem_request(L);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int na = 0;
  static const bool pdl = getenv("MBP_NO_PDL") == nullptr;  // MBP_NO_PDL set: plain stream serialisation
  if (pdl) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  if (g.split > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = 1;
    attr[na].val.clusterDim.y = g.split;
    attr[na].val.clusterDim.z = 1;
    ++na;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  return cudaLaunchKernelEx(&cfg, fn, p) == cudaSuccess ? MBP_OK : MBP_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int mbp_gemv_plan(int n_out, int k, int m, mbp_gemv_geom* geom) {
  if (!geom) return MBP_ERR_ARG;
  if (n_out <= 0 || n_out % 16 || k <= 0 || k % 64) return MBP_ERR_SHAPE;
  if (m < 1) return MBP_ERR_M;
  return plan_impl(FMT_C12, n_out / 16, k / 64, m, false, ESC_DENSE, geom);
}

int mbp_gemv_plan_ex(int n_out, int k, int m, int flags, mbp_gemv_geom* geom) {
  if (!geom || (flags & ~(MBP_PLAN_ESCAPES | MBP_PLAN_F32_OUT | MBP_PLAN_DENSE_ESCAPES))) return MBP_ERR_ARG;
  if (n_out <= 0 || n_out % 16 || k <= 0 || k % 64) return MBP_ERR_SHAPE;
  if (m < 1) return MBP_ERR_M;
  const int cls = (flags & MBP_PLAN_DENSE_ESCAPES) ? ESC_DENSE : (flags & MBP_PLAN_ESCAPES) ? ESC_SPARSE : ESC_NONE;
  return plan_impl(FMT_C12, n_out / 16, k / 64, m, (flags & MBP_PLAN_F32_OUT) != 0, cls, geom);
}

int mbp_gemv_c12(const mbp_c12* w, const uint16_t* x, int m, int n_out, uint16_t* out, int ldo,
                 const mbp_gemv_geom* geom, cudaStream_t stream) {
  if (!w || !w->units || !w->bases || !w->esc_off || !x || !out) return MBP_ERR_ARG;
  if (w->n_esc > 0 && !w->esc) return MBP_ERR_ARG;
  if (w->n % 16 || w->k % 64 || w->k / 64 > 32766 || n_out > w->n) return MBP_ERR_SHAPE;
  void* outs[1] = {out};
  return launch(FMT_C12, w->units, w->bases, w->esc_off, w->esc, esc_class(w->n_esc, w->n, w->k), w->k / 64, w->k,
                n_out, x, w->k, m, outs, 1, ldo, false, geom, stream);
}

int mbp_gemv_c12_f32(const mbp_c12* w, const uint16_t* x, int m, int n_out, float* out, int ldo,
                     const mbp_gemv_geom* geom, cudaStream_t stream) {
  if (!w || !w->units || !w->bases || !w->esc_off || !x || !out) return MBP_ERR_ARG;
  if (w->n_esc > 0 && !w->esc) return MBP_ERR_ARG;
  if (w->n % 16 || w->k % 64 || w->k / 64 > 32766 || n_out > w->n) return MBP_ERR_SHAPE;
  void* outs[1] = {out};
  return launch(FMT_C12, w->units, w->bases, w->esc_off, w->esc, esc_class(w->n_esc, w->n, w->k), w->k / 64, w->k,
                n_out, x, w->k, m, outs, 1, ldo, true, geom, stream);
}

int mbp_gemv_c12_epi(const mbp_c12* w, const uint16_t* x, int m, int n_out, const mbp_epilogue* epi, void* out,
                     int ldo, const mbp_gemv_geom* geom, cudaStream_t stream) {
  if (!w || !w->units || !w->bases || !w->esc_off || !x || !out) return MBP_ERR_ARG;
  if (w->n_esc > 0 && !w->esc) return MBP_ERR_ARG;
  if (w->n % 16 || w->k % 64 || w->k / 64 > 32766 || n_out > w->n) return MBP_ERR_SHAPE;
  EpiArgs e;
  const int rc = check_epilogue(epi, n_out, out, ldo, &e);
  if (rc) return rc;
  void* outs[1] = {out};
  return launch(FMT_C12, w->units, w->bases, w->esc_off, w->esc, esc_class(w->n_esc, w->n, w->k), w->k / 64, w->k,
                n_out, x, w->k, m, outs, 1, ldo, e.out_f32 != 0, geom, stream, nullptr, 0, 0, nullptr, &e);
}

int mbp_gemv_c12_multi(const mbp_c12* w, const uint16_t* x, int ldx, int m, int n_out, void* const* outs, int nout,
                       int ldo, int out_kind, const int* epoch, long long parity_stride, const mbp_gemv_geom* geom,
                       cudaStream_t stream) {
  if (!w || !w->units || !w->bases || !w->esc_off || !x || !outs) return MBP_ERR_ARG;
  if (w->n_esc > 0 && !w->esc) return MBP_ERR_ARG;
  if (out_kind < MBP_OUT_BF16 || out_kind > MBP_OUT_TAGGED_F32) return MBP_ERR_ARG;
  if (w->n % 16 || w->k % 64 || w->k / 64 > 32766 || n_out > w->n) return MBP_ERR_SHAPE;
  const bool f32 = out_kind == MBP_OUT_F32 || out_kind == MBP_OUT_TAGGED_F32;
  const int tagged = out_kind >= MBP_OUT_TAGGED_BF16X2 ? out_kind : 0;
  return launch(FMT_C12, w->units, w->bases, w->esc_off, w->esc, esc_class(w->n_esc, w->n, w->k), w->k / 64, w->k,
                n_out, x, ldx, m, outs, nout, ldo, f32, geom, stream, epoch, parity_stride, tagged);
}

int mbp_gemv_c12_tp(const mbp_c12* w, const uint16_t* x, int ldx, int m, const mbp_tp_exchange* ex, uint16_t* out,
                    const mbp_gemv_geom* geom, cudaStream_t stream) {
  if (!w || !w->units || !w->bases || !w->esc_off || !x || !ex || !out || !ex->counter) return MBP_ERR_ARG;
  if (w->n_esc > 0 && !w->esc) return MBP_ERR_ARG;
  if (ex->P < 1 || ex->P > kMaxOuts || ex->rank < 0 || ex->rank >= ex->P) return MBP_ERR_SHAPE;
  if (ex->mode != MBP_TP_GATHER_BF16 && ex->mode != MBP_TP_SUM_F32 && ex->mode != MBP_TP_RSAG) return MBP_ERR_ARG;
  if (w->n % 16 || w->k % 64 || w->k / 64 > 32766) return MBP_ERR_SHAPE;
  const bool gather = ex->mode == MBP_TP_GATHER_BF16;
  if (ex->n != (gather ? w->n * ex->P : w->n)) return MBP_ERR_SHAPE;
  if (m < 1 || m > 32) return MBP_ERR_M;
  if (((uintptr_t)out & 15u) || (ex->parity_stride & 15) || ex->parity_stride < 0) return MBP_ERR_ALIGN;
  void* outs[kMaxOuts];
  const long long off = gather ? (long long)ex->rank * (w->n / 2) * 8 : (long long)ex->rank * m * ex->n * 8;
  for (int r = 0; r < ex->P; ++r) {
    if (!ex->bufs[r]) return MBP_ERR_ARG;
    outs[r] = static_cast<char*>(ex->bufs[r]) + off;
  }
  RecvArgs rv{static_cast<const uint8_t*>(ex->bufs[ex->rank]), out, ex->counter, ex->n, ex->P, 0, ex->rank, 0, 0};
  if (ex->mode == MBP_TP_RSAG) {
    // gather region after the P slots sized for 32 tokens: [32][n/2] words
    rv.rsag = 1;
    rv.goff = (long long)ex->P * 32 * ex->n * 8;
    rv.gdelta = rv.goff - off;
    if (ex->parity_stride < rv.goff + 32LL * (ex->n / 2) * 8) return MBP_ERR_SHAPE;
  }
  return launch(FMT_C12, w->units, w->bases, w->esc_off, w->esc, esc_class(w->n_esc, w->n, w->k), w->k / 64, w->k,
                w->n, x, ldx, m, outs, ex->P, gather ? ex->n / 2 : ex->n, !gather, geom, stream, ex->counter,
                ex->parity_stride, gather ? MBP_OUT_TAGGED_BF16X2 : MBP_OUT_TAGGED_F32, &rv);
}

int mbp_router_hilo(const mbp_hilo* w, const uint16_t* x, int m, float* out, int ldo, const mbp_gemv_geom* geom,
                    cudaStream_t stream) {
  if (!w || !w->units || !x || !out) return MBP_ERR_ARG;
  if (w->n % 16 || w->k % 64 || w->k / 64 > 32766) return MBP_ERR_SHAPE;
  if (m < 1) return MBP_ERR_M;
  if (!geom && m >= MBP_ROUTER_TC_MIN_M && w->k <= MBP_ROUTER_TC_MAX_K)
    return mbp_router_hilo_tc(w, x, m, out, ldo, 0, 0, stream);
  mbp_gemv_geom g;
  if (!geom) {
    const int rc = plan_impl(FMT_HILO, w->n / 16, w->k / 64, m, true, ESC_NONE, &g);
    if (rc) return rc;
    geom = &g;
  }
  void* outs[1] = {out};
  return launch(FMT_HILO, w->units, nullptr, nullptr, nullptr, ESC_NONE, w->k / 64, w->k, w->n, x, w->k, m, outs, 1,
                ldo, true, geom, stream);
}

}  // extern "C"

int mbp_status_gemv(int* v, int clear) { return read_status_here(v, clear); }
