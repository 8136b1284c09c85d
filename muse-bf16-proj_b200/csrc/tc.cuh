// tcgen05 / TMEM helpers shared by the projection GEMM and the expert GEMM: descriptors, MMA issue, the decoded-A
// store, the accumulator load, and the tensor map of packed weight units.
#pragma once
#include "common.cuh"
#include "tmap.h"

namespace mbp {

MBP_DEV void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

MBP_DEV void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
MBP_DEV void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// K-major, 128-byte-swizzled operand: rows of 128 bytes, 8-row atoms of 1024 bytes (SBO), LBO unused (1).
MBP_DEV uint64_t smem_desc_sw128(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// kind::f16 instruction descriptor: BF16 x BF16 -> FP32, both K-major, M = 128, N = n.
MBP_DEV uint32_t idesc_bf16(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// A from TMEM (M=128 lanes = rows, 8 columns per K=16: a column holds two consecutive K elements, low half first).
MBP_DEV void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// 4 x 4 transpose across the 4 lanes of a quad (t = lane & 3): afterwards lane t holds, at index a, what lane a
// held at index t.  Two butterfly stages (partners t ^ 2, then t ^ 1), each exchanging the two elements whose
// index differs from t in that stage's bit.
MBP_DEV void quad_transpose(uint32_t& m0, uint32_t& m1, uint32_t& m2, uint32_t& m3, int t) {
  const bool b1 = (t & 2) != 0, b0 = (t & 1) != 0;
  uint32_t s0 = b1 ? m0 : m2, s1 = b1 ? m1 : m3;
  s0 = __shfl_xor_sync(0xffffffffu, s0, 2);
  s1 = __shfl_xor_sync(0xffffffffu, s1, 2);
  if (b1) {
    m0 = s0;
    m1 = s1;
  } else {
    m2 = s0;
    m3 = s1;
  }
  s0 = b0 ? m0 : m1;
  s1 = b0 ? m2 : m3;
  s0 = __shfl_xor_sync(0xffffffffu, s0, 1);
  s1 = __shfl_xor_sync(0xffffffffu, s1, 1);
  if (b0) {
    m0 = s0;
    m2 = s1;
  } else {
    m1 = s0;
    m3 = s1;
  }
}

// A decoded unit into TMEM: 16 lanes (rows) x 32 columns (64 K, two bf16 per column, natural K order).
// The decoder leaves lane 4g + t with the K pairs 8t .. 8t+7 of rows g and g + 8 (register 2s + rh = pair 8t + s
// of row g + 8rh: the unit's lane layout).  The .16x128b.x8 store puts register i of lane 4g + t at row
// g + 8 (i % 2), column 4 (i / 2) + t, i.e. lane t must hold the pairs 4c + t, c = 0..7.  Pair 4c + t lives in lane
// c / 2 at s = 4 (c % 2) + t: for each half h = c % 2 and row rh that is a 4 x 4 transpose across the quad.
// Weights packed in mma order (TURN = false) hold pair 4s + t at lane t's s already: the registers go as they are.
template <bool TURN>
MBP_DEV void tc_st_a(uint32_t taddr, const uint32_t (&A)[16], int t) {
  uint32_t a[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) a[i] = A[i];
#pragma unroll
  for (int h = 0; TURN && h < 2; ++h)
#pragma unroll
    for (int rh = 0; rh < 2; ++rh) {
      uint32_t m0 = A[2 * (4 * h + 0) + rh], m1 = A[2 * (4 * h + 1) + rh], m2 = A[2 * (4 * h + 2) + rh],
               m3 = A[2 * (4 * h + 3) + rh];
      quad_transpose(m0, m1, m2, m3, t);  // now m_j = pair 4(2j + h) + t of row rh (column c = 2j + h)
      a[2 * (2 * 0 + h) + rh] = m0;
      a[2 * (2 * 1 + h) + rh] = m1;
      a[2 * (2 * 2 + h) + rh] = m2;
      a[2 * (2 * 3 + h) + rh] = m3;
    }
  __syncwarp();  // .sync.aligned: the lanes may come from branches of their own
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(a[4]), "r"(a[5]), "r"(a[6]), "r"(a[7]), "r"(a[8]), "r"(a[9]),
      "r"(a[10]), "r"(a[11]), "r"(a[12]), "r"(a[13]), "r"(a[14]), "r"(a[15])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

MBP_DEV void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

MBP_DEV void tc_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Eight columns of the accumulator (lane = row).
MBP_DEV void tc_ld8(uint32_t taddr, float (&v)[8]) {
  uint32_t u[8];
  __syncwarp();
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]);
}

// Weight units as a 3-D tensor of u64 with a box of 8 row tiles x 2 sub-tiles per stage:
//   12-bit units [R][C][1536 bytes] -> {192, C, R}, box {192, 2, 8} (chunks c, c + 1; {192, 1, 8} for a matrix of
//   one chunk);
//   hi/lo units  [R][C][2][2048 bytes] -> {256, 2C, R}, box {256, 2, 8} (chunk c = indices 2c, 2c + 1).
// (Measured alternative: 128-byte rows with a 128-byte swizzle and a ring as deep as shared memory allows was
// 10-15 % slower; the decoders' instruction issue, not the copy engine, bounds the small-M calls.)
inline bool encode_units_3d(CUtensorMap* map, const void* units, int R, int C, bool hilo) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t inner = hilo ? 256 : 192, mid = hilo ? 2 * (cuuint64_t)C : (cuuint64_t)C;
  const cuuint64_t row = (cuuint64_t)C * (hilo ? 2 * MBP_RAW_UNIT_BYTES : MBP_C12_UNIT_BYTES);
  const cuuint64_t dims[3] = {inner, mid, (cuuint64_t)R};
  const cuuint64_t strides[2] = {inner * 8, row};
  const cuuint32_t box[3] = {(cuuint32_t)inner, mid >= 2 ? 2u : 1u, 8};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT64, 3, const_cast<void*>(units), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace mbp
