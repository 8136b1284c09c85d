// Epilogue of a projection: out = residual + mul * act(y + bias), on the FP32 accumulator y, rounded once to the
// output type; and the lookup of a token tile among rows sorted by expert.  Shared by the GEMV and the GEMM.
#pragma once
#include "common.cuh"

namespace mbp {

// By value in the kernels' parameters (mbp_epilogue with the output type and the leading dimensions widened).
struct EpiArgs {
  const void* bias;      // [n] (of one expert: [experts][n]) or null
  const void* mul;       // [m][ld_mul] or null
  const void* residual;  // [m][ld_res] or null; may be the output itself: each element is read by its writer, before
  long long ld_mul, ld_res;
  int bias_f32, mul_f32, res_f32, act, out_f32;
  int wide;  // mul, residual and out are BF16 (or absent), each row on 16 bytes: eight columns move at once
};

// Rows sorted by expert: rows offsets[e] .. offsets[e+1] are expert e's (null: one matrix, no experts).
struct GroupArgs {
  const int32_t* offsets;
  int experts, rows;
  int zero_tail;  // output rows from offsets[experts] on are set to zero (else left as they are)
};

// N elements of an operand at `at + off(i)`, 0 where !in(i).  One uniform branch on the type around all loads and the
// conversions after them: a branch per element made each load wait for the one before.  epi_bits leaves the conversion
// (epi_value) to the place that needs the number.
template <int N, class Off, class In>
MBP_DEV void epi_bits(const void* p, int f32, long long at, Off&& off, In&& in, uint32_t (&v)[N]) {
  if (f32) {
    const uint32_t* q = static_cast<const uint32_t*>(p) + at;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = in(i) ? q[off(i)] : 0u;
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(p) + at;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = in(i) ? q[off(i)] : 0u;
  }
}
MBP_DEV float epi_value(uint32_t bits, int f32) { return __uint_as_float(f32 ? bits : bits << 16); }

template <int N, class Off, class In>
MBP_DEV void epi_load(const void* p, int f32, long long at, Off&& off, In&& in, float (&v)[N]) {
  if (f32) {
    const float* q = static_cast<const float*>(p) + at;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = in(i) ? q[off(i)] : 0.f;
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(p) + at;
    uint16_t raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = in(i) ? q[off(i)] : (uint16_t)0;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float((uint32_t)raw[i] << 16);
  }
}

// 1 / (1 + e^-u) from e^-|u|, which cannot overflow: the denominator stays in [1, 2], where __fdividef is good to 2 units
// in the last place (it gives 0 for one above 2^126, so 1 / (1 + e^-u) itself is 0 below u = -87.3, where silu is still
// 1e-36).  Over that form it costs expert products whose epilogue paces them 5 % (64 experts of 6144 x 1536, 1024 tokens,
// silu and multiplier: 411 -> 434 us) and the others under 1 %; clamping u in place of the select is no cheaper.
MBP_DEV float logistic(float u) {
  const float t = expf(-fabsf(u));
  return __fdividef(u < 0.f ? t : 1.f, 1.f + t);
}

// The activations in forms whose relative error does not grow where they approach zero: erfc and a logistic
// instead of 1 + erf and 1 + tanh.  A NaN stays a NaN (relu compares so that it does).  The choice is made once for
// N results: made per result it cost a 256-token tile 12 us.
template <int N>
MBP_DEV void epi_act(float (&z)[N], int act) {
  switch (act) {
    case MBP_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = z[i] < 0.f ? 0.f : z[i];
      break;
    case MBP_ACT_RELU2:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = z[i] < 0.f ? 0.f : z[i] * z[i];
      break;
    case MBP_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = 0.5f * z[i] * erfcf(z[i] * -0.70710678118654752f);
      break;
    case MBP_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i)  // 2 sqrt(2 / pi)
        z[i] *= logistic(1.5957691216057308f * (z[i] + 0.044715f * z[i] * z[i] * z[i]));
      break;
    case MBP_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] *= logistic(z[i]);
      break;
    case MBP_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = logistic(z[i]);
      break;
    default: break;
  }
}

// N results of one thread, result i at element at + off(i, ld) of a matrix of row stride ld (at: row `row` of token
// tok), where in(i); bias(i) is its bias.  Every operand is loaded before any result is stored, so the loads are in
// flight together.
template <int N, class Off, class In, class Bias>
MBP_DEV void epi_emit(const EpiArgs& e, void* out, long long ldo, float (&y)[N], Bias&& bias, int row, int tok,
                      Off&& off, In&& in) {
  uint32_t a[N], r[N];  // as they are in memory: a conversion of the first operand would hold up the second's
                        // loads (64 experts of 6144 x 1536, 1024 tokens, silu, bias, mul, FP32 residual: 873 -> 748 us)
  if (e.mul)
    epi_bits<N>(e.mul, e.mul_f32, tok * e.ld_mul + row, [&](int i) { return off(i, e.ld_mul); }, in, a);
  if (e.residual)
    epi_bits<N>(e.residual, e.res_f32, tok * e.ld_res + row, [&](int i) { return off(i, e.ld_res); }, in, r);
  if (e.bias) {
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] += bias(i);
  }
  epi_act<N>(y, e.act);
  if (e.mul) {
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] *= epi_value(a[i], e.mul_f32);
  }
  if (e.residual) {
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] += epi_value(r[i], e.res_f32);
  }
  if (e.out_f32) {
    float* o = static_cast<float*>(out) + tok * ldo + row;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in(i)) o[off(i, ldo)] = y[i];
  } else {
    uint16_t* o = static_cast<uint16_t*>(out) + tok * ldo + row;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in(i)) o[off(i, ldo)] = __bfloat16_as_ushort(__float2bfloat16_rn(y[i]));
  }
}

// One row of the weights, tokens tok .. tok + n - 1 (n <= N).
template <int N>
MBP_DEV void epi_column(const EpiArgs& e, void* out, long long ldo, float (&y)[N], float bias, int row, int tok, int n) {
  epi_emit<N>(e, out, ldo, y, [&](int) { return bias; }, row, tok, [](int i, long long ld) { return i * ld; },
              [&](int i) { return i < n; });
}

// An mma.sync accumulator: rows row and row + 8, tokens tok and tok + 1 (n >= 1 of them), v = (row, tok), (row, tok + 1),
// (row + 8, tok), (row + 8, tok + 1).  b: the two rows' bias (epi_fragment_bias).
MBP_DEV void epi_fragment(const EpiArgs& e, void* out, long long ldo, float4 v, const float2 b, int row, int tok, int n) {
  float y[4] = {v.x, v.y, v.z, v.w};
  epi_emit<4>(e, out, ldo, y, [&](int i) { return i < 2 ? b.x : b.y; }, row, tok,
              [](int i, long long ld) { return 8 * (i >> 1) + (i & 1) * ld; }, [&](int i) { return (i & 1) < n; });
}

// Bias elements `at` and at + 8 (0 without one).
MBP_DEV float2 epi_fragment_bias(const EpiArgs& e, long long at) {
  float b[2] = {0.f, 0.f};
  if (e.bias) epi_load<2>(e.bias, e.bias_f32, at, [](int i) { return 8 * i; }, [](int) { return true; }, b);
  return make_float2(b[0], b[1]);
}

// One element of the bias (0 without one).
MBP_DEV float epi_bias(const EpiArgs& e, long long at) {
  float v[1] = {0.f};
  if (e.bias) epi_load<1>(e.bias, e.bias_f32, at, [](int) { return 0; }, [](int) { return true; }, v);
  return v[0];
}

// Pulls the multiplier's and the residual's elements of columns [c0, c1), tokens [t0, t1) into L2 (hints; threads
// tid of nthr, any alignment), long before the epilogue reads them.
MBP_DEV void epi_prefetch(const EpiArgs& e, int c0, int c1, int t0, int t1, int tid, int nthr) {
  const auto rows = [&](const void* p, int f32, long long ld) {
    if (!p) return;
    const int es = f32 ? 4 : 2, lines = ((c1 - c0) * es + 127) / 128;  // (the last line of an unaligned row is left out)
    for (int i = tid; i < (t1 - t0) * lines; i += nthr) {
      const int t = i / lines;
      const char* q = static_cast<const char*>(p) + ((t0 + t) * ld + c0) * es + (long long)(i - t * lines) * 128;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
    }
  };
  rows(e.mul, e.mul_f32, e.ld_mul);
  rows(e.residual, e.res_f32, e.ld_res);
}

// Zeroes columns [c0, c1) of the output rows from offsets[experts] on: rows first, first + step, ... of them, by the
// block's threads.
MBP_DEV void zero_tail(const GroupArgs& g, const EpiArgs& e, void* out, long long ldo, int c0, int c1, int first,
                       int step, int tid, int nthr) {
  const int total = min(max(g.offsets[g.experts], 0), g.rows);
  for (long long r = (long long)total + first; r < g.rows; r += step)
    for (int c = c0 + tid; c < c1; c += nthr) {
      if (e.out_f32)
        static_cast<float*>(out)[r * ldo + c] = 0.f;
      else
        static_cast<uint16_t*>(out)[r * ldo + c] = 0;
    }
}

// ---- host ----
// Largest number of tiles of `tile` rows that `rows` rows of `experts` experts can make (the last tile of an expert
// may hold a single row).
inline long long max_tiles(int experts, int rows, int tile) {
  const int used = experts < rows ? experts : rows;
  return used + (rows - used) / tile;
}

inline int check_epilogue(const mbp_epilogue* epi, int n_out, const void* out, int ldo, EpiArgs* e) {
  *e = EpiArgs{};
  const auto wide = [](const void* p, int f32, long long ld) {
    return !p || (!f32 && ((uintptr_t)p & 15u) == 0 && ld % 8 == 0);
  };
  e->wide = wide(out, 0, ldo);
  if (!epi) return MBP_OK;
  const auto flag = [](int v) { return v == 0 || v == 1; };
  const auto off = [](const void* p, int f32) { return ((uintptr_t)p & (f32 ? 3u : 1u)) != 0; };
  if (epi->activation < MBP_ACT_NONE || epi->activation > MBP_ACT_SIGMOID) return MBP_ERR_ARG;
  if (!flag(epi->bias_f32) || !flag(epi->mul_f32) || !flag(epi->residual_f32) || !flag(epi->out_f32)) return MBP_ERR_ARG;
  if ((epi->mul && epi->ld_mul < n_out) || (epi->residual && epi->ld_residual < n_out)) return MBP_ERR_SHAPE;
  if (off(epi->bias, epi->bias_f32) || off(epi->mul, epi->mul_f32) || off(epi->residual, epi->residual_f32) ||
      off(out, epi->out_f32))
    return MBP_ERR_ALIGN;
  *e = EpiArgs{epi->bias,     epi->mul,     epi->residual,     epi->ld_mul,     epi->ld_residual,
               epi->bias_f32, epi->mul_f32, epi->residual_f32, epi->activation, epi->out_f32,
               wide(out, epi->out_f32, ldo) && wide(epi->mul, epi->mul_f32, epi->ld_mul) &&
                   wide(epi->residual, epi->residual_f32, epi->ld_residual)};
  return MBP_OK;
}

}  // namespace mbp
