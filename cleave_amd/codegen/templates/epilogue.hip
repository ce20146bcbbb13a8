// ---- what follows a matrix product before it is stored: y = act(x w + bias) + residual -----------------
//
// The sums of the product are f32 and stay so: bias and residual are widened, the activation is taken in f32, and the result
// is rounded to the element type once.  (A product stored in the element type, and read again by a kernel that adds and
// activates, is rounded twice and moves 4 M N bytes more.)
//   CL_EPI_ACT   0 none, 1 relu, 2 silu, 3 gelu, 4 gelu's tanh form     CL_EPI_BIAS  a row (1, N)     CL_EPI_RES  (M, N)
//
// silu(x) = x / (1 + e^-x).  The tanh form of gelu is x / 2 (1 + tanh u) = x / (1 + e^-2u), u = sqrt(2 / pi) (x + 0.044715 x^3).
// Where e^.. overflows, the quotient is -0 and x, as the limits are.
// gelu(x) = x / 2 erfc(-x / sqrt 2).  With u = |x| sqrt(log2(e) / 2), erfc(|x| / sqrt 2) / 2 = 2^(-u^2) q(u), and q is a polynomial in t = 1 /
// (1 + 0.325 |x|) without a constant term, fitted here to e^(x^2 / 2) erfc(|x| / sqrt 2) / 2 over [0, 200] by reweighted least squares:
// relative error 6.7e-7, with f32 arithmetic 8e-7 for positive x (to f16 a six-hundredth of a rounding) and, where 2^(-u^2) rounds u^2, 2e-6
// down to x = -5; erfc(-z) = 2 - erfc(z).  Vector instructions bound it, 16 and two of quarter rate: f16 4096 x 4096 x 1024, us, no
// activation 32.5, silu 33.7, gelu's tanh form 34.8, gelu 39.1 (40.3 with nine coefficients and factors of their own).
CL_DEVICE float ep_exp(float x) { return fast_exp2(x * 1.4426950408889634f); }

CL_DEVICE float ep_act(float x) {
#if CL_EPI_ACT == 1
  return x < 0.f ? 0.f : x;                 // (NaN stays NaN)
#elif CL_EPI_ACT == 2
  return x * fast_rcp(1.0f + ep_exp(-x));
#elif CL_EPI_ACT == 3
  const float u = fabsf(x) * 0.8493217825889587f;
  const float t = fast_rcp(__builtin_fmaf(u, 0.3826582431793213f, 1.0f));
  float q = 0.0338912196457386f;
  q = __builtin_fmaf(q, t, -0.11376706510782242f);
  q = __builtin_fmaf(q, t, 0.08563332259654999f);
  q = __builtin_fmaf(q, t, 0.025832246989011765f);
  q = __builtin_fmaf(q, t, 0.09359048306941986f);
  q = __builtin_fmaf(q, t, 0.11549093574285507f);
  q = __builtin_fmaf(q, t, 0.1296730637550354f);
  q = __builtin_fmaf(q, t, 0.1296561360359192f);
  const float tail = (q * t) * fast_exp2(-(u * u));
  return x * (x < 0.f ? tail : 1.0f - tail);
#elif CL_EPI_ACT == 4
  return x * fast_rcp(1.0f + ep_exp(x * __builtin_fmaf(x * x, -0.07135481282687187f, -1.5957691216057308f)));
#else
  return x;
#endif
}

// W neighbouring elements from column n of a row on (past the row's end: its last ones again; their results are not stored)
template <int W> CL_DEVICE void ep_read(const elem_t* row, int n, float (&v)[W]) {
  if constexpr (W > 1 && CL_N % W == 0) {
    typedef elem_t piece_t __attribute__((ext_vector_type(W)));
    const piece_t piece = *reinterpret_cast<const piece_t*>(row + (n < CL_N ? n : CL_N - W));
#pragma unroll
    for (int r = 0; r < W; ++r) v[r] = to_f32(piece[r]);
  } else {
#pragma unroll
    for (int r = 0; r < W; ++r) v[r] = to_f32(row[n + r < CL_N ? n + r : CL_N - 1]);
  }
}
// Columns n .. n + W - 1 of row m of the product, in place (n a multiple of W where rows are whole pieces of W)
template <int W> CL_DEVICE void ep_finish(float (&v)[W], const elem_t* __restrict__ bias, const elem_t* __restrict__ res, int m, int n) {
  float add[W];
#if CL_EPI_BIAS
  ep_read<W>(bias, n, add);
#pragma unroll
  for (int r = 0; r < W; ++r) v[r] += add[r];
#endif
#pragma unroll
  for (int r = 0; r < W; ++r) v[r] = ep_act(v[r]);
#if CL_EPI_RES
  ep_read<W>(res + (i64)(m < CL_M ? m : CL_M - 1) * CL_N, n, add);
#pragma unroll
  for (int r = 0; r < W; ++r) v[r] += add[r];
#endif
  (void)add;
}
CL_DEVICE f32x4 ep_apply(f32x4 v, const elem_t* __restrict__ bias, const elem_t* __restrict__ res, int m, int n) {
  float f[4] = {v[0], v[1], v[2], v[3]};
  ep_finish<4>(f, bias, res, m, n);
  return (f32x4){f[0], f[1], f[2], f[3]};
}
// The same in two halves, for wave tiles of many fragments: the pieces of bias and residual are asked for all at once, ahead of the
// first use (fragment by fragment every wait was in sight: 4096 x 4096 x 1024 with a residual 42.5 us, 40.7 this way, the bare
// product 32.1), and each fragment is finished with what has come.
CL_DEVICE elem4 ep_piece(const elem_t* __restrict__ row, int n) {
  if constexpr (CL_N % 4 == 0) return *reinterpret_cast<const elem4*>(row + (n < CL_N ? n : CL_N - 4));
  elem4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = row[n + r < CL_N ? n + r : CL_N - 1];
  return v;
}
CL_DEVICE elem4 ep_bias(const elem_t* __restrict__ bias, int n) {
#if CL_EPI_BIAS
  return ep_piece(bias, n);
#else
  return (elem4){};
#endif
}
CL_DEVICE const elem_t* ep_res_row(const elem_t* __restrict__ res, int m) { return res + (i64)(m < CL_M ? m : CL_M - 1) * CL_N; }
CL_DEVICE f32x4 ep_with(f32x4 v, elem4 bias, elem4 res) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    v[r] = ep_act(CL_EPI_BIAS ? v[r] + to_f32(bias[r]) : v[r]);
    if (CL_EPI_RES) v[r] += to_f32(res[r]);
  }
  return v;
}
#if CL_EPI_BIAS
#define EP_BIAS CL_ARG_BIAS
#else
#define EP_BIAS nullptr
#endif
#if CL_EPI_RES
#define EP_RES CL_ARG_RES
#else
#define EP_RES nullptr
#endif
