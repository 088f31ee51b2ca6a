// The loop of a softmax warp of text_fwd_kernel over an item's key tiles, in that kernel's scope. It is included once for every number of terms in which a probability goes into its
// product, with TWO set: a lambda called for either number cost the kernels with one number a share of their time (six prompts 268 -> 276 us, relative attention 87 -> 88.5).
for (int i = 0, kt = w.key_tile(0); i < w.n_kv; ++i, kt = i == w.ns ? w.lo : kt + 1) {
  if (kt >= my_hi || (kt < my_lo && kt >= w.ns)) continue;
  const int k0 = kt * TK;
  ok = text_wait<DH == 128>(&s_full[t], done & 1, &abort_s);
  if (!ok) break;
  tc_fence_after();
  uint32_t sv[PIECES][32];
#pragma unroll
  for (int c = 0; c < PIECES; ++c) tmem_ld_32x32b_x32(s_tile + c * 32, sv[c]);
  tmem_wait_ld();
  float mul = sl2, add = 0.f;           // exponent = mul * score + add - m
  if (BIAS) {
    const int d = k0 - row0;
    if (d - 31 >= lut.near) add = lut.behind();
    else if (d + TK - 1 <= -lut.near) add = lut.before();
    else {
      const float* b = lut.from(d - lane);
      mul = 1.f;
#pragma unroll
      for (int c = 0; c < PIECES; ++c)
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 u = *reinterpret_cast<const float4*>(b + c * 32 + e);
          const float2 x01 = ffma2(make_float2(__uint_as_float(sv[c][e]), __uint_as_float(sv[c][e + 1])), make_float2(sl2, sl2), make_float2(u.x, u.y));
          const float2 x23 = ffma2(make_float2(__uint_as_float(sv[c][e + 2]), __uint_as_float(sv[c][e + 3])), make_float2(sl2, sl2), make_float2(u.z, u.w));
          sv[c][e] = __float_as_uint(x01.x);
          sv[c][e + 1] = __float_as_uint(x01.y);
          sv[c][e + 2] = __float_as_uint(x23.x);
          sv[c][e + 3] = __float_as_uint(x23.y);
        }
    }
  }
  if (k0 > whole_hi || (!BIAS && k0 < whole_lo && k0 + TK > a.sinks)) {
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
      const uint32_t see = BIAS ? bits_below(valid - k0 - c * 32) : text_mask(a, valid, p0 + lane, k0 + c * 32);
      if (__all_sync(0xffffffffu, see == 0xffffffffu)) continue;
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (!(see >> e & 1u)) sv[c][e] = 0xff800000u;        // -inf
    }
  }
  float mc[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int e = 0; e < 32; e += 8 / PIECES)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      constexpr int PER = 4 / PIECES;                 // chains in a piece
      const int c = n / PER, at = e + 2 * (n % PER);
      mc[n] = max3_nan(mc[n], __uint_as_float(sv[c][at]), __uint_as_float(sv[c][at + 1]));
    }
  const float mx = fmaf(max_nan(max3_nan(mc[0], mc[1], mc[2]), mc[3]), mul, add);
  if (fresh) {
    if (!(mx <= m_used)) {                // larger, or NaN
      l_run *= exp2f(m_used - mx);
      m_used = max_nan(m_used, mx);
    }
  } else {
    // The reference is raised when a row has outgrown it by more than 2^8, and with the first key that a row sees.
    const bool need = !(mx <= m_used + 8.0f);      // NaN, too
    if (__any_sync(0xffffffffu, need)) {
      ok = text_wait<DH == 128>(&o_full[t], (done - 1) & 1, &abort_s);
      if (!ok) break;
      tc_fence_after();
      const float alpha = need ? exp2f(m_used - mx) : 1.0f;
      if (need) m_used = max_nan(m_used, mx);
      l_run *= alpha;
#pragma unroll 1
      for (int c = 0; c < DH / 16; ++c) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(o_addr + c * 16, r);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
        tmem_st_32x32b_x16(o_addr + c * 16, r);
      }
      tmem_wait_st();
    }
  }
  // No key so far: every exponent is -inf. A score of +inf: NaN, as the difference of two such scores; all of the row's exponents, for the
  // polynomial takes a share of them and does not know NaN.
  const float m_now = m_used == -INFINITY ? 0.f : m_used < INFINITY ? m_used : NAN;
  float2 sum_a = make_float2(0.f, 0.f), sum_b = make_float2(0.f, 0.f);
  const float2 mul2 = make_float2(mul, mul), nm2 = make_float2(add - m_now, add - m_now);
  // four neighbours' exponentials, those of columns e and e + 2 in u, of e + 1 and e + 3 in v
  const auto exps = [&](int c, int e, float2& u, float2& v) {
    // Half of every second group of four exponentials runs on the FMA pipe, the rest on the special-function unit (1 x 4096 x 37 x 64, all keys
    // visible: 208 us, 216 without). Beside the biases of heads of 64 instructions are scarcer: all on the unit (232 us, 249 with).
    const float2 x01 = ffma2(make_float2(__uint_as_float(sv[c][e]), __uint_as_float(sv[c][e + 1])), mul2, nm2);
    const float2 x23 = ffma2(make_float2(__uint_as_float(sv[c][e + 2]), __uint_as_float(sv[c][e + 3])), mul2, nm2);
    u = make_float2(ex2_approx(x01.x), ex2_approx(x23.x));
    if (!(DH == 64 && BIAS) && (e >> 2) % 2 == 1) v = ex2_poly2(make_float2(x01.y, x23.y), -127.f);
    else v = make_float2(ex2_approx(x01.y), ex2_approx(x23.y));
    sum_a = fadd2(sum_a, u);
    sum_b = fadd2(sum_b, v);
  };
  const auto publish = [&](int c) {      // 64 keys
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&p_full[t][c >> 1]);
  };
  if constexpr (TWO) {
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pk[8], low[8];
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          float2 u, v;
          exps(c, h * 16 + e, u, v);
          pk[e >> 1] = pack_bf16x2(u.x, v.x);
          pk[(e >> 1) + 1] = pack_bf16x2(u.y, v.y);
          const float2 h0 = unpack_bf16x2(pk[e >> 1]), h1 = unpack_bf16x2(pk[(e >> 1) + 1]);
          low[e >> 1] = pack_bf16x2(u.x - h0.x, v.x - h0.y);
          low[(e >> 1) + 1] = pack_bf16x2(u.y - h1.x, v.y - h1.y);
        }
        tmem_st_32x32b_x8(s_tile + c * 16 + h * 8, pk);
        tmem_st_32x32b_x8(s_tile + TK / 2 + c * 16 + h * 8, low);
      }
      if (c & 1) publish(c);
    }
  } else {
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
      uint32_t pk[16];
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        float2 u, v;
        exps(c, e, u, v);
        pk[e >> 1] = pack_bf16x2(u.x, v.x);
        pk[(e >> 1) + 1] = pack_bf16x2(u.y, v.y);
      }
      tmem_st_32x32b_x16(s_tile + c * 16, pk);          // over scores that are in registers by now
      if (c & 1) publish(c);
    }
  }
  l_run += (sum_a.x + sum_a.y) + (sum_b.x + sum_b.y);
  ++done;
  fresh = false;
}
