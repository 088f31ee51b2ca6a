// The loop of a math warp of text_bwd_kernel over the streamed tiles, in that kernel's scope. It is included once for every number of terms in which P and dS go into their products,
// with FINE (two) set: as a lambda called for either number it cost the kernels with one number registers (relative attention's training step 225.7 -> 228.5 us), and two bodies of the
// whole kernel the packed one's instruction cache (139 us instead of 133 for dq).
for (int i = i_begin; i < n_c; i += BUFS) {
  const uint32_t par = (BUFS == 2 ? i >> 1 : i) & 1;
  const int place = i & (PLACES - 1), half = place * 32;      // where this tile's queries are staged
  uint64_t* staged = &lv_full[g][place];
  if (KEYS) {
    while (in_head >= per_head) in_head -= per_head;
    // Two buffers: the place was last read for tile i - 2, and the warpgroup's four warps have all arrived on pds_full[g] for it. One buffer: also for
    // tile i - 2, and the scores of tile i - 1, which this warp has seen, were only formed after all warps had arrived for it. By then
    // all warps have also left their wait for the queries of tile i - 2, the place's barrier's last phase. (A barrier for both places would
    // not do: a warp may still wait for tile i - 1's phase, and could not tell it from the one after tile i's, which has its parity.)
    bool lv_ok = true;
    if (stager) {
      if (BUFS == 2 && i >= 2) lv_ok = mbar_wait(&pds_full[g], par ^ 1u, &abort_s);
      s_lse[g][half + mt] = next_nlse;
      s_delta[g][half + mt] = next_ndelta;
      mbar_arrive(staged);
    }
    if (stager && i + BUFS < n_c) fetch(BUFS);
    ok = text_wait<DH == 128>(staged, (i >> 1) & 1, &abort_s);
    ok = __all_sync(0xffffffffu, ok && lv_ok);
    if (!ok) break;
  }
  const int c0 = tile_of(in_head) * TC;          // first key (dq) or query (KEYS) of the tile
  ok = text_wait<DH == 128>(&xy_full[BUFS == 2 ? g : 0], par, &abort_s);
  if (!ok) break;
  tc_fence_after();
  constexpr int NC = BUFS;                       // pieces of 32 columns of a thread: all of the tile's, or one
  const int piece0 = BUFS == 1 ? g : 0;
  uint32_t xr[NC][32], yr[NC][32];
  float run[NC][32];                             // BIAS dq: dS
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    tmem_ld_32x32b_x32(xa + (piece0 + c) * 32, xr[c]);
    tmem_ld_32x32b_x32(ya + (piece0 + c) * 32, yr[c]);
  }
  tmem_wait_ld();
  bool whole;       // every pair of the tile is visible, or its row or query lies behind the last one and has a probability of zero anyway
  if (BIAS) whole = KEYS ? r0 + TR <= sight.valid : c0 + TC <= sight.valid;
  else if (KEYS) whole = r0 + TR <= sight.valid && r0 + TR - 1 <= sight.start + c0 && (sight.start + c0 + TC - 1 - a.window < r0 || r0 + TR <= a.sinks);
  else whole = c0 + TC <= sight.valid && c0 + TC - 1 <= sight.start + r0 && (sight.start + r0 + TR - 1 - a.window < c0 || c0 + TC <= a.sinks);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int b0 = c0 + (piece0 + c) * 32;
    uint32_t see = 0xffffffffu;
    if (!whole) {
      if (BIAS) see = KEYS ? (row < sight.valid ? see : 0u) : bits_below(sight.valid - b0);
      else if (KEYS) see = row < sight.valid ? ~bits_below(row - sight.start - b0) & (row < a.sinks ? see : bits_below(row + a.window - sight.start - b0)) : 0u;
      else see = text_mask(a, sight.valid, sight.start + row, b0);
    }
    // BIAS: distances of the warp's 32 x 32 block lie in d0 - 31 .. d0 + 31
    const int d0 = KEYS ? r0 + quad * 32 - b0 : b0 - (r0 + quad * 32);
    const bool uniform = BIAS && (d0 - 31 >= near || d0 + 31 <= -near);
    float one_bias = 0.f;
    const float* b = nullptr;
    if (BIAS) {
      // four neighbours in one load: distances grow along the keys, and fall along the queries
      if (uniform) one_bias = d0 > 0 ? lut.behind() : lut.before();
      else b = lut.from(KEYS ? row - b0 - 3 : b0 - row);
    }
    uint32_t pk[16], dk[16];      // FINE: of 16 columns, [0, 8), and what their rounding left, [8, 16)
    const float2 sl2_2 = make_float2(sl2, sl2);
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
      float nl[4], nd[4];
      if (KEYS) {
        const float4 u = *reinterpret_cast<const float4*>(&s_lse[g][half + c * 32 + e]), w = *reinterpret_cast<const float4*>(&s_delta[g][half + c * 32 + e]);
        nl[0] = u.x; nl[1] = u.y; nl[2] = u.z; nl[3] = u.w;
        nd[0] = w.x; nd[1] = w.y; nd[2] = w.z; nd[3] = w.w;
      } else {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          nl[m] = my_nlse;
          nd[m] = my_ndelta;
        }
      }
      if (BIAS) {
        float4 u = make_float4(one_bias, one_bias, one_bias, one_bias);
        if (!uniform) u = *reinterpret_cast<const float4*>(b + (KEYS ? -e : e));
        nl[0] += KEYS ? u.w : u.x;
        nl[1] += KEYS ? u.z : u.y;
        nl[2] += KEYS ? u.y : u.z;
        nl[3] += KEYS ? u.x : u.w;
      }
      const float2 x01 = ffma2(make_float2(__uint_as_float(xr[c][e]), __uint_as_float(xr[c][e + 1])), sl2_2, make_float2(nl[0], nl[1]));
      const float2 x23 = ffma2(make_float2(__uint_as_float(xr[c][e + 2]), __uint_as_float(xr[c][e + 3])), sl2_2, make_float2(nl[2], nl[3]));
      float2 p01 = make_float2(ex2_approx(x01.x), ex2_approx(x01.y)), p23 = make_float2(ex2_approx(x23.x), ex2_approx(x23.y));
      if (!whole) {
        if (!(see >> e & 1u)) p01.x = 0.f;
        if (!(see >> (e + 1) & 1u)) p01.y = 0.f;
        if (!(see >> (e + 2) & 1u)) p23.x = 0.f;
        if (!(see >> (e + 3) & 1u)) p23.y = 0.f;
      }
      const float2 d01 = fmul2(p01, fadd2(make_float2(__uint_as_float(yr[c][e]), __uint_as_float(yr[c][e + 1])), make_float2(nd[0], nd[1])));
      const float2 d23 = fmul2(p23, fadd2(make_float2(__uint_as_float(yr[c][e + 2]), __uint_as_float(yr[c][e + 3])), make_float2(nd[2], nd[3])));
      const int at = (FINE ? e & 15 : e) >> 1;
      pk[at] = pack_bf16x2(p01.x, p01.y);
      pk[at + 1] = pack_bf16x2(p23.x, p23.y);
      dk[at] = pack_bf16x2(d01.x, d01.y);
      dk[at + 1] = pack_bf16x2(d23.x, d23.y);
      if constexpr (FINE) {
        const auto rest = [](float2 x, uint32_t rounded) {
          const float2 h = unpack_bf16x2(rounded);
          return pack_bf16x2(x.x - h.x, x.y - h.y);
        };
        if (KEYS) {
          pk[at + 8] = rest(p01, pk[at]);
          pk[at + 9] = rest(p23, pk[at + 1]);
        }
        dk[at + 8] = rest(d01, dk[at]);
        dk[at + 9] = rest(d23, dk[at + 1]);
        if ((e & 15) == 12) {
          const auto store = [&](uint32_t to, const uint32_t (&w)[16]) {
            uint32_t high[8], low[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) {
              high[m] = w[m];
              low[m] = w[m + 8];
            }
            tmem_st_32x32b_x8(to, high);
            tmem_st_32x32b_x8(to + 16, low);
          };
          if (KEYS) store(xa + (piece0 + c) * 32 + (e >> 4) * 8, pk);
          store(ya + (piece0 + c) * 32 + (e >> 4) * 8, dk);
        }
      }
      if (BIAS && !KEYS) {
        run[c][e] = d01.x;
        run[c][e + 1] = d01.y;
        run[c][e + 2] = d23.x;
        run[c][e + 3] = d23.y;
      }
    }
    if constexpr (!FINE) {
      if (KEYS) tmem_st_32x32b_x16(xa + (piece0 + c) * 32, pk);      // over scores of this piece: they are in registers by now
      tmem_st_32x32b_x16(ya + (piece0 + c) * 32, dk);
    }
  }
  tmem_wait_st();
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(&pds_full[BUFS == 2 ? g : 0]);
  if (SUMMED && a.d_table != nullptr) {
    // with the tile's products under way
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int b0 = c0 + (piece0 + c) * 32, d0 = b0 - (r0 + quad * 32);
      const int r_lo = run_of[min(max(sum_end - (r0 + quad * 32) - 32 + near, 0), 2 * near)], r_hi = run_of[min(max(d0 + 31 + near, 0), 2 * near)];
      // running sums of four pieces of eight, then of the whole
#pragma unroll
      for (int e = 1; e < 8; ++e)
#pragma unroll
        for (int m = 0; m < 32; m += 8) run[c][m + e] += run[c][m + e - 1];
#pragma unroll
      for (int m = 8; m < 32; m += 8) {
        const float base = run[c][m - 1];
        if (r_lo == r_hi) {
          run[c][m + 7] += base;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) run[c][m + e] += base;
        }
      }
      if (r_lo != r_hi) {
        float* mine = sums + ((warp - 2) * 32 + lane) * RUN_LD;
#pragma unroll
        for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(mine + e) = make_float4(run[c][e], run[c][e + 1], run[c][e + 2], run[c][e + 3]);
        // Bucket r + 1 of this row begins at key `at`: what came before it. Where that key lies in a tile of the other warpgroup, the sum so far.
#pragma unroll 4
        for (int r = r_lo; r < r_hi; ++r) {
          const int at = run_start[r + 1] + row;
          const float upto = at > b0 ? mine[min(at - b0, 32) - 1] : 0.f;
          if (at >= sum_end && at < b0 + 32) bins[r * 256 + slot] = sum_all + upto;
        }
      }
      sum_all += run[c][31];
      sum_end = b0 + 32;
    }
  }
  in_head += BUFS;
}
