// Body of the 128-row kernel of bank4_read.hip, which says what it does (DK, DVC, PARTS, F16, CAUSAL, the arguments `a` and `again` are the including function's).
  typedef typename ReadType<PARTS>::T T;
  constexpr bool KEYS_F16 = F16 && PARTS > 1, SHIFT = F16 && PARTS == 3;
  typedef std::conditional_t<KEYS_F16, f16x8, bf16x8> K8;
  typedef std::conditional_t<F16, f16x8, bf16x8> V8;
  constexpr int QP = KEYS_F16 ? PARTS - 1 : PARTS, PP = F16 && PARTS == 1 ? 1 : PARTS == 3 && !F16 ? 3 : 2;
  constexpr float LAG = F16 ? PARTS == 1 ? 7.f : 3.f : MAX_LAG, P_UP = F16 ? PARTS == 1 ? 8.f : 12.f : 0.f;        // weights are exp2(logit - (maximum - P_UP)), up to 2^(LAG + P_UP)
  constexpr int VS = DVC + 16, NT = DVC / 32, VB = DVC / 32, VE = 64 * VB, VL = (VE + 255) / 256;
  extern __shared__ __align__(16) __bf16 vt[];         // two buffers of 64 rows
  __shared__ uint64_t nan_blocks[2][4][VL];            // causal: the value blocks of a buffer that stand for NaN, a bit a lane of the wave that stored it
  __shared__ uint32_t key_limit;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int nvc = a.value_dim / DVC, chunk = blockIdx.z % nvc, bh = blockIdx.z / nvc, b = bh / a.heads, h = bh - b * a.heads;
  const int split = blockIdx.x, row0 = blockIdx.y * 128, r = row0 + wave * 32 + col;
  const int64_t len = read_len(a, b);
  const int cnt = read_count(a, b), t = r / a.group;
  const bool live = r < a.rows && t < cnt;
  const int limit = live && CAUSAL ? (int)read_limit(a, len, cnt, t) : (int)len;
  int last_t = (row0 + 127 < a.rows ? row0 + 127 : a.rows - 1) / a.group;
  last_t = last_t < cnt ? last_t : cnt - 1;
  const int seen = row0 / a.group < cnt ? (int)read_limit(a, len, cnt, last_t) : 0;
  const int per = ((seen + 63) / 64 + a.nsplit - 1) / a.nsplit * 64;
  const int s0 = (int64_t)split * per < seen ? split * per : seen, s1 = seen - s0 < per ? seen : s0 + per;
  int low = limit;                                   // over the wave's rows
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_xor(low, d);
    low = x < low ? x : low;
  }
  low = __builtin_amdgcn_readfirstlane(low);

  QueryCols<DK, QP, K8> q;
  float lost = 0.f;
  const float back = q.template load<SHIFT>((const T *)a.q + b * a.qb + (int64_t)(live ? t : 0) * a.qt + (int64_t)(h * a.group + (live ? r - t * a.group : 0)) * a.qh, half, live, a.q_vec, a.q_sign, lost);
  const float scale = SHIFT ? row_scale(a.scale_log2, back) : a.scale_log2;
  uint32_t key_most = kBank4F16Most;
  if constexpr (SHIFT) {                                // over the workgroup's rows
    if (tid == 0) key_limit = kBank4F16Most;
    __syncthreads();
    if (lost != 0.f) atomicMin(&key_limit, key_byte_limit(lost, scale));
    __syncthreads();
    key_most = __builtin_amdgcn_readfirstlane(key_limit);
  }
  f32x16 o[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
  float m = -INFINITY, l = 0.f;
  const int v_row = a.value_dim / 2, vs_row = a.value_dim / 32;
  const uint8_t *kc = a.kc + (int64_t)bh * a.slots * (DK / 2), *ks = a.ks + (int64_t)bh * a.slots * (DK / 32);
  const uint8_t *vc = a.vc + (int64_t)bh * a.slots * v_row + chunk * (DVC / 2), *vs = a.vs + (int64_t)bh * a.slots * vs_row + chunk * VB;
  KeyRow<DK> ka[2], kb[2];
  u32x4 vn[VL];
  uint32_t vsn[VL];

  auto load_keys = [&](KeyRow<DK> *to, int base) {
    const int64_t n = s1 - base, at = base;
    const auto rk = bank_rows(kc + at * (DK / 2), n * (DK / 2)), rs = bank_rows(ks + at * (DK / 32), n * (DK / 32));
    to[0].load(rk, rs, 0, col, half);
    to[1].load(rk, rs, 32, col, half);
  };
  auto load_values = [&](int base) {
    const int64_t n = s1 - base, at = base;
    const auto rv = bank_rows(vc + at * v_row, n * v_row - chunk * (DVC / 2)), rw = bank_rows(vs + at * vs_row, n * vs_row - chunk * VB);
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      if (VE < 256 && tid >= VE) break;
      vn[i] = __builtin_amdgcn_raw_buffer_load_b128(rv, tid / VB * v_row + tid % VB * 16, i * (256 / VB) * v_row, 0);
      vsn[i] = __builtin_amdgcn_raw_buffer_load_b8(rw, tid / VB * vs_row + tid % VB, i * (256 / VB) * vs_row, 0);
    }
  };
  bool outside = false;                                // F16: a block that fp16 does not hold
  u16x2 k_most = {0, 0};                               // and, of keys that stay bf16, their largest scale bytes
  auto store_values = [&](int buf) {
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int e = i * 256 + tid, vr = e / VB, blk = e % VB;
      if (VE < 256 && e >= VE) {
        if (CAUSAL) nan_blocks[buf][wave][i] = 0;
        break;
      }
      float sc = bank4_scale(vsn[i]);
      if (F16) outside |= !bank4_fits_f16(vsn[i], vn[i]);
      if (CAUSAL) {
        nan_blocks[buf][wave][i] = __ballot(vsn[i] == kBank4NanScale);
        sc = vsn[i] == kBank4NanScale ? 1.f : sc;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<V8 *>(vt + (buf * 64 + vr) * VS + blk * 32 + j * 8) = unpack8<V8>(vn[i][j], sc);
    }
  };
  // Causal: a value block that stands for NaN makes it NaN for the rows that see its slot and is finite for the others, whose weight there is 0.
  auto add_nans = [&](int buf, int base) {
    uint64_t any = 0;
#pragma unroll
    for (int i = 0; i < 4 * VL; ++i) any |= nan_blocks[buf][i / VL][i % VL];
    if (!any) return;
    for (int i = 0; i < 4 * VL; ++i) {
      for (uint64_t bad = nan_blocks[buf][i / VL][i % VL]; bad; bad &= bad - 1) {
        const int e = i % VL * 256 + i / VL * 64 + __builtin_ctzll(bad);
        const float add = base + e / VB < limit ? NAN : 0.f;
#pragma unroll
        for (int c = 0; c < NT; ++c)
          if (c == e % VB) o[c] += add;
      }
    }
  };

  // The logits run one step ahead: their products are issued among the exponentials of the step before, their maximum among its second
  // products.  The order inside a step is the compiler's: written out by hand, one product and at most four vector instructions behind it, the
  // step takes a tenth fewer cycles and the chip holds a tenth less clock (fp32 on bf16 numbers: 57 % of the cycles matrix work at 1.78 GHz,
  // against 46 % at 2.05; fp16 numbers: 43 % at 1.77): power is what bounds this kernel, as it bounds a large library product (1.2 of the 2.5 PFLOP/s).
  float top;
  auto row_top = [&](const f32x16 (&x)[2]) {
    float t = fmaxf(x[0][0], x[1][0]);
#pragma unroll
    for (int j = 1; j < 16; ++j) t = fmaxf(fmaxf(t, x[0][j]), x[1][j]);
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(t), __float_as_uint(t), false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * scale;
  };
  auto settle = [&](f32x16 (&x)[2], int base) {      // masks the logits of a step that not all rows see, moves the maximum if it has to
    if (base + 64 > low || base + 64 > s1) {
      const int lim = limit < s1 ? limit : s1;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < 16; ++j) x[s][j] = base + s * 32 + mfma32_row(j, lane) < lim ? x[s][j] : -INFINITY;
      top = row_top(x);
    }
    if (__any(top > m + LAG)) {
      const float mn = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i] *= alpha;
    }
  };
  auto step = [&](f32x16 (&x)[2], f32x16 (&xn)[2], const KeyRow<DK> (&k)[2], KeyRow<DK> (&kn)[2], int base, int buf) {
    if (CAUSAL) add_nans(buf, base);
    load_values(base + 64);                  // (behind the slice: nothing is read, zeros come back)
    load_keys(kn, base + 128);
    const float mu = m == -INFINITY ? 0.f : m - P_UP;
    if (KEYS_F16 && wave == 0) outside |= !k[0].fits_f16(key_most) || !k[1].fits_f16(key_most);      // (all waves hold the same keys)
    if (F16 && !KEYS_F16) { k[0].most(k_most); k[1].most(k_most); }
    xn[0] = q.dot(k[0]);
    xn[1] = q.dot(k[1]);
    V8 pf[4][PP];
#pragma unroll
    for (int s = 0; s < 4; ++s) {           // 16 slots: keys 16 s + {0..3, 8..11} + 4 half
      f32x8 p;
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[s / 2][(s & 1) * 8 + j], scale, -mu));
      split8<PP>(p, pf[s]);
#pragma unroll
      for (int j = 0; j < 8; ++j) l += p[j];
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const __bf16 *at = vt + (buf * 64 + s * 16 + half * 4 + (lane & 15) / 4) * VS + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + i * 32));
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + i * 32 + 8 * VS));
        const V8 vf = __builtin_bit_cast(V8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int w = 0; w < PP; ++w) o[i] = mfma32(vf, pf[s][w], o[i]);
      }
    }
    top = row_top(xn);
    store_values(buf ^ 1);
    __syncthreads();
    settle(xn, base + 64);
  };
  f32x16 xa[2], xb[2];
  if (s0 < s1) {
    load_keys(ka, s0);
    load_values(s0);
    if (KEYS_F16 && wave == 0) outside |= !ka[0].fits_f16(key_most) || !ka[1].fits_f16(key_most);
    if (F16 && !KEYS_F16) { ka[0].most(k_most); ka[1].most(k_most); }
    xa[0] = q.dot(ka[0]);
    xa[1] = q.dot(ka[1]);
    load_keys(ka, s0 + 64);
    store_values(0);
    top = row_top(xa);
    settle(xa, s0);
  }
  __syncthreads();
  for (int base = s0; base < s1; base += 128) {
    step(xa, xb, ka, kb, base, 0);
    if (base + 64 >= s1) break;
    step(xb, xa, kb, ka, base + 64, 1);
  }
  l += __shfl_xor(l, 32);
  m -= P_UP;
  if constexpr (F16) {
    if (!KEYS_F16) outside |= k_most[0] > kBank4F16Most || k_most[1] > kBank4F16Most;
    again = __syncthreads_or(outside);
  }
  if (r < a.rows && !again) {
    const float inv = live && l != 0.f ? 1.f / l : 0.f;
    if (a.part_o) {
      const int64_t at = ((int64_t)bh * a.nsplit + split) * a.rows + r;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f32x4 *>(a.part_o + at * a.value_dim + chunk * DVC + i * 32 + j * 8 + half * 4) =
              inv == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : f32x4{o[i][4 * j] * inv, o[i][4 * j + 1] * inv, o[i][4 * j + 2] * inv, o[i][4 * j + 3] * inv};
      if (half == 0 && chunk == 0) *reinterpret_cast<f32x2 *>(a.part_ml + at * 2) = live ? f32x2{m, l} : f32x2{-INFINITY, 0.f};
    } else {
      T *out = (T *)a.out + (((int64_t)b * a.tokens + t) * a.heads * a.group + h * a.group + r - t * a.group) * a.value_dim + chunk * DVC;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          typedef T Tx4 __attribute__((ext_vector_type(4)));
          Tx4 y;
#pragma unroll
          for (int c = 0; c < 4; ++c) y[c] = (T)(inv == 0.f ? 0.f : o[i][4 * j + c] * inv);
          *reinterpret_cast<Tx4 *>(out + i * 32 + j * 8 + half * 4) = y;
        }
    }
  }
