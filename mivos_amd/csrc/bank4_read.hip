// Attention over the 4-bit memory bank:  out[t, j] = sum_s softmax_s(scale * q[t, j] . k[s, j / G]) v[s, j / G],  G query heads a bank head,
// softmax over the visible slots of the stream (all of them, or causally those up to the token's own place), a row that sees nothing is 0;
// and, when asked, weight[s] += sum over the rows (tokens x G) of their softmax weight on slot s.
//
// Arithmetic.  A bank value has at most two significant bits and is exact in bf16, so both products run on the bf16 matrix cores with
// exact bank operands: q and the softmax weight p are written as sums of bf16 numbers - q in 1 for bf16 inputs (exact), 2 for fp16 (exact), 3 for
// fp32 (24 bits), p in 2, 2 and 3 (16, 16 and 24 bits).  That is what few rows take, where bytes are the cost.  Where many rows make the products the
// cost they run on fp16 numbers, one part fewer (bank4_block_kernel).
// Running maximum, sum and accumulators are fp32.
//
// Layout.  S^T = K Q^T on 16x16x32: lane l holds bank row l % 16 and channels (l / 16) * DK / 4 .. + DK / 4 of it - contiguous codes in memory,
// mostly of one scale block, so K needs no staging; Q is kept in registers in the same channel order.  The result gives a lane one query
// (column l % 16) and four keys a tile, which is the B operand of O^T = V^T P^T as it stands (the 8 keys of a lane in a pair of tiles are
// the same 8 in both operands).  V rows are widened to bf16 in a wave's own LDS patch and read back transposed (ds_read_b64_tr_b16).
#include <type_traits>

#include "bank4.h"

namespace mivos {

constexpr float LOG2E = 1.4426950408889634f;
// Rows a bank head from which the 128-row kernel runs.  Both kernels, us without / with the weights gathered (bf16; 16-row tiles | 128 rows):
//   4 heads x 16 384 slots, 2 streams   32 rows 28 / 41 | 25 / 30     64 rows 38 / 65 | 28 / 33     200 rows 60 / 155 | 41 / 53
//   2 heads x 65 536 slots              32 rows 30 / 38 | 33 / 38     64 rows 37 / 59 | 33 / 40     200 rows 63 / 171 | 46 / 58
//   8 heads x 4096 slots x 64, 4        32 rows 16 / 36 | 18 / 22     64 rows 24 / 58 | 19 / 24     200 rows 39 / 142 | 30 / 41
//   1 head x 8192 slots, values of 512  32 rows 15 / 29 | 25 / 30     64 rows 17 / 49 | 26 / 31     200 rows 33 / 127 | 30 / 40
// (fp32: 32 rows 32 | 32, 32 | 41, 18 | 24, 16 | 36; 64 rows 47 | 36, 42 | 43, 27 | 25, 19 | 38, weights 74 | 47, 65 | 52, 61 | 36, 51 | 47)
constexpr int BLOCK_ROWS_MIN = 33;

struct ReadArgs {
  const uint8_t *kc, *ks, *vc, *vs;
  float *weight;
  const int32_t *lens, *count;
  const void *q;
  void *out;
  int64_t qb, qt, qh;
  float *part_o, *part_ml, *logits, *row_max, *row_inv, *row_scale;
  uint32_t *row_limit;    // bank4_weigh: the key_byte_limit of 32 rows, at the first of them
  __bf16 *q_pack;
  _Float16 *q_pack_f16;
  int32_t *redo;          // fp16 and fp32 queries: a flag a workgroup, fp16 products met a block that they do not hold, the bf16 ones do it again
  int64_t slots, logit_stride, row_stride;
  int batch, heads, group, tokens, rows, key_dim, value_dim, nsplit, causal, q_vec;
  float scale_log2;       // |scale| * log2(e): the softmax runs in powers of two; the sign of scale goes to the queries
  float q_sign;           // (0 where scale is: -inf * 0 of a masked logit is never formed)
};

__device__ __forceinline__ int64_t read_len(const ReadArgs &a, int b) {
  const int64_t n = a.lens[b];
  return n < 0 ? 0 : n > a.slots ? a.slots : n;
}
__device__ __forceinline__ int read_count(const ReadArgs &a, int b) {
  const int n = a.count ? a.count[b] : a.tokens;
  return n < 0 ? 0 : n > a.tokens ? a.tokens : n;
}
// slots a row (token t of a stream) sees: [0, limit)
__device__ __forceinline__ int64_t read_limit(const ReadArgs &a, int64_t len, int cnt, int t) {
  if (t >= cnt) return 0;
  if (!a.causal) return len;
  const int64_t n = len - cnt + t + 1;
  return n < 0 ? 0 : n;
}

__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// x as a sum of PARTS bf16 or fp16 numbers
template <typename E, int PARTS, typename V>
__device__ __forceinline__ void split8_as(f32x8 x, V (&p)[PARTS]) {
#pragma unroll
  for (int k = 0; k < PARTS; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[k][j] = (E)x[j];
      x[j] -= (float)p[k][j];
    }
}
template <int PARTS> __device__ __forceinline__ void split8(f32x8 x, bf16x8 (&p)[PARTS]) { split8_as<__bf16>(x, p); }
template <int PARTS> __device__ __forceinline__ void split8(f32x8 x, f16x8 (&p)[PARTS]) {
  p[0] = __builtin_convertvector(x, f16x8);
  if constexpr (PARTS == 2) {
    float one = 1.f;
    asm("" : "+s"(one));               // (a factor that the compiler cannot drop: x * one - p and its rounding are one instruction, else three)
#pragma unroll
    for (int j = 0; j < 8; ++j) p[1][j] = (_Float16)__builtin_fmaf(x[j], one, -(float)p[0][j]);
  }
}

template <typename V> __device__ __forceinline__ V unpack8(uint32_t codes, float scale);
template <> __device__ __forceinline__ bf16x8 unpack8<bf16x8>(uint32_t codes, float scale) { return bank4_unpack8(codes, scale); }
template <> __device__ __forceinline__ f16x8 unpack8<f16x8>(uint32_t codes, float scale) { return bank4_unpack8_f16(codes, scale); }
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Exponent of the power of two that brings a row of fp32 queries with the largest magnitude `top` to [2^13, 2^14) (rows below 2^-87: less far up)
__device__ __forceinline__ int query_shift(float top) {
  const int t = 13 + 127 - (int)(__float_as_uint(top) >> 23);
  return t > 100 ? 100 : t < -114 ? -114 : t;
}
// what brings such a row's products to powers of two of a softmax weight; never 0 (a masked logit is -inf) nor infinite (a product may be 0):
// where it is held back the products of fp16 blocks are far below 1 or far past every weight all the same
__device__ __forceinline__ float row_scale(float scale_log2, float back) { return fminf(fmaxf(scale_log2 * back, 0x1p-126f), 0x1.fffffep127f); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 .. 127

// A row's channels as two fp16 numbers each: 2^-22 of the channel, but below 2^-3 (2^-16 of the row's largest) half of 2^-24.  What that leaves out
// beyond 2^-22 of a channel, summed over the row, bounds the error of its logits by the keys they meet; keys that could take it past 2^-22 are for
// bf16 numbers: the largest scale byte that may stay (normal rows against normal keys of 128 channels reach that at 2^16 times their size).
__device__ __forceinline__ float left_out(f32x8 x, const f16x8 (&p)[2]) {
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float r = __builtin_fabsf((x[j] - (float)p[0][j]) - (float)p[1][j]);
    sum += r > 0x1p-22f * __builtin_fabsf(x[j]) ? r : 0.f;
  }
  return sum;
}
__device__ __forceinline__ uint32_t key_byte_limit(float lost, float scale) {
  const uint32_t byte = __float_as_uint(0x1p-22f / 6.f / (lost * scale)) >> 23;       // 6 * 2^(byte - 127) * lost * scale <= 2^-22; nothing lost: 255
  return byte < kBank4F16Most ? byte : kBank4F16Most;
}

template <int PARTS> struct ReadType;
template <> struct ReadType<1> { typedef __bf16 T; };
template <> struct ReadType<2> { typedef _Float16 T; };
template <> struct ReadType<3> { typedef float T; };

typedef __attribute__((address_space(3))) s16x4 *lds_s16x4;
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// Rows [0, n) of a bank array behind a wave-uniform address: loads take one per-lane offset and answer 0 behind the last row (codes 0, scale
// byte 0: the value 0), so that what lies behind a stream's length is neither addressed nor looked at.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t bank_rows(const uint8_t *p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, (int)(bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : bytes), 0x00020000);
}

constexpr int block_occupancy(int dk, int dvc, int parts) { return parts == 1 && dk <= 128 && dvc <= 128 ? 2 : 1; }
inline int query_parts(int dtype) { return dtype == MIVOS_BF16 ? 1 : dtype == MIVOS_F16 ? 2 : 3; }
constexpr float MAX_LAG = 8.f;      // the running maximum follows a logit that passes it by more than this (powers of two): fewer rescales

// ------------------------------------------------------------------------------------------ few rows: 16 a workgroup
// One workgroup: 16 rows x one slice of the slots x DVC value channels; its four waves take 64 slots in turn, each with a running
// softmax of its own, and meet in LDS at the end.  A step's codes and scales are fetched a step ahead, 64 slots x (DK + DVC) * 17 / 32 bytes a wave.
// (The block-scaled 4 x 8-bit products would take the codes as they are and the query in two 8-bit floats a channel, but they line up a
// product's terms in a window of about 13 bits: logits off by 2^-12, weights by 0.2 %.  They are not used.)
template <int DK, int DVC, int PARTS>
__global__ __launch_bounds__(256, PARTS == 1 && DK <= 128 ? 3 : 2) void bank4_rows_kernel(ReadArgs a) {
  typedef typename ReadType<PARTS>::T T;
  constexpr int PP = PARTS == 3 ? 3 : 2;
  constexpr int CPL = DK / 4, KSTEPS = DK / 32, VPAD = DVC + 16, OPAD = DVC + 4, NT = DVC / 16, VB = DVC / 32;
  constexpr int LDS_V = 4 * 32 * VPAD * 2, LDS_O = 4 * 16 * OPAD * 4;
  __shared__ __align__(16) char lds[LDS_V > LDS_O ? LDS_V : LDS_O];
  __shared__ float stat[4][16][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, grp = lane >> 4;
  const int nvc = a.value_dim / DVC, chunk = blockIdx.z % nvc, bh = blockIdx.z / nvc, b = bh / a.heads, h = bh - b * a.heads;
  const int split = blockIdx.x, row0 = blockIdx.y * 16;
  const int len = (int)read_len(a, b), cnt = read_count(a, b);
  const int r = row0 + col, t = r / a.group;
  const bool live = r < a.rows && t < cnt;
  const int limit = live ? (int)read_limit(a, len, cnt, t) : 0;
  int last_t = (row0 + 15 < a.rows ? row0 + 15 : a.rows - 1) / a.group;
  last_t = last_t < cnt ? last_t : cnt - 1;
  const int seen = row0 / a.group < cnt ? (int)read_limit(a, len, cnt, last_t) : 0;   // slots any row of the tile sees
  const int per = ((seen + 63) / 64 + a.nsplit - 1) / a.nsplit * 64;
  const int s0 = (int64_t)split * per < seen ? split * per : seen, s1 = seen - s0 < per ? seen : s0 + per;
  int low = live ? limit : seen;                                                      // slots all rows see
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    const int x = __shfl_xor(low, d);
    low = x < low ? x : low;
  }
  low = __builtin_amdgcn_readfirstlane(low);

  bf16x8 qf[KSTEPS][PARTS];
  const T *qrow = (const T *)a.q + b * a.qb + (int64_t)(live ? t : 0) * a.qt + (int64_t)(h * a.group + (live ? r - t * a.group : 0)) * a.qh;
#pragma unroll
  for (int i = 0; i < KSTEPS; ++i) {
    f32x8 x = load8(qrow + grp * CPL + i * 8, a.q_vec);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = live ? x[j] * a.q_sign : 0.f;
    split8<PARTS>(x, qf[i]);
  }
  f32x4 o[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  __bf16 *vt = reinterpret_cast<__bf16 *>(lds) + wave * 32 * VPAD;
  const int v_row = a.value_dim / 2, vs_row = a.value_dim / 32;
  const uint8_t *kc = a.kc + (int64_t)bh * a.slots * (DK / 2), *ks = a.ks + (int64_t)bh * a.slots * (DK / 32);
  const uint8_t *vc = a.vc + (int64_t)bh * a.slots * v_row + chunk * (DVC / 2), *vs = a.vs + (int64_t)bh * a.slots * vs_row + chunk * VB;
  const int k_at = col * (DK / 2) + grp * (CPL / 2), ks_at = col * (DK / 32) + grp * CPL / 32;
  const int v_at = lane / VB * v_row + lane % VB * 16, vs_at = lane / VB * vs_row + lane % VB;

  struct Step {
    uint32_t kc[4][KSTEPS], ks[4];
    u32x4 vc[VB];
    uint32_t vs[VB];
  } now, next;
  auto fetch = [&](Step &f, int base) {
    const int64_t n = s1 - base, at = base;
    const auto rk = bank_rows(kc + at * (DK / 2), n * (DK / 2)), rs = bank_rows(ks + at * (DK / 32), n * (DK / 32));
    const auto rv = bank_rows(vc + at * v_row, n * v_row - chunk * (DVC / 2)), rw = bank_rows(vs + at * vs_row, n * vs_row - chunk * VB);
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      if constexpr (KSTEPS == 2) *reinterpret_cast<u32x2 *>(f.kc[kt]) = __builtin_amdgcn_raw_buffer_load_b64(rk, k_at + kt * 8 * DK, 0, 0);
      else
#pragma unroll
        for (int i = 0; i < KSTEPS / 4; ++i)
          *reinterpret_cast<u32x4 *>(f.kc[kt] + 4 * i) = __builtin_amdgcn_raw_buffer_load_b128(rk, k_at + kt * 8 * DK + i * 16, 0, 0);
      if constexpr (KSTEPS == 8) f.ks[kt] = __builtin_amdgcn_raw_buffer_load_b16(rs, ks_at + kt * (DK / 2), 0, 0);
      else f.ks[kt] = __builtin_amdgcn_raw_buffer_load_b8(rs, ks_at + kt * (DK / 2), 0, 0);
    }
#pragma unroll
    for (int i = 0; i < VB; ++i) {       // 64 rows x VB blocks of 16 bytes over 64 lanes
      f.vc[i] = __builtin_amdgcn_raw_buffer_load_b128(rv, v_at, i * (64 / VB) * v_row, 0);
      f.vs[i] = __builtin_amdgcn_raw_buffer_load_b8(rw, vs_at, i * (64 / VB) * vs_row, 0);
    }
  };
  if (s0 + wave * 64 < s1) fetch(next, s0 + wave * 64);
  for (int base = s0 + wave * 64; base < s1; base += 256) {
    now = next;
    if (base + 256 < s1) fetch(next, base + 256);
    // ---- logits of 64 slots
    f32x4 x[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      x[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KSTEPS; ++i) {
        const bf16x8 kf = bank4_unpack8(now.kc[kt][i], bank4_scale(KSTEPS == 8 ? (now.ks[kt] >> (i / 4 * 8)) & 255 : now.ks[kt]));
#pragma unroll
        for (int p = 0; p < PARTS; ++p) x[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[i][p], x[kt], 0, 0, 0);
      }
    }
    if (base + 64 > low || base + 64 > s1) {
      const int lim = limit < s1 ? limit : s1;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[kt][j] = base + kt * 16 + grp * 4 + j < lim ? x[kt][j] : -INFINITY;
    }
    if (a.logits && chunk == 0 && r < a.rows)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
        *reinterpret_cast<f32x4 *>(a.logits + ((int64_t)bh * a.rows + r) * a.logit_stride + base + kt * 16 + grp * 4) = x[kt];
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) top = fmaxf(top, fmaxf(fmaxf(x[kt][0], x[kt][1]), fmaxf(x[kt][2], x[kt][3])));
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32)) * a.scale_log2;
    if (__any(top > m + MAX_LAG)) {
      const float mn = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i] *= alpha;
    }
    const float mu = m == -INFINITY ? 0.f : m;
    if (a.causal) {        // a value block that stands for NaN makes it NaN for the rows that see its slot, and is 0 for the others (0 x NaN is none)
#pragma unroll
      for (int i = 0; i < VB; ++i) {
        uint64_t bad = __ballot(now.vs[i] == kBank4NanScale);
        if (now.vs[i] == kBank4NanScale) { now.vs[i] = 127; now.vc[i] = u32x4{0u, 0u, 0u, 0u}; }
        for (; bad; bad &= bad - 1) {
          const int e = i * 64 + __builtin_ctzll(bad);
          const float add = base + e / VB < limit ? NAN : 0.f;
#pragma unroll
          for (int c = 0; c < VB; ++c)
            if (c == e % VB) { o[2 * c] += add; o[2 * c + 1] += add; }
        }
      }
    }
    // ---- V in two halves of 32 slots
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      f32x8 p;
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[half * 2 + j / 4][j % 4], a.scale_log2, -mu));
      bf16x8 pf[PP];
      split8<PP>(p, pf);
#pragma unroll
      for (int j = 0; j < 8; ++j) l += p[j];
      wave_lds_fence();
#pragma unroll
      for (int i = 0; i < VB / 2; ++i) {
        const int e = i * 64 + lane, vr = e / VB, blk = e % VB;
        const float sc = bank4_scale(now.vs[half * (VB / 2) + i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<bf16x8 *>(vt + vr * VPAD + blk * 32 + j * 8) = bank4_unpack8(now.vc[half * (VB / 2) + i][j], sc);
      }
      wave_lds_fence();
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const __bf16 *at = vt + (grp * 4 + col / 4) * VPAD + i * 16 + (col % 4) * 4;
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at));
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 16 * VPAD));
        const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int q = 0; q < PP; ++q) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[q], o[i], 0, 0, 0);
      }
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  // ---- the four waves meet
  __syncthreads();
  float *om = reinterpret_cast<float *>(lds);
#pragma unroll
  for (int i = 0; i < NT; ++i) *reinterpret_cast<f32x4 *>(om + (wave * 16 + col) * OPAD + i * 16 + grp * 4) = o[i];
  if (grp == 0) { stat[wave][col][0] = m; stat[wave][col][1] = l; }
  __syncthreads();
  for (int e = tid; e < 16 * DVC; e += 256) {
    const int rr = e / DVC, dv = e % DVC, row = row0 + rr;
    if (row >= a.rows) break;
    const int tt = row / a.group;
    const bool valid = tt < cnt;      // (a padded token's queries are zeros, its logits only masked where a valid row's are)
    const float mm = fmaxf(fmaxf(stat[0][rr][0], stat[1][rr][0]), fmaxf(stat[2][rr][0], stat[3][rr][0]));
    const float mu = mm == -INFINITY ? 0.f : mm;
    float acc = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(stat[w][rr][0] - mu);
      acc += f * om[(w * 16 + rr) * OPAD + dv];
      sum += f * stat[w][rr][1];
    }
    if (a.part_o) {
      const int64_t at = ((int64_t)bh * a.nsplit + split) * a.rows + row;
      a.part_o[at * a.value_dim + chunk * DVC + dv] = valid && sum != 0.f ? acc / sum : 0.f;
      if (dv == 0 && chunk == 0) *reinterpret_cast<f32x2 *>(a.part_ml + at * 2) = valid ? f32x2{mm, sum} : f32x2{-INFINITY, 0.f};
    } else {
      const int j = h * a.group + row - tt * a.group;
      ((T *)a.out)[(((int64_t)b * a.tokens + tt) * a.heads * a.group + j) * a.value_dim + chunk * DVC + dv] = (T)(valid && sum != 0.f ? acc / sum : 0.f);
    }
  }
}

// ------------------------------------------------------------------------------------------ many rows: 128 a workgroup
// K rows of a tile in a lane's registers: 32x32 products take row l % 32, channels i * 64 + (l / 32) * 32 .. + 31 of it.
template <int DK>
struct KeyRow {
  static constexpr int KI = DK / 64;
  u32x4 codes[KI];
  uint32_t scales[(KI + 1) / 2];        // byte 2 (i % 2) of word i / 2: the scale of the lane's block i
  // row `col` + `row` of the arrays behind rk / rs
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rk, __amdgpu_buffer_rsrc_t rs, int row, int col, int half) {
#pragma unroll
    for (int i = 0; i < KI; ++i) codes[i] = __builtin_amdgcn_raw_buffer_load_b128(rk, col * (DK / 2) + half * 16, row * (DK / 2) + i * 32, 0);
    if constexpr (KI == 1) scales[0] = __builtin_amdgcn_raw_buffer_load_b8(rs, col * 2 + half, row * 2, 0);
    else
#pragma unroll
      for (int i = 0; i < KI / 2; ++i) scales[i] = __builtin_amdgcn_raw_buffer_load_b32(rs, col * (DK / 32), row * (DK / 32) + i * 4, 0) >> (8 * half);
  }
  __device__ __forceinline__ uint32_t byte(int i) const { return (scales[i / 2] >> (16 * (i & 1))) & 255; }
  __device__ __forceinline__ float scale(int i) const { return bank4_scale(byte(i)); }
  __device__ __forceinline__ void most(u16x2 &m) const {      // the largest scale bytes of words' halves
#pragma unroll
    for (int i = 0; i < (KI + 1) / 2; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, scales[i] & 0x00ff00ffu));
  }
  __device__ __forceinline__ bool fits_f16(uint32_t most = kBank4F16Most) const {
    bool ok = true;
#pragma unroll
    for (int i = 0; i < KI; ++i) ok &= bank4_fits_f16(byte(i), codes[i], most);
    return ok;
  }
};

// Queries of a lane (column l % 32), in the channel order of KeyRow.
template <int DK, int PARTS, typename V>
struct QueryCols {
  V f[DK / 16][PARTS];
  // SHIFT: the row times 2^t, t its query_shift -> 2^-t; lost: left_out of it
  template <bool SHIFT, typename T>
  __device__ __forceinline__ float load(const T *row, int half, bool live, bool vec, float sign, float &lost) {
    auto channels = [&](int i) {
      f32x8 x = load8(row + i / 4 * 64 + half * 32 + i % 4 * 8, vec);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = live ? x[j] * sign : 0.f;
      return x;
    };
    float up = 1.f, back = 1.f;
    if constexpr (SHIFT) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < DK / 16; ++i) {
        const f32x8 x = channels(i);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, __builtin_fabsf(x[j]));
      }
      const int t = query_shift(fmaxf(top, __shfl_xor(top, 32)));
      up = pow2(t);
      back = pow2(-t);
    }
#pragma unroll
    for (int i = 0; i < DK / 16; ++i) {
      const f32x8 x = SHIFT ? channels(i) * up : channels(i);
      split8<PARTS>(x, f[i]);
      if constexpr (SHIFT) lost += left_out(x, f[i]);
    }
    if (SHIFT) lost += __shfl_xor(lost, 32);
    return back;
  }
  __device__ __forceinline__ f32x16 dot(const KeyRow<DK> &k) const {       // [32 keys][32 queries]
    f32x16 c;
#pragma unroll
    for (int r = 0; r < 16; ++r) c[r] = 0.f;
#pragma unroll
    for (int i = 0; i < DK / 64; ++i) {
      const float sc = k.scale(i);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const V kf = unpack8<V>(k.codes[i][u], sc);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) c = mfma32(kf, f[i * 4 + u][p], c);
      }
    }
    return c;
  }
};

// One workgroup: 128 rows (32 a wave) x one slice of the slots x DVC value channels, 64 slots a step.  Every wave reads the step's K
// codes straight into registers; the V rows are widened once for the workgroup into one of two LDS buffers while the matrix cores work on
// the other.  S^T = K Q^T and O^T = V^T P^T on 32x32 products: a lane holds one query, 16 keys of each 32, and these are again the
// operand of the second product.  The running maximum is moved (and the accumulators rescaled) only when a logit passes it by 2^LAG.
// F16: the products on fp16 numbers, which carry three bits more than bf16 ones.  fp16 and fp32 queries: q in 1 / 2 of them (fp32 rows brought to
// 2^14 first), the softmax weight times 2^12 in 2 (2^-22 of itself or 2^-37 of the row's largest; the maximum is followed closer, by 2^3).  bf16
// queries: keys and q as bf16, the weight times 2^8 in 1 (2^-11 of itself or 2^-33 of the row's largest).  One bf16 number, 2^-8 of the weight, put
// the error of 3 x 1021 causal tokens over 16 300 slots at 1.3 times that of fp32 weights, two take 489 us there: 359, 372 and 489.
// A 4-bit value is exact in fp16 from 2^-24 to 6 * 2^13.  A workgroup that has met a block outside (of keys under bf16 queries: above, where logits may
// lie so far apart that such weights lose channels), or an fp32 row that loses channels to its keys (key_byte_limit), does its work again on
// bf16 numbers: where all do, 1000 tokens, 4 over 2 heads, 16 384 slots take 99 us instead of 59 (bf16) and 165 instead of 85 (fp32).
// 2 x 1620 fp32 rows x 32 400 slots, 128 / 512: 400 us instead of 471 on bf16 numbers alone, 0.81 PFLOP/s issued; all 512 value channels in one
// workgroup would need registers it does not have.
// F16: `again` says that the workgroup has met such a block or row; then it has written nothing.
// (The body is in bank4_block.h, once as a kernel's own text and once as a function's: in a function that a kernel calls, the compiler orders a step
// otherwise, and 3 x 1021 causal fp32 tokens over 16 300 slots take 860 us instead of 800.)
// fp16 and fp32 queries: F16 raises the workgroup's flag, and the bf16 kernel is launched behind (5 us where no flag is up).
template <int DK, int DVC, int PARTS, bool F16, bool CAUSAL>
__global__ __launch_bounds__(256, block_occupancy(DK, DVC, PARTS)) void bank4_block_kernel(ReadArgs a) {
  int32_t *redo = a.redo + (blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
  if (!F16 && !*redo) return;
  bool again = false;
#include "bank4_block.h"
  if (F16 && threadIdx.x == 0) *redo = again;
}

// bf16 queries: both in one launch (a second one is 2 us of a call over few slots).
template <int DK, int DVC, bool F16, bool CAUSAL>
__device__ __forceinline__ bool block_rows_bf16(const ReadArgs &a) {
  constexpr int PARTS = 1;
  bool again = false;
#include "bank4_block.h"
  return again;
}
template <int DK, int DVC, bool CAUSAL>
__global__ __launch_bounds__(256, block_occupancy(DK, DVC, 1)) void bank4_block_bf16_kernel(ReadArgs a) {
  if (block_rows_bf16<DK, DVC, true, CAUSAL>(a)) block_rows_bf16<DK, DVC, false, CAUSAL>(a);
}

// weight[s] += sum over the rows of exp2(logit - maximum) / sum, each row's maximum and 1 / sum from bank4_join (one number, their logarithm
// together, would cost every weight of a row 2^-24 of it): the logits once more, now S = Q K^T, so that a lane holds one slot and its sum
// runs over registers, the rows in order.  One workgroup: 128 * NS slots, NS x 32 a wave, their keys widened once into registers; 32 rows a
// step go through LDS, copied as bank4_join has packed them in operand order.  (A wave that reads its rows as they lie in memory touches a
// cache line a lane and load, and with 64 slots a workgroup the queries cross the L2 1.3 GB at 1620 x 32 400 x 2: 150 and 115 us.)
// fp16 products (V8 = f16x8) and their flags as in bank4_block_kernel; SHIFT: fp32 rows were packed times a power of two of their own.
template <int DK, int PARTS, int NS, typename V8, bool SHIFT>
__global__ __launch_bounds__(256) void bank4_weigh_kernel(ReadArgs a) {
  constexpr bool F16 = std::is_same_v<V8, f16x8>;
  constexpr int KS = DK / 16, TILE = KS * PARTS * 64, TL = TILE / 256;       // 16-byte words a tile, a thread
  extern __shared__ __align__(16) u32x4 qs[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int bh = blockIdx.y, b = bh / a.heads, first = blockIdx.x * (128 * NS), base = first + wave * (32 * NS);
  const int len = (int)read_len(a, b), cnt = read_count(a, b);
  const int rows = cnt * a.group;                       // (rows behind the count have no weight)
  if (first >= len || rows == 0) return;
  int32_t *redo = a.redo + blockIdx.y * gridDim.x + blockIdx.x;
  if (!F16 && PARTS > 1 && !*redo) return;            // (bf16 queries: these products alone)
  const int64_t row_base = (int64_t)bh * a.slots;
  const auto rk = bank_rows(a.kc + (row_base + base) * (DK / 2), (int64_t)(len - base) * (DK / 2));
  const auto rs = bank_rows(a.ks + (row_base + base) * (DK / 32), (int64_t)(len - base) * (DK / 32));
  V8 kf[NS][KS];
  bool outside = false;
  uint32_t key_byte = 0;                                // SHIFT: the largest scale byte of the lane's blocks that are not zeros
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    KeyRow<DK> k;
    k.load(rk, rs, s * 32, col, half);
    if (F16) outside |= !k.fits_f16();
    if (SHIFT)
#pragma unroll
      for (int i = 0; i < DK / 64; ++i)
        if (!bank4_zeros(k.codes[i]) && k.byte(i) > key_byte) key_byte = k.byte(i);
#pragma unroll
    for (int i = 0; i < DK / 64; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) kf[s][i * 4 + u] = unpack8<V8>(k.codes[i][u], k.scale(i));
  }
  if constexpr (SHIFT) {
    __shared__ uint32_t key_limit;
    if (tid == 0) key_limit = kBank4F16Most;
    __syncthreads();
    for (int i = tid * 32; i < rows; i += 256 * 32) {
      const uint32_t limit = a.row_limit[(int64_t)bh * a.row_stride + i];
      if (limit < kBank4F16Most) atomicMin(&key_limit, limit);
    }
    __syncthreads();
    outside |= key_byte > key_limit;
  }
  if constexpr (F16) {
    const int any = __syncthreads_or(outside);
    if (tid == 0) *redo = any;
    if (any) return;
  }
  float acc[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) acc[s] = 0.f;
  const u32x4 *q = (F16 ? reinterpret_cast<const u32x4 *>(a.q_pack_f16) : reinterpret_cast<const u32x4 *>(a.q_pack)) + (int64_t)bh * (a.row_stride / 32) * TILE + tid;
  const int64_t row_at = (int64_t)bh * a.row_stride + half * 4;
  const float *row_max = a.row_max + row_at, *row_inv = a.row_inv + row_at, *row_factor = a.row_scale + row_at;      // (rows behind the last hold anything: not added)
  const int tiles = (rows + 31) / 32;
  int tile0 = 0;                                        // causal: the first rows that see the workgroup's first slot
  if (a.causal) {
    const int64_t t0 = (int64_t)first - len + cnt;      // token t sees slots < len - cnt + t + 1
    tile0 = t0 > 0 ? (int)(t0 * a.group / 32) : 0;
  }
  u32x4 next[TL];
#pragma unroll
  for (int i = 0; i < TL; ++i) qs[i * 256 + tid] = q[(int64_t)tile0 * TILE + i * 256];
  __syncthreads();
  for (int tile = tile0, buf = 0; tile < tiles; ++tile, buf ^= 1) {
    const int more = tile + 1 < tiles ? tile + 1 : tile;
#pragma unroll
    for (int i = 0; i < TL; ++i) next[i] = q[(int64_t)more * TILE + i * 256];
    const int r0 = tile * 32;
    f32x4 shift[4], inv[4], scale[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      shift[g] = *reinterpret_cast<const f32x4 *>(row_max + r0 + g * 8);
      inv[g] = *reinterpret_cast<const f32x4 *>(row_inv + r0 + g * 8);
      scale[g] = f32x4{a.scale_log2, a.scale_log2, a.scale_log2, a.scale_log2};
      if constexpr (SHIFT) scale[g] = *reinterpret_cast<const f32x4 *>(row_factor + r0 + g * 8);
    }
    f32x16 x[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int j = 0; j < 16; ++j) x[s][j] = 0.f;
    const V8 *qt = reinterpret_cast<const V8 *>(qs) + buf * TILE + lane;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const V8 qf = qt[(i * PARTS + p) * 64];
#pragma unroll
        for (int s = 0; s < NS; ++s) x[s] = mfma32(qf, kf[s][i], x[s]);
      }
    if (r0 + 32 > rows || (a.causal && read_limit(a, len, cnt, r0 / a.group) < base + 32 * NS)) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int row = r0 + mfma32_row(j, lane), lim = row < rows ? (int)read_limit(a, len, cnt, row / a.group) : 0;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const float p = inv[j / 4][j % 4] * __builtin_amdgcn_exp2f(__builtin_fmaf(x[s][j], scale[j / 4][j % 4], -shift[j / 4][j % 4]));
          acc[s] += base + s * 32 + col < lim ? p : 0.f;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int s = 0; s < NS; ++s)
          acc[s] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(x[s][j], scale[j / 4][j % 4], -shift[j / 4][j % 4])), inv[j / 4][j % 4], acc[s]);
    }
#pragma unroll
    for (int i = 0; i < TL; ++i) qs[(buf ^ 1) * TILE + i * 256 + tid] = next[i];
    __syncthreads();
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    acc[s] += __shfl_xor(acc[s], 32);
    const int slot = base + s * 32 + col;
    if (half == 0 && slot < len) a.weight[row_base + slot] += acc[s];
  }
}

// A row's slices: lane s holds slice s (and s + 64).  Gives every lane the row's maximum, 1 / sum of the weights, and the shares of its slices in that
// sum.  A slice's partial output is divided by its own sum already: the maximum that this sum is taken against differs between the
// workgroups of a row's value channels where some run on fp16 numbers and some on bf16 ones, and only the first leaves its maximum and sum here.
struct RowJoin {
  float f[2], inv, top;
  __device__ __forceinline__ RowJoin(const ReadArgs &a, int bh, int row, int lane) {
    const float *ml = a.part_ml + ((int64_t)bh * a.nsplit * a.rows + row) * 2;
    float m[2], l[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int s = lane + 64 * k;
      const f32x2 v = s < a.nsplit ? *reinterpret_cast<const f32x2 *>(ml + (int64_t)s * a.rows * 2) : f32x2{-INFINITY, 0.f};
      m[k] = v.x;
      l[k] = v.y;
    }
    float mm = fmaxf(m[0], m[1]);
    for (int d = 1; d < 64; d <<= 1) mm = fmaxf(mm, __shfl_xor(mm, d));
    const float mu = mm == -INFINITY ? 0.f : mm;
    f[0] = __builtin_amdgcn_exp2f(m[0] - mu) * l[0];
    f[1] = __builtin_amdgcn_exp2f(m[1] - mu) * l[1];
    float sum = f[0] + f[1];
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    inv = sum != 0.f ? 1.f / sum : 0.f;
    top = mu;
  }
};

// Joins the slices of a row (first `out_blocks` workgroups, a wave a row and 4 * QL value channels, 64 / QL slices at a time)
// and adds the rows' weights to the slots (the others, 1024 slots each, the rows in order: the sum does not depend on timing) or, ahead of
// bank4_weigh, packs its queries.
template <int PARTS, int QL>
__global__ __launch_bounds__(256) void bank4_join_kernel(ReadArgs a, int out_blocks) {
  typedef typename ReadType<PARTS>::T T;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if ((int)blockIdx.x < out_blocks) {
    const int64_t g = (int64_t)blockIdx.x * 4 + wave;
    const int chunks = (a.value_dim + QL * 4 - 1) / (QL * 4);
    const int64_t gr = g / chunks;
    const int chunk = (int)(g - gr * chunks);
    if (gr >= (int64_t)a.batch * a.heads * a.rows) return;
    const int bh = (int)(gr / a.rows), row = (int)(gr - (int64_t)bh * a.rows), b = bh / a.heads, h = bh - b * a.heads;
    const RowJoin J(a, bh, row, lane);
    if (a.row_max && chunk == 0 && lane == 0) { a.row_max[(int64_t)bh * a.row_stride + row] = J.top; a.row_inv[(int64_t)bh * a.row_stride + row] = J.inv; }
    const int t = row / a.group, j = h * a.group + row - t * a.group;
    T *out = (T *)a.out + (((int64_t)b * a.tokens + t) * a.heads * a.group + j) * a.value_dim;
    const float *part = a.part_o + ((int64_t)bh * a.nsplit * a.rows + row) * a.value_dim;
    const int64_t stride = (int64_t)a.rows * a.value_dim;
    const int dv = chunk * QL * 4 + lane % QL * 4;
    const float *from = part + (dv < a.value_dim ? dv : 0);
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s0 = 0; s0 < a.nsplit; s0 += 64 / QL) {
      const int s = s0 + lane / QL;
      const float f0 = __shfl(J.f[0], s & 63), f1 = __shfl(J.f[1], s & 63), f = s < 64 ? f0 : f1;
      const f32x4 x = *reinterpret_cast<const f32x4 *>(from + (s < a.nsplit ? s : 0) * stride);      // (no branch: all loads go out together)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c] += s < a.nsplit ? f * x[c] : 0.f;
    }
#pragma unroll
    for (int d = QL; d < 64; d <<= 1)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c] += __shfl_xor(acc[c], d);
    if (lane < QL && dv < a.value_dim) {
      typedef T Tx4 __attribute__((ext_vector_type(4)));
      Tx4 y;
#pragma unroll
      for (int c = 0; c < 4; ++c) y[c] = (T)(J.inv == 0.f ? 0.f : acc[c] * J.inv);
      *reinterpret_cast<Tx4 *>(out + dv) = y;
    }
    return;
  }
  if (a.q_pack) {                     // 32 rows a wave, as bf16 parts in the order of bank4_weigh's operand
    const int tiles = (int)(a.row_stride / 32), KS = a.key_dim / 16;
    const int64_t g = (int64_t)(blockIdx.x - out_blocks) * 4 + wave;
    if (g >= (int64_t)a.batch * a.heads * tiles) return;
    const int bh = (int)(g / tiles), tile = (int)(g - (int64_t)bh * tiles), b = bh / a.heads, h = bh - b * a.heads, half = lane >> 5;
    const int r = tile * 32 + (lane & 31), t = r / a.group;
    const bool live = r < a.rows && t < read_count(a, b);
    const T *row = (const T *)a.q + b * a.qb + (int64_t)(live ? t : 0) * a.qt + (int64_t)(h * a.group + (live ? r - t * a.group : 0)) * a.qh;
    bf16x8 *to = reinterpret_cast<bf16x8 *>(a.q_pack) + g * (KS * PARTS * 64) + lane;
    auto channels = [&](int i) {
      f32x8 y = load8(row + (i / 4) * 64 + half * 32 + (i & 3) * 8, a.q_vec);
#pragma unroll
      for (int c = 0; c < 8; ++c) y[c] = live ? y[c] * a.q_sign : 0.f;
      return y;
    };
    float up = 1.f, scale = 1.f, lost = 0.f;
    if constexpr (PARTS == 3) {
      float top = 0.f;
      for (int i = 0; i < KS; ++i) {
        const f32x8 y = channels(i);
#pragma unroll
        for (int c = 0; c < 8; ++c) top = fmaxf(top, __builtin_fabsf(y[c]));
      }
      const int t = query_shift(fmaxf(top, __shfl_xor(top, 32)));
      up = pow2(t);
      scale = row_scale(a.scale_log2, pow2(-t));
      if (half == 0) a.row_scale[(int64_t)bh * a.row_stride + r] = scale;
    }
    for (int i = 0; i < KS; ++i) {
      const f32x8 y = channels(i);
      bf16x8 qf[PARTS];
      split8<PARTS>(y, qf);
#pragma unroll
      for (int p = 0; p < PARTS; ++p) to[(i * PARTS + p) * 64] = qf[p];
      if constexpr (PARTS > 1) {
        f16x8 hf[PARTS - 1];
        split8<PARTS - 1>(y * up, hf);
        if constexpr (PARTS == 3) lost += left_out(y * up, hf);
#pragma unroll
        for (int p = 0; p < PARTS - 1; ++p) (reinterpret_cast<f16x8 *>(a.q_pack_f16) + g * (KS * (PARTS - 1) * 64) + lane)[(i * (PARTS - 1) + p) * 64] = hf[p];
      }
    }
    if constexpr (PARTS == 3) {
      uint32_t limit = key_byte_limit(lost + __shfl_xor(lost, 32), scale);
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t x = __shfl_xor(limit, d);
        limit = x < limit ? x : limit;
      }
      if (lane == 0) a.row_limit[(int64_t)bh * a.row_stride + tile * 32] = limit;
    }
    return;
  }
  __shared__ float top[BLOCK_ROWS_MIN], inv[BLOCK_ROWS_MIN];
  __shared__ int lim[BLOCK_ROWS_MIN];
  const int per = (int)((a.slots + 1023) / 1024), g = blockIdx.x - out_blocks, bh = g / per, b = bh / a.heads;
  const int64_t slot = (int64_t)(g - bh * per) * 1024 + tid * 4;
  const int64_t len = read_len(a, b);
  if (slot - tid * 4 >= len) return;
  const int cnt = read_count(a, b);
  for (int i = wave; i < a.rows; i += 4) {
    const RowJoin J(a, bh, i, lane);
    if (lane == 0) { top[i] = J.top; inv[i] = J.inv; lim[i] = (int)read_limit(a, len, cnt, i / a.group); }
  }
  __syncthreads();
  if (slot >= len) return;
  f32x4 acc{0.f, 0.f, 0.f, 0.f};
  const float *x0 = a.logits + (int64_t)bh * a.rows * a.logit_stride + slot;
#pragma unroll 4
  for (int i = 0; i < a.rows; ++i) {
    const f32x4 x = *reinterpret_cast<const f32x4 *>(x0 + (int64_t)i * a.logit_stride);   // written up to the row's limit only
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] += slot + j < lim[i] ? inv[i] * __builtin_amdgcn_exp2f(__builtin_fmaf(x[j], a.scale_log2, -top[i])) : 0.f;
  }
  float *w = a.weight + (int64_t)bh * a.slots + slot;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (slot + j < len) w[j] += acc[j];
}

// ---------------------------------------------------------------------------------------------- launch plan
struct ReadPlan {
  int rows, tiles, nsplit, nvc, dvc;
  bool block;                        // 128 rows a workgroup (else 16)
  bool parts;                        // partial results go through the workspace
  int64_t part_o, part_ml, logits, row_stat, q_pack, q_pack_f16, redo, logit_stride, row_stride;      // bytes; strides in elements
  int64_t bytes() const { return part_o + part_ml + logits + row_stat + q_pack + q_pack_f16 + redo; }
};

// Value channels a workgroup accumulates: every chunk computes the logits again, so as many as the registers hold.
static int read_dvc(int dk, int dv, bool block) {
  if (block && dk <= 128 && dv % 256 == 0) return 256;
  return dv % 128 ? 64 : 128;
}

static int read_plan(const mivos_bank4 *k, int q_heads, int tokens, int weigh, int dtype, ReadPlan *p) {
  if (q_heads < 1 || q_heads % k->heads || tokens < 0) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: %d query heads over %d bank heads, %d tokens", q_heads, k->heads, tokens);
  if (k->key_dim != 64 && k->key_dim != 128 && k->key_dim != 256) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: keys of %d channels (64, 128 or 256)", k->key_dim);
  if (k->value_dim % 64) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: values of %d channels (a multiple of 64)", k->value_dim);
  const int64_t rows = (int64_t)tokens * (q_heads / k->heads);
  if (rows > (1 << 20)) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: %lld rows a bank head (at most 2^20)", (long long)rows);
  p->rows = (int)rows;
  p->block = rows >= BLOCK_ROWS_MIN;
  p->tiles = cdiv(rows, p->block ? 128 : 16);
  p->dvc = read_dvc(k->key_dim, k->value_dim, p->block);
  p->nvc = k->value_dim / p->dvc;
  const int64_t groups = (int64_t)p->tiles * k->batch * k->heads * p->nvc;
  if (p->block) {
    // Slices of a row tile's slots: the fewest rounds of the workgroups that run at once (two a CU where their registers allow it), a slice
    // costing its join (its accumulators are written and read once more) and its start.
    const int at_once = 256 * block_occupancy(k->key_dim, p->dvc, query_parts(dtype));
    const int most = (int)(k->slots / 512 < 1 ? 1 : k->slots / 512 > 128 ? 128 : k->slots / 512);     // (8 steps a slice pay for its start)
    double best = 1e30;
    for (int n = 1; n <= most; ++n) {
      const double cost = (double)((groups * n + at_once - 1) / at_once) / n * (1 + 0.01 * n);
      if (cost < best - 1e-9) { best = cost; p->nsplit = n; }
    }
  } else {
    const int64_t want = groups ? (2048 + groups - 1) / groups : 1, most = (k->slots + 255) / 256;
    p->nsplit = (int)(want < most ? want : most);
    p->nsplit = p->nsplit > 128 ? 128 : p->nsplit < 1 || k->slots <= 1024 ? 1 : p->nsplit;
    // (a short bank: no second launch; 1 token, 1 to 64 heads, values of 64 to 512: 8.3 - 10.5 us at 1024 slots, 11.7 - 11.8 in slices at 1025; with
    // the weights gathered, which take that launch anyway, 15.7 and 11.9.  The plan knows the capacity only: 1000 slots filled of 65 536 take 19 us)
  }
  p->parts = p->nsplit > 1 || weigh;
  const int64_t n = (int64_t)k->batch * k->heads * p->nsplit * rows;
  p->part_o = p->parts ? n * k->value_dim * 4 : 0;
  p->part_ml = p->parts ? (n * 8 + 15) / 16 * 16 : 0;
  p->logit_stride = (k->slots + 63) / 64 * 64;
  p->logits = weigh && !p->block ? (int64_t)k->batch * k->heads * rows * p->logit_stride * 4 : 0;
  p->row_stride = (rows + 31) / 32 * 32;
  const int64_t packed = weigh && p->block ? (int64_t)k->batch * k->heads * p->row_stride : 0, f16 = query_parts(dtype) - 1;
  p->row_stat = packed * 16;
  p->q_pack = packed * k->key_dim * 2 * (f16 + 1);
  p->q_pack_f16 = packed * k->key_dim * 2 * f16;
  const int64_t flags = groups * p->nsplit, flags_weigh = weigh ? (int64_t)k->batch * k->heads * ((k->slots + 127) / 128) : 0;
  p->redo = p->block && f16 ? ((flags > flags_weigh ? flags : flags_weigh) * 4 + 15) / 16 * 16 : 0;
  return MIVOS_OK;
}

template <int DK, int DVC, int PARTS, bool F16, bool CAUSAL>
static int block_launch_one(const ReadArgs &a, const dim3 grid, hipStream_t s) {
  constexpr size_t lds = 2 * 64 * (DVC + 16) * 2;
  void (*kernel)(ReadArgs);
  if constexpr (PARTS == 1) kernel = bank4_block_bf16_kernel<DK, DVC, CAUSAL>;
  else kernel = bank4_block_kernel<DK, DVC, PARTS, F16, CAUSAL>;
  if constexpr (lds > 65536) {
    static std::atomic<uint64_t> raised{0};
    if (int rc = ensure_dynamic_lds((const void *)kernel, lds, raised, "bank4_read")) return rc;
  }
  kernel<<<grid, 256, lds, s>>>(a);
  return MIVOS_OK;
}

template <int DK, int DVC, int PARTS>
static int block_launch(const ReadArgs &a, const dim3 grid, hipStream_t s) {
  if (int rc = a.causal ? block_launch_one<DK, DVC, PARTS, true, true>(a, grid, s) : block_launch_one<DK, DVC, PARTS, true, false>(a, grid, s)) return rc;
  if constexpr (PARTS > 1) return a.causal ? block_launch_one<DK, DVC, PARTS, false, true>(a, grid, s) : block_launch_one<DK, DVC, PARTS, false, false>(a, grid, s);
  return MIVOS_OK;
}

template <int DK, int PARTS>
static int read_launch(const ReadArgs &a, const ReadPlan &p, hipStream_t s) {
  const dim3 grid(p.nsplit, p.tiles, a.batch * a.heads * p.nvc);
  if (p.block) {
    if constexpr (DK <= 128)
      if (p.dvc == 256) return block_launch<DK, 256, PARTS>(a, grid, s);
    return p.dvc == 64 ? block_launch<DK, 64, PARTS>(a, grid, s) : block_launch<DK, 128, PARTS>(a, grid, s);
  }
  if (p.dvc == 64) bank4_rows_kernel<DK, 64, PARTS><<<grid, 256, 0, s>>>(a);
  else bank4_rows_kernel<DK, 128, PARTS><<<grid, 256, 0, s>>>(a);
  return MIVOS_OK;
}

template <int DK>
static int read_launch(const ReadArgs &a, const ReadPlan &p, int dtype, hipStream_t s) {
  if (dtype == MIVOS_BF16) return read_launch<DK, 1>(a, p, s);
  return dtype == MIVOS_F16 ? read_launch<DK, 2>(a, p, s) : read_launch<DK, 3>(a, p, s);
}

// Lanes over the value channels of a joined row: few rows are bound by the chain of their slices (one token over 8192 slots, values of 512: 13 us a
// call instead of 28; 65 536 slots: 22 instead of 32), many by bytes.
static int join_lanes(int64_t rows, int value_dim) { return value_dim <= 64 || rows <= 512 ? 16 : value_dim <= 128 ? 32 : 64; }

template <int PARTS>
static void join_launch(const ReadArgs &a, int lanes, int blocks, int out_blocks, hipStream_t s) {
  if (lanes == 16) bank4_join_kernel<PARTS, 16><<<blocks, 256, 0, s>>>(a, out_blocks);
  else if (lanes == 32) bank4_join_kernel<PARTS, 32><<<blocks, 256, 0, s>>>(a, out_blocks);
  else bank4_join_kernel<PARTS, 64><<<blocks, 256, 0, s>>>(a, out_blocks);
}

template <int DK, int PARTS, int NS, typename V8, bool SHIFT>
static int weigh_launch_one(const ReadArgs &a, hipStream_t s) {
  constexpr size_t lds = 2 * (DK / 16) * PARTS * 64 * 16;
  if constexpr (lds > 65536) {
    static std::atomic<uint64_t> raised{0};
    if (int rc = ensure_dynamic_lds((const void *)bank4_weigh_kernel<DK, PARTS, NS, V8, SHIFT>, lds, raised, "bank4_read")) return rc;
  }
  bank4_weigh_kernel<DK, PARTS, NS, V8, SHIFT><<<dim3(cdiv(a.slots, 128 * NS), a.batch * a.heads), 256, lds, s>>>(a);
  return MIVOS_OK;
}

template <int DK, int PARTS, int NS>
static int weigh_launch_two(const ReadArgs &a, hipStream_t s) {
  if constexpr (PARTS > 1)
    if (int rc = weigh_launch_one<DK, PARTS - 1, NS, f16x8, PARTS == 3>(a, s)) return rc;
  return weigh_launch_one<DK, PARTS, NS, bf16x8, false>(a, s);
}

// 256 slots a workgroup where that still gives every CU one; else 128
template <int DK, int PARTS>
static int weigh_launch(const ReadArgs &a, hipStream_t s) {
  if (a.batch * a.heads * (a.slots / 256) >= 240) return weigh_launch_two<DK, PARTS, 2>(a, s);
  return weigh_launch_two<DK, PARTS, 1>(a, s);
}

template <int DK>
static int weigh_launch(const ReadArgs &a, int dtype, hipStream_t s) {
  return dtype == MIVOS_BF16 ? weigh_launch<DK, 1>(a, s) : dtype == MIVOS_F16 ? weigh_launch<DK, 2>(a, s) : weigh_launch<DK, 3>(a, s);
}

}  // namespace mivos

using namespace mivos;

extern "C" int64_t mivos_bank4_read_workspace_bytes(const mivos_bank4 *bank, int q_heads, int tokens, int dtype, int weigh) {
  ReadPlan p;
  if (int rc = bank4_check(bank, "bank4_read")) return rc;
  if (int rc = read_plan(bank, q_heads, tokens, weigh, dtype, &p)) return rc;
  return p.bytes();
}

extern "C" int mivos_bank4_read(const mivos_bank4 *bank, const void *q, int64_t qb, int64_t qt, int64_t qh, int dtype, int q_heads, int tokens,
                                const int32_t *count, float scale, int causal, int weigh, void *out, void *workspace, int64_t workspace_bytes,
                                void *stream) {
  ReadPlan p;
  if (int rc = bank4_check(bank, "bank4_read")) return rc;
  if (!dtype_ok(dtype) || (tokens > 0 && (!q || !out)) || !(scale >= -1e38f && scale <= 1e38f))
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: bad argument (|scale| up to 1e38)");
  if (int rc = read_plan(bank, q_heads, tokens, weigh, dtype, &p)) return rc;
  if (p.rows == 0) return MIVOS_OK;
  const int64_t need = p.bytes();
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: workspace of %lld bytes, 16-byte aligned", (long long)need);
  if (p.tiles > 65535 || (int64_t)bank->batch * bank->heads * p.nvc > 65535) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: too many row tiles");
  // the join's workgroups: four rows (or shares of their channels) each; then the weights of 1024 slots each, or four tiles of queries to pack
  const int64_t heads = (int64_t)bank->batch * bank->heads, lanes = join_lanes(heads * p.rows, bank->value_dim);
  const int64_t out_blocks = (heads * p.rows * cdiv(bank->value_dim, 4 * lanes) + 3) / 4;
  const int64_t blocks = out_blocks + (p.logits ? heads * ((bank->slots + 1023) / 1024) : 0) + (p.q_pack ? (heads * (p.row_stride / 32) + 3) / 4 : 0);
  if (p.parts && blocks >= 1 << 24) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: too many rows");
  hipStream_t s = (hipStream_t)stream;
  ReadArgs a{};
  a.kc = bank->key_codes; a.ks = bank->key_scales; a.vc = bank->value_codes; a.vs = bank->value_scales;
  a.weight = bank->weight; a.lens = bank->lens; a.count = count; a.q = q; a.out = out; a.qb = qb; a.qt = qt; a.qh = qh;
  char *ws = (char *)workspace;
  if (p.parts) { a.part_o = (float *)ws; a.part_ml = (float *)(ws + p.part_o); }
  if (p.logits) a.logits = (float *)(ws + p.part_o + p.part_ml);
  if (p.row_stat) {
    a.row_max = (float *)(ws + p.part_o + p.part_ml);
    a.row_inv = a.row_max + p.row_stat / 16;
    a.row_scale = a.row_inv + p.row_stat / 16;
    a.row_limit = (uint32_t *)(a.row_scale + p.row_stat / 16);
    a.q_pack = (__bf16 *)(ws + p.part_o + p.part_ml + p.row_stat);
    a.q_pack_f16 = (_Float16 *)((char *)a.q_pack + p.q_pack);
  }
  if (p.redo) a.redo = (int32_t *)(ws + need - p.redo);
  a.slots = bank->slots; a.logit_stride = p.logit_stride; a.row_stride = p.row_stride;
  a.batch = bank->batch; a.heads = bank->heads; a.group = q_heads / bank->heads; a.tokens = tokens; a.rows = p.rows;
  a.key_dim = bank->key_dim; a.value_dim = bank->value_dim; a.nsplit = p.nsplit; a.causal = causal; a.scale_log2 = scale * LOG2E;
  // logits are compared before they are scaled: a scale above 0, its sign (or the 0) with the queries
  a.q_sign = scale < 0.f ? -1.f : scale > 0.f ? 1.f : 0.f;
  a.scale_log2 = scale != 0.f ? a.scale_log2 * a.q_sign : 1.f;
  a.q_vec = (((qb | qt | qh) * dtype_bytes(dtype)) & 15) == 0 && ((uintptr_t)q & 15) == 0;
  if (int rc = bank->key_dim == 64 ? read_launch<64>(a, p, dtype, s) : bank->key_dim == 128 ? read_launch<128>(a, p, dtype, s) : read_launch<256>(a, p, dtype, s))
    return rc;
  if (int rc = check_launch("bank4_read")) return rc;
  if (!p.parts) return MIVOS_OK;
  if (dtype == MIVOS_BF16) join_launch<1>(a, (int)lanes, (int)blocks, (int)out_blocks, s);
  else if (dtype == MIVOS_F16) join_launch<2>(a, (int)lanes, (int)blocks, (int)out_blocks, s);
  else join_launch<3>(a, (int)lanes, (int)blocks, (int)out_blocks, s);
  if (int rc = check_launch("bank4_read")) return rc;
  if (!a.row_max) return MIVOS_OK;
  if (int rc = bank->key_dim == 64 ? weigh_launch<64>(a, dtype, s) : bank->key_dim == 128 ? weigh_launch<128>(a, dtype, s) : weigh_launch<256>(a, dtype, s))
    return rc;
  return check_launch("bank4_read");
}
