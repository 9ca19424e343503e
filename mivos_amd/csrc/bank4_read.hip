// Attention over the 4-bit memory bank:  out[t, j] = sum_s softmax_s(scale * q[t, j] . k[s, j / G]) v[s, j / G],  G query heads a bank head,
// softmax over the visible slots of the stream (all of them, or causally those up to the token's own place), a row that sees nothing is 0;
// and, when asked, weight[s] += sum over the rows (tokens x G) of their softmax weight on slot s.
//
// Arithmetic.  A bank value has at most two significant bits and is exact in bf16, so both products run on the bf16 matrix cores with
// exact bank operands: q (and the softmax weight p) is written as a sum of PARTS bf16 numbers - 1 for bf16 inputs (q exact, p rounded once,
// 2^-8 of each term, the size of the output's own rounding), 2 for fp16 (11 bits of q exactly, 16 bits of p), 3 for fp32 (24 bits of both).
// Running maximum, sum and accumulators are fp32.
//
// Layout.  S^T = K Q^T on 16x16x32: lane l holds bank row l % 16 and channels (l / 16) * DK / 4 .. + DK / 4 of it - contiguous codes in memory,
// mostly of one scale block, so K needs no staging; Q is kept in registers in the same channel order.  The result gives a lane one query
// (column l % 16) and four keys a tile, which is the B operand of O^T = V^T P^T as it stands (the 8 keys of a lane in a pair of tiles are
// the same 8 in both operands).  V rows are widened to bf16 in a wave's own LDS patch and read back transposed (ds_read_b64_tr_b16).
#include "bank4.h"

namespace mivos {

constexpr float LOG2E = 1.4426950408889634f;

struct ReadArgs {
  const uint8_t *kc, *ks, *vc, *vs;
  float *weight;
  const int32_t *lens, *count;
  const void *q;
  void *out;
  int64_t qb, qt, qh;
  float *part_o, *part_ml, *logits;
  int64_t slots, logit_stride;
  int batch, heads, group, tokens, rows, value_dim, nsplit, causal, weigh, q_vec;
  float scale_log2;       // scale * log2(e): the softmax runs in powers of two
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

template <int PARTS>
__device__ __forceinline__ void split8(f32x8 x, bf16x8 (&p)[PARTS]) {
#pragma unroll
  for (int k = 0; k < PARTS; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[k][j] = (__bf16)x[j];
      x[j] -= (float)p[k][j];
    }
}

template <int PARTS> struct ReadType;
template <> struct ReadType<1> { typedef __bf16 T; };
template <> struct ReadType<2> { typedef _Float16 T; };
template <> struct ReadType<3> { typedef float T; };

// One workgroup: 16 rows x one slice of the slots x DVC value channels; its four waves take 64 slots in turn, each with a running
// softmax of its own, and meet in LDS at the end.
template <int DK, int DVC, int PARTS>
__global__ __launch_bounds__(256) void bank4_rows_kernel(ReadArgs a) {
  typedef typename ReadType<PARTS>::T T;
  constexpr int CPL = DK / 4, KSTEPS = DK / 32, VPAD = DVC + 16, OPAD = DVC + 4, NT = DVC / 16;
  constexpr int LDS_V = 4 * 32 * VPAD * 2, LDS_O = 4 * 16 * OPAD * 4;
  __shared__ __align__(16) char lds[LDS_V > LDS_O ? LDS_V : LDS_O];
  __shared__ float stat[4][16][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;
  const int nvc = a.value_dim / DVC, chunk = blockIdx.z % nvc, bh = blockIdx.z / nvc, b = bh / a.heads, h = bh - b * a.heads;
  const int split = blockIdx.x, row0 = blockIdx.y * 16;
  const int64_t len = read_len(a, b);
  const int cnt = read_count(a, b);
  const int r = row0 + col, t = r / a.group;
  const int64_t limit = r < a.rows ? read_limit(a, len, cnt, t) : 0;
  const int last_row = row0 + 15 < a.rows ? row0 + 15 : a.rows - 1;
  int last_t = last_row / a.group;
  last_t = last_t < cnt ? last_t : cnt - 1;
  const int64_t seen = row0 / a.group < cnt ? read_limit(a, len, cnt, last_t) : 0;   // slots any row of the tile sees
  const int64_t per = ((seen + 63) / 64 + a.nsplit - 1) / a.nsplit * 64;
  const int64_t s0 = split * per, s1 = s0 + per < seen ? s0 + per : seen;

  bf16x8 qf[KSTEPS][PARTS];
  {
    const bool live = r < a.rows && t < cnt;
    const T *qrow = (const T *)a.q + b * a.qb + (live ? t : 0) * a.qt + (int64_t)(h * a.group + (live ? r - t * a.group : 0)) * a.qh + grp * CPL;
#pragma unroll
    for (int i = 0; i < KSTEPS; ++i) {
      f32x8 x = load8(qrow + i * 8, a.q_vec);
      if (!live)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
      split8<PARTS>(x, qf[i]);
    }
  }
  f32x4 o[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const int64_t row_base = (int64_t)bh * a.slots;
  __bf16 *vt = reinterpret_cast<__bf16 *>(lds) + wave * 32 * VPAD;
  const int vs_row = a.value_dim / 32;

  for (int64_t base = s0 + wave * 64; base < s1; base += 256) {
    // ---- logits of 64 slots
    f32x4 x[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const int64_t slot = base + kt * 16 + col, row = row_base + (slot < a.slots ? slot : a.slots - 1);
      const uint32_t *codes = reinterpret_cast<const uint32_t *>(a.kc + row * (DK / 2) + grp * (CPL / 2));
      const uint8_t *sc = a.ks + row * (DK / 32) + grp * CPL / 32;
      x[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KSTEPS; ++i) {
        const bf16x8 kf = bank4_unpack8(codes[i], bank4_scale(sc[i * 8 / 32]));
#pragma unroll
        for (int p = 0; p < PARTS; ++p) x[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[i][p], x[kt], 0, 0, 0);
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t slot = base + kt * 16 + grp * 4 + j;
        x[kt][j] = slot < limit && slot < s1 ? x[kt][j] * a.scale_log2 : -INFINITY;
        top = fmaxf(top, x[kt][j]);
      }
      if (a.weigh && chunk == 0 && r < a.rows)
        *reinterpret_cast<f32x4 *>(a.logits + ((int64_t)bh * a.rows + r) * a.logit_stride + base + kt * 16 + grp * 4) = x[kt];
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float mn = fmaxf(m, top), mu = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m - mu);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] *= alpha;
    // ---- V in two halves of 32 slots
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      f32x8 p;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(x[half * 2 + j / 4][j % 4] - mu);
        l += p[j];
      }
      bf16x8 pf[PARTS];
      split8<PARTS>(p, pf);
      wave_lds_fence();
#pragma unroll
      for (int i = 0; i < DVC / 64; ++i) {       // 32 rows x DVC / 32 blocks of 16 bytes over 64 lanes
        const int e = i * 64 + lane, vr = e / (DVC / 32), blk = e % (DVC / 32);
        const int64_t slot = base + half * 32 + vr, row = row_base + (slot < a.slots ? slot : a.slots - 1);
        u32x4 codes = *reinterpret_cast<const u32x4 *>(a.vc + row * (a.value_dim / 2) + chunk * (DVC / 2) + blk * 16);
        uint32_t byte = a.vs[row * vs_row + chunk * (DVC / 32) + blk];
        if (slot >= s1) { codes = u32x4{0u, 0u, 0u, 0u}; byte = 127; }      // never-written memory may stand for NaN
        const float sc = bank4_scale(byte);
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<bf16x8 *>(vt + vr * VPAD + blk * 32 + j * 8) = bank4_unpack8(codes[j], sc);
      }
      wave_lds_fence();
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        typedef __attribute__((address_space(3))) s16x4 *lds_p;
        const __bf16 *at = vt + (grp * 4 + col / 4) * VPAD + i * 16 + (col % 4) * 4;
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(at));
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(at + 16 * VPAD));
        const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int q = 0; q < PARTS; ++q) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[q], o[i], 0, 0, 0);
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
      a.part_o[at * a.value_dim + chunk * DVC + dv] = acc;
      if (dv == 0 && chunk == 0) { a.part_ml[at * 2] = mm; a.part_ml[at * 2 + 1] = sum; }
    } else {
      const int tt = row / a.group, j = h * a.group + row - tt * a.group;
      ((T *)a.out)[(((int64_t)b * a.tokens + tt) * a.heads * a.group + j) * a.value_dim + chunk * DVC + dv] = (T)(sum != 0.f ? acc / sum : 0.f);
    }
  }
}

// Joins the slices of a row (first `out_blocks` workgroups, one wave a row) and adds the rows' weights to the slots (the others,
// 1024 slots each, the rows in order: the sum does not depend on timing).
template <int PARTS>
__global__ __launch_bounds__(256) void bank4_join_kernel(ReadArgs a, int out_blocks) {
  typedef typename ReadType<PARTS>::T T;
  __shared__ float lse[256];
  __shared__ int lim[256];
  const int tid = threadIdx.x, lane = tid & 63;
  const int n_bh = a.batch * a.heads;
  if ((int)blockIdx.x < out_blocks) {
    const int64_t g = (int64_t)blockIdx.x * 4 + (tid >> 6);
    if (g >= (int64_t)n_bh * a.rows) return;
    const int bh = (int)(g / a.rows), row = (int)(g - (int64_t)bh * a.rows), b = bh / a.heads, h = bh - b * a.heads;
    const float *ml = a.part_ml + ((int64_t)bh * a.nsplit * a.rows + row) * 2;
    float mm = -INFINITY, sum = 0.f;
    for (int s = 0; s < a.nsplit; ++s) mm = fmaxf(mm, ml[(int64_t)s * a.rows * 2]);
    const float mu = mm == -INFINITY ? 0.f : mm;
    for (int s = 0; s < a.nsplit; ++s) sum += __builtin_amdgcn_exp2f(ml[(int64_t)s * a.rows * 2] - mu) * ml[(int64_t)s * a.rows * 2 + 1];
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    const int t = row / a.group, j = h * a.group + row - t * a.group;
    T *out = (T *)a.out + (((int64_t)b * a.tokens + t) * a.heads * a.group + j) * a.value_dim;
    for (int dv = lane; dv < a.value_dim; dv += 64) {
      float acc = 0.f;
      for (int s = 0; s < a.nsplit; ++s)
        acc += __builtin_amdgcn_exp2f(ml[(int64_t)s * a.rows * 2] - mu) * a.part_o[(((int64_t)bh * a.nsplit + s) * a.rows + row) * a.value_dim + dv];
      out[dv] = (T)(acc * inv);
    }
    return;
  }
  const int per = (int)((a.slots + 1023) / 1024), g = blockIdx.x - out_blocks, bh = g / per, b = bh / a.heads;
  const int64_t slot = (int64_t)(g - bh * per) * 1024 + tid * 4;
  const int64_t len = read_len(a, b);
  const int cnt = read_count(a, b);
  f32x4 acc{0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < a.rows; r0 += 256) {
    const int n = a.rows - r0 < 256 ? a.rows - r0 : 256;
    __syncthreads();
    if (tid < n) {
      const float *ml = a.part_ml + ((int64_t)bh * a.nsplit * a.rows + r0 + tid) * 2;
      float mm = -INFINITY, sum = 0.f;
      for (int s = 0; s < a.nsplit; ++s) mm = fmaxf(mm, ml[(int64_t)s * a.rows * 2]);
      const float mu = mm == -INFINITY ? 0.f : mm;
      for (int s = 0; s < a.nsplit; ++s) sum += __builtin_amdgcn_exp2f(ml[(int64_t)s * a.rows * 2] - mu) * ml[(int64_t)s * a.rows * 2 + 1];
      lse[tid] = sum != 0.f ? mu + __builtin_amdgcn_logf(sum) : 0.f;
      lim[tid] = (int)read_limit(a, len, cnt, (r0 + tid) / a.group);
    }
    __syncthreads();
    if (slot < len)
      for (int i = 0; i < n; ++i) {
        if (slot >= lim[i]) continue;
        const f32x4 x = *reinterpret_cast<const f32x4 *>(a.logits + ((int64_t)bh * a.rows + r0 + i) * a.logit_stride + slot);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += slot + j < lim[i] ? __builtin_amdgcn_exp2f(x[j] - lse[i]) : 0.f;
      }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (slot + j < len) a.weight[(int64_t)bh * a.slots + slot + j] += acc[j];
}

// ---------------------------------------------------------------------------------------------- launch plan
struct ReadPlan {
  int rows, tiles, nsplit, nvc, dvc;
  bool parts;                        // partial results go through the workspace
  int64_t part_o, part_ml, logits, logit_stride;      // bytes
};

static int read_plan(const mivos_bank4 *k, int q_heads, int tokens, int weigh, ReadPlan *p) {
  if (q_heads < 1 || q_heads % k->heads || tokens < 0) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: %d query heads over %d bank heads, %d tokens", q_heads, k->heads, tokens);
  if (k->key_dim != 64 && k->key_dim != 128 && k->key_dim != 256) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: keys of %d channels (64, 128 or 256)", k->key_dim);
  if (k->value_dim % 64) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: values of %d channels (a multiple of 64)", k->value_dim);
  const int64_t rows = (int64_t)tokens * (q_heads / k->heads);
  if (rows > (1 << 20)) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: %lld rows a bank head (at most 2^20)", (long long)rows);
  p->rows = (int)rows;
  p->tiles = cdiv(rows, 16);
  p->dvc = k->value_dim % 128 ? 64 : 128;
  p->nvc = k->value_dim / p->dvc;
  const int64_t groups = (int64_t)p->tiles * k->batch * k->heads * p->nvc;
  const int64_t want = groups ? (2048 + groups - 1) / groups : 1, most = (k->slots + 255) / 256;
  p->nsplit = (int)(want < most ? want : most);
  p->nsplit = p->nsplit > 128 ? 128 : p->nsplit < 1 ? 1 : p->nsplit;
  p->parts = p->nsplit > 1 || weigh;
  const int64_t n = (int64_t)k->batch * k->heads * p->nsplit * rows;
  p->part_o = p->parts ? n * k->value_dim * 4 : 0;
  p->part_ml = p->parts ? (n * 8 + 15) / 16 * 16 : 0;
  p->logit_stride = (k->slots + 63) / 64 * 64;
  p->logits = weigh ? (int64_t)k->batch * k->heads * rows * p->logit_stride * 4 : 0;
  return MIVOS_OK;
}

template <int DK, int DVC>
static void rows_launch(const ReadArgs &a, const ReadPlan &p, int dtype, hipStream_t s) {
  const dim3 grid(p.nsplit, p.tiles, a.batch * a.heads * p.nvc);
  if (dtype == MIVOS_BF16) bank4_rows_kernel<DK, DVC, 1><<<grid, 256, 0, s>>>(a);
  else if (dtype == MIVOS_F16) bank4_rows_kernel<DK, DVC, 2><<<grid, 256, 0, s>>>(a);
  else bank4_rows_kernel<DK, DVC, 3><<<grid, 256, 0, s>>>(a);
}

}  // namespace mivos

using namespace mivos;

extern "C" int64_t mivos_bank4_read_workspace_bytes(const mivos_bank4 *bank, int q_heads, int tokens, int weigh) {
  ReadPlan p;
  if (int rc = bank4_check(bank, "bank4_read")) return rc;
  if (int rc = read_plan(bank, q_heads, tokens, weigh, &p)) return rc;
  return p.part_o + p.part_ml + p.logits;
}

extern "C" int mivos_bank4_read(const mivos_bank4 *bank, const void *q, int64_t qb, int64_t qt, int64_t qh, int dtype, int q_heads, int tokens,
                                const int32_t *count, float scale, int causal, int weigh, void *out, void *workspace, int64_t workspace_bytes,
                                void *stream) {
  ReadPlan p;
  if (int rc = bank4_check(bank, "bank4_read")) return rc;
  if (!dtype_ok(dtype) || (tokens > 0 && (!q || !out))) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: bad argument");
  if (int rc = read_plan(bank, q_heads, tokens, weigh, &p)) return rc;
  if (p.rows == 0) return MIVOS_OK;
  const int64_t need = p.part_o + p.part_ml + p.logits;
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: workspace of %lld bytes, 16-byte aligned", (long long)need);
  if (p.tiles > 65535 || (int64_t)bank->batch * bank->heads * p.nvc > 65535) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: too many row tiles");
  hipStream_t s = (hipStream_t)stream;
  ReadArgs a{};
  a.kc = bank->key_codes; a.ks = bank->key_scales; a.vc = bank->value_codes; a.vs = bank->value_scales;
  a.weight = bank->weight; a.lens = bank->lens; a.count = count; a.q = q; a.out = out; a.qb = qb; a.qt = qt; a.qh = qh;
  char *ws = (char *)workspace;
  if (p.parts) { a.part_o = (float *)ws; a.part_ml = (float *)(ws + p.part_o); }
  if (weigh) a.logits = (float *)(ws + p.part_o + p.part_ml);
  a.slots = bank->slots; a.logit_stride = p.logit_stride;
  a.batch = bank->batch; a.heads = bank->heads; a.group = q_heads / bank->heads; a.tokens = tokens; a.rows = p.rows;
  a.value_dim = bank->value_dim; a.nsplit = p.nsplit; a.causal = causal; a.weigh = weigh; a.scale_log2 = scale * LOG2E;
  a.q_vec = (((qb | qt | qh) * dtype_bytes(dtype)) & 15) == 0 && ((uintptr_t)q & 15) == 0;
#define GO(DK) (p.dvc == 64 ? rows_launch<DK, 64>(a, p, dtype, s) : rows_launch<DK, 128>(a, p, dtype, s))
  if (bank->key_dim == 64) GO(64);
  else if (bank->key_dim == 128) GO(128);
  else GO(256);
#undef GO
  if (int rc = check_launch("bank4_read")) return rc;
  if (!p.parts) return MIVOS_OK;
  const int64_t out_blocks = ((int64_t)a.batch * a.heads * a.rows + 3) / 4;
  const int64_t blocks = out_blocks + (weigh ? (int64_t)a.batch * a.heads * ((a.slots + 1023) / 1024) : 0);
  if (blocks > 0x7fffffff) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_read: too many rows");
  if (dtype == MIVOS_BF16) bank4_join_kernel<1><<<(int)blocks, 256, 0, s>>>(a, (int)out_blocks);
  else if (dtype == MIVOS_F16) bank4_join_kernel<2><<<(int)blocks, 256, 0, s>>>(a, (int)out_blocks);
  else bank4_join_kernel<3><<<(int)blocks, 256, 0, s>>>(a, (int)out_blocks);
  return check_launch("bank4_read");
}
