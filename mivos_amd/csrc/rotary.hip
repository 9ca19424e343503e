// Rotary positions with several axes (time, height, width), alone or behind the norm of each head's query / key, and their gradients.
//
//   n = w * x * (mean(x^2) + eps)^(-1/2)                      (norm; w per channel, shared by the heads)          or n = x
//   y[u] = n[u] cos a_i - n[v] sin a_i,  y[v] = n[v] cos a_i + n[u] sin a_i        a_i = position[axis_i] * f_i,   pair i = channels (u, v)
// with pairs (2i, 2i + 1) or (i, i + pairs); channels behind the pairs keep n.  Backward: g = the rotation by -a of dy,
//   dx = r (w g - x r^2 mean(w g x)),  r = (mean(x^2) + eps)^(-1/2),      dw = sum over the rows of g x r.
//
// The angle.  A position times a frequency is needed modulo a turn only, so the frequency is kept as a 64-bit fraction of a turn and the
// product taken modulo 2^64 and rounded to 2^-32 turns: off by 2^-33 turns, and 2^-34 for the frequency, at every 32-bit position (an fp32
// product is off by 0.004 radian at position 70 000).  Sine and cosine are Taylor polynomials on an eighth of a turn to either side
// (error < 2^-24), once a token and pair: a workgroup puts them in LDS and all heads of its tokens read them there.
//
// Bound: bytes.  Every row is read once and written once (backward: x and dy once, dx once); a row of 16 * U channels is held by
// 2^ceil(log2 U) neighbouring lanes, 16 channels a lane, so the mean is log2 lane exchanges and nothing is staged.
#include <type_traits>

#include "bank4.h"

namespace mivos {

struct RotaryRows {
  const void *x, *g;
  void *y;
  const float *weight;
  int64_t xb, xn, xh, gb, gn, gh;
  int heads;
  uint32_t magic;     // row / heads = the high word of row * magic for rows of a tile (row * heads < 2^32)
};
struct RotaryArgs {
  RotaryRows rows[2];
  const int32_t *pos;
  int64_t pb, pn, pa;
  const uint64_t *freq;
  const int32_t *axis;
  float *partial;                     // backward: a share of a weight gradient a row of dim, `split` rows of q_weight's, then k_weight's
  int batch, tokens, dim, pairs, interleaved, norm, tile, n_tiles, split;
  float eps, sign;
};

// sine and cosine of pos * freq turns (freq in 2^-64 turns)
__device__ __forceinline__ void turn_sincos(int32_t pos, uint64_t freq, float sign, float &s, float &c) {
  const uint32_t turn = (uint32_t)(((uint64_t)(int64_t)pos * freq + 0x80000000u) >> 32);      // (rounded to 2^-32 turns)
  const uint32_t quarter = (turn + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(turn - (quarter << 30)) * 1.4629180792671596e-9f;      // 2 pi / 2^32: [-pi/4, pi/4)
  const float z = x * x;
  const float sx = x * (1.f + z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880)))));
  const float cx = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
  float sn = quarter & 1 ? cx : sx, cs = quarter & 1 ? sx : cx;
  if (quarter & 2) sn = -sn;
  if ((quarter + 1) & 2) cs = -cs;
  s = sign * sn;
  c = cs;
}

// ------------------------------------------------------------------------------------------ any width, any alignment: one wave a row
// Lane l holds channels l, l + 64, ...; dim <= 512.  Every channel computes its own sine and cosine and loads are 2 or 4 bytes a lane: bound by
// instructions, 638 us (norm) and 1340 (gradient) for 32 400 tokens x 20 heads of 128 channels, bf16, where the rows below take 68 and 135.
template <typename T, bool GRAD>
__global__ __launch_bounds__(256) void rotary_any_kernel(RotaryArgs a) {
  __shared__ float dw[4][2][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per_token = a.rows[0].heads + a.rows[1].heads;
  const int64_t total = (int64_t)a.batch * a.tokens * per_token;
  float acc[2][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[0][j] = acc[1][j] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < total; row += (int64_t)gridDim.x * 4) {
    const int64_t bn = row / per_token;
    int h = (int)(row - bn * per_token);
    const int b = (int)(bn / a.tokens), n = (int)(bn - (int64_t)b * a.tokens), which = h >= a.rows[0].heads;
    if (which) h -= a.rows[0].heads;
    const RotaryRows &R = a.rows[which];
    const T *x = (const T *)R.x + b * R.xb + n * R.xn + h * R.xh;
    const T *g = GRAD ? (const T *)R.g + b * R.gb + n * R.gn + h * R.gh : x;
    float xs[8], ps[8], sn[8], cs[8], ss = 0.f;      // own channel of the rotated operand, its partner's, and the turn
    const T *rot = GRAD ? g : x;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = lane + 64 * j;
      xs[j] = ps[j] = sn[j] = 0.f;
      cs[j] = 1.f;
      if (c >= a.dim) continue;
      xs[j] = (float)rot[c];
      if (c < 2 * a.pairs) {
        const int i = a.interleaved ? c >> 1 : c < a.pairs ? c : c - a.pairs;
        const bool second = a.interleaved ? c & 1 : c >= a.pairs;
        const int partner = a.interleaved ? c ^ 1 : second ? c - a.pairs : c + a.pairs;
        ps[j] = (float)rot[partner];
        if (a.norm && !GRAD) { ps[j] *= R.weight[partner]; }
        turn_sincos(a.pos[b * a.pb + n * a.pn + a.axis[i] * a.pa], a.freq[i], second ? a.sign : -a.sign, sn[j], cs[j]);
      }
      ss += xs[j] * xs[j];
    }
    float r = 1.f;
    if (a.norm && !GRAD) {
      for (int d = 1; d < 64; d <<= 1) ss += __shfl_xor(ss, d);
      r = 1.f / sqrtf(ss / a.dim + a.eps);
    }
    T *y = (T *)R.y + ((int64_t)bn * R.heads + h) * a.dim;
    if constexpr (!GRAD) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = lane + 64 * j;
        if (c < a.dim) y[c] = (T)(r * ((a.norm ? xs[j] * R.weight[c] : xs[j]) * cs[j] + ps[j] * sn[j]));
      }
    } else {
      float xx[8], gw[8], dot = 0.f;
      ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = lane + 64 * j;
        xx[j] = gw[j] = 0.f;
        if (c >= a.dim) continue;
        xx[j] = (float)x[c];
        xs[j] = xs[j] * cs[j] + ps[j] * sn[j];       // g
        gw[j] = xs[j] * R.weight[c];
        ss += xx[j] * xx[j];
        dot += gw[j] * xx[j];
      }
      for (int d = 1; d < 64; d <<= 1) { ss += __shfl_xor(ss, d); dot += __shfl_xor(dot, d); }
      r = 1.f / sqrtf(ss / a.dim + a.eps);
      const float k = r * r * dot / a.dim;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = lane + 64 * j;
        if (c < a.dim) y[c] = (T)(r * (gw[j] - xx[j] * k));
        if (which) acc[1][j] += xs[j] * xx[j] * r;
        else acc[0][j] += xs[j] * xx[j] * r;
      }
    }
  }
  if constexpr (GRAD) {
#pragma unroll
    for (int j = 0; j < 8; ++j) { dw[wave][0][lane + 64 * j] = acc[0][j]; dw[wave][1][lane + 64 * j] = acc[1][j]; }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.dim; i += 256) {
      const int w = i / a.dim, c = i - w * a.dim;
      a.partial[((int64_t)w * gridDim.x + blockIdx.x) * a.dim + c] = dw[0][w][c] + dw[1][w][c] + dw[2][w][c] + dw[3][w][c];
    }
  }
}

// ------------------------------------------------------------------------------------------ 16 channels a lane
// A lane's unit: 8 pairs (two runs of 8 channels `pairs` apart, or 16 neighbours), or 16 channels behind the pairs.
template <bool INTER>
__device__ __forceinline__ void unit_channels(int u, int pairs, int &c0, int &c1, bool &rot) {
  rot = 8 * u < pairs;
  if (rot && !INTER) { c0 = 8 * u; c1 = pairs + 8 * u; }
  else { c0 = 16 * u; c1 = 16 * u + 8; }
}
// rotates the unit (lo, hi) by the table's angles
template <bool INTER>
__device__ __forceinline__ void unit_turn(f32x8 &lo, f32x8 &hi, const f32x2 *cs) {
  f32x8 ol, oh;
  if constexpr (INTER) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 e = cs[j], f = cs[4 + j];
      ol[2 * j] = lo[2 * j] * e.x - lo[2 * j + 1] * e.y;
      ol[2 * j + 1] = lo[2 * j + 1] * e.x + lo[2 * j] * e.y;
      oh[2 * j] = hi[2 * j] * f.x - hi[2 * j + 1] * f.y;
      oh[2 * j + 1] = hi[2 * j + 1] * f.x + hi[2 * j] * f.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const f32x2 e = cs[j];
      ol[j] = lo[j] * e.x - hi[j] * e.y;
      oh[j] = hi[j] * e.x + lo[j] * e.y;
    }
  }
  lo = ol;
  hi = oh;
}

// x summed over a row's lanes (neighbours, a power of two): lane permutations inside the 16 lanes of a row, no LDS round trip
__device__ __forceinline__ float lanes_sum(float x, int lanes) {
  auto add = [&](auto ctrl) { x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true)); };
  if (lanes >= 2) add(std::integral_constant<int, 0xb1>{});      // neighbours
  if (lanes >= 4) add(std::integral_constant<int, 0x4e>{});      // pairs of a quad
  if (lanes >= 8) add(std::integral_constant<int, 0x141>{});     // half row mirrored: the other quad
  if (lanes >= 16) add(std::integral_constant<int, 0x140>{});    // row mirrored: the other eight
  if (lanes >= 32) x += __shfl_xor(x, 16);
  return x;
}

// A workgroup's tokens in tiles: the tile's sines and cosines in LDS once, then the rows of its queries and of its keys, `slots` at a time; the
// next row is fetched while one is worked on, the first ones while the table is built.  Backward: the first `a.split` workgroups take the queries,
// the others the keys (one set of weights and sums in registers, so that three workgroups fit a CU: 61 -> 58 us at 16 200 tokens x 20 heads x 128).
template <typename T, bool INTER, bool NORM, bool GRAD>
__global__ __launch_bounds__(256, GRAD || sizeof(T) == 4 ? 3 : 4) void rotary_rows_kernel(RotaryArgs a, int lanes /* a row, a power of two */) {
  extern __shared__ __align__(16) f32x2 table[];     // [tile][pairs] (cos, sin); backward: the weight gradients afterwards
  const int tid = threadIdx.x, units = a.dim / 16, slots = 256 / lanes, u = tid & (lanes - 1), row0 = tid / lanes;
  int c0, c1;
  bool rot;
  unit_channels<INTER>(u, a.pairs, c0, c1, rot);
  const bool live = u < units;
  constexpr int KINDS = GRAD ? 1 : 2;                // operands a workgroup works on: rows[kind0], rows[kind0 + 1], ...
  const int kind0 = GRAD ? blockIdx.x >= a.split : 0, group = GRAD && kind0 ? blockIdx.x - a.split : blockIdx.x;
  const int groups = !GRAD ? gridDim.x : kind0 ? gridDim.x - a.split : a.split;
  f32x8 acc0, acc1, w[KINDS][2];
  if constexpr (NORM || GRAD) {
#pragma unroll
    for (int k = 0; k < KINDS; ++k)
      if (live && a.rows[kind0 + k].heads) {
        w[k][0] = load8(a.rows[kind0 + k].weight + c0, false);
        w[k][1] = load8(a.rows[kind0 + k].weight + c1, false);
      }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) acc0[j] = acc1[j] = 0.f;

  struct Row { u32x4 v[GRAD ? 4 : 2][sizeof(T) / 2]; int t, h; };      // as they lie in memory: x | x, or dy | dy | x | x
  auto take = [&](Row &f, int i, const T *p) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) f.v[i][j] = reinterpret_cast<const u32x4 *>(p)[j];
  };
  auto wide = [&](const Row &f, int i) { return load8(reinterpret_cast<const T *>(f.v[i]), true); };
  for (int tile = group; tile < a.n_tiles; tile += groups) {
    const uint32_t first = (uint32_t)tile * a.tile, all = (uint32_t)a.batch * a.tokens;       // at most 2^30 tokens
    const int n_tok = (int)(all - first < (uint32_t)a.tile ? all - first : a.tile);
    const uint32_t b0 = first / a.tokens, n0 = first - b0 * a.tokens;
    auto place = [&](int t, uint32_t &b, uint32_t &n) {
      b = b0;
      n = n0 + t;
      if (n >= (uint32_t)a.tokens) { const uint32_t q = n / a.tokens; b += q; n -= q * a.tokens; }
    };
    auto fetch = [&](Row &f, const RotaryRows &R, int row) {
      f.t = R.heads == 1 ? row : (int)__umulhi((uint32_t)row, R.magic);       // row / heads
      f.h = row - f.t * R.heads;
#pragma unroll
      for (int i = 0; i < (GRAD ? 4 : 2); ++i)
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) f.v[i][j] = u32x4{0u, 0u, 0u, 0u};
      if (!live || row >= n_tok * R.heads) return;
      uint32_t b, n;
      place(f.t, b, n);
      const T *x = (const T *)R.x + b * R.xb + n * R.xn + f.h * R.xh;
      if constexpr (GRAD) {
        const T *g = (const T *)R.g + b * R.gb + n * R.gn + f.h * R.gh;
        take(f, 0, g + c0);
        take(f, 1, g + c1);
        take(f, 2, x + c0);
        take(f, 3, x + c1);
      } else {
        take(f, 0, x + c0);
        take(f, 1, x + c1);
      }
    };
    Row now, next;
    fetch(next, a.rows[kind0], row0);
    __syncthreads();
    for (int e = tid; e < n_tok * a.pairs; e += 256) {
      const int t = e / a.pairs, i = e - t * a.pairs;
      uint32_t b, n;
      place(t, b, n);
      float s, c;
      turn_sincos(a.pos[b * a.pb + n * a.pn + a.axis[i] * a.pa], a.freq[i], a.sign, s, c);
      table[t * a.pairs + i] = f32x2{c, s};
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KINDS; ++k) {
      const RotaryRows &R = a.rows[kind0 + k];
      const int n_rows = n_tok * R.heads;
      for (int row = row0; row < n_rows; row += slots) {
        now = next;
        if (row + slots < n_rows) fetch(next, R, row + slots);
        else if (k + 1 < KINDS) fetch(next, a.rows[1], row0);
        f32x8 lo = wide(now, 0), hi = wide(now, 1);
        if constexpr (NORM) {
          float ss = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) ss += lo[j] * lo[j] + hi[j] * hi[j];
          ss = lanes_sum(ss, lanes);
          const float r = 1.f / sqrtf(ss / a.dim + a.eps);
          lo *= r * w[k][0];
          hi *= r * w[k][1];
        }
        if (rot && live) unit_turn<INTER>(lo, hi, table + now.t * a.pairs + 8 * u);
        if constexpr (GRAD) {
          const f32x8 gl = lo * w[k][0], gh = hi * w[k][1], xl = wide(now, 2), xh = wide(now, 3);
          float ss = 0.f, dot = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            ss += xl[j] * xl[j] + xh[j] * xh[j];
            dot += live ? gl[j] * xl[j] + gh[j] * xh[j] : 0.f;
          }
          ss = lanes_sum(ss, lanes);
          dot = lanes_sum(dot, lanes);
          const float r = 1.f / sqrtf(ss / a.dim + a.eps), q = r * r * dot / a.dim;
          acc0 += lo * xl * r;
          acc1 += hi * xh * r;
          lo = r * (gl - xl * q);
          hi = r * (gh - xh * q);
        }
        if (live) {
          T *y = (T *)R.y + ((int64_t)(first + now.t) * R.heads + now.h) * a.dim;
          store8(y + c0, lo);
          store8(y + c1, hi);
        }
      }
      if (k + 1 < KINDS && row0 >= n_rows) fetch(next, a.rows[1], row0);      // (a slot without a query row)
    }
  }
  if constexpr (GRAD) {                               // the workgroup's share of its weight gradient, its row slots in order
    float *dw = reinterpret_cast<float *>(table);     // [slots][16 * lanes]
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) { dw[tid * 16 + j] = acc0[j]; dw[tid * 16 + 8 + j] = acc1[j]; }
    __syncthreads();
    for (int i = tid; i < units * 16; i += 256) {
      int d0, d1;
      bool r2;
      unit_channels<INTER>(i / 16, a.pairs, d0, d1, r2);
      const int c = (i & 8 ? d1 : d0) + (i & 7);
      float sum = 0.f;
      for (int s = 0; s < slots; ++s) sum += dw[s * 16 * lanes + i];
      a.partial[(int64_t)blockIdx.x * a.dim + c] = sum;
    }
  }
}

// dw[k][c] = the shares of workgroups [k ? split : 0, k ? groups : split) in order: 16 columns a workgroup, 16 runs of shares each
__global__ __launch_bounds__(256) void rotary_weight_sum_kernel(const float *__restrict__ partial, int split, int groups, int dim, float *dq, float *dk) {
  __shared__ float part[16][17];
  const int k = blockIdx.y, col = blockIdx.x * 16 + (threadIdx.x & 15), run = threadIdx.x >> 4;
  const int first = k ? split : 0, end = k ? groups : split, per = (end - first + 15) / 16, g0 = first + run * per, g1 = g0 + per < end ? g0 + per : end;
  float sum = 0.f;
  if (col < dim)
#pragma unroll 16
    for (int g = g0; g < g1; ++g) sum += partial[(int64_t)g * dim + col];
  part[run][threadIdx.x & 15] = sum;
  __syncthreads();
  if (run == 0 && col < dim) {
    float t = 0.f;
    for (int r = 0; r < 16; ++r) t += part[r][threadIdx.x];
    (k ? dk : dq)[col] = t;
  }
}

constexpr int ROTARY_GRAD_GROUPS = 1024;   // workgroups of a backward launch (4 a CU); their shares are 2 * dim floats each

struct RotaryPlan {
  bool rows;            // 16 channels a lane (else one wave a row)
  int lanes, grid, groups;      // groups: shares of the weight gradients
  size_t lds;
};

static int rotary_plan(const mivos_rotary *d, RotaryArgs *a, RotaryPlan *p, bool grad) {
  const int es = dtype_bytes(d->dtype);
  uintptr_t bits = 0;
  for (int k = 0; k < 2; ++k) {
    const mivos_rotary_rows &r = d->rows[k];
    a->rows[k] = RotaryRows{r.x, r.g, r.y, r.weight, r.xb, r.xn, r.xh, r.gb, r.gn, r.gh, r.heads, r.heads > 1 ? 0xffffffffu / (uint32_t)r.heads + 1 : 0};
    if (!r.heads) continue;
    bits |= (uintptr_t)r.x | (uintptr_t)r.y | (uintptr_t)((r.xb | r.xn | r.xh) * es);
    if (grad) bits |= (uintptr_t)r.g | (uintptr_t)((r.gb | r.gn | r.gh) * es);
  }
  a->pos = d->positions; a->pb = d->pb; a->pn = d->pn; a->pa = d->pa;
  a->freq = d->freq; a->axis = d->axis; a->partial = (float *)d->workspace;
  a->batch = d->batch; a->tokens = d->tokens; a->dim = d->dim; a->pairs = d->pairs; a->interleaved = d->interleaved;
  a->norm = grad || d->eps >= 0.f; a->eps = d->eps; a->sign = d->inverse ? -1.f : 1.f;
  const int64_t all = (int64_t)d->batch * d->tokens;
  p->rows = (bits & 15) == 0 && d->dim % 16 == 0 && d->pairs % 8 == 0 && d->dim <= 512;
  if (p->rows) {
    p->lanes = 1;
    while (p->lanes < d->dim / 16) p->lanes *= 2;
    int64_t tile = all / 1024;                            // tokens a workgroup: enough workgroups first, then more heads on one table
    tile = tile < 1 ? 1 : tile > 16 ? 16 : tile;
    a->tile = (int)tile;
    a->n_tiles = (int)((all + tile - 1) / tile);
    p->lds = (size_t)tile * d->pairs * 8;
    if (grad && p->lds < 256 * 16 * 4) p->lds = 256 * 16 * 4;
    p->grid = a->n_tiles;
    if (!grad && p->grid > (1 << 20)) p->grid = 1 << 20;
    if (grad) {                                           // shared out by their heads
      const int hq = d->rows[0].heads, hk = d->rows[1].heads, most = ROTARY_GRAD_GROUPS;
      const int gq = hk ? (int)((int64_t)most * hq / (hq + hk)) : most, gk = most - gq;
      a->split = gq < 1 ? 1 : gq < a->n_tiles ? gq : a->n_tiles;
      p->groups = a->split + (hk ? (gk < 1 ? 1 : gk < a->n_tiles ? gk : a->n_tiles) : 0);
      p->grid = p->groups;
    }
  } else {
    const int64_t rows = all * (d->rows[0].heads + d->rows[1].heads);
    const int64_t most = grad ? ROTARY_GRAD_GROUPS : 256 * 64;
    p->grid = (int)((rows + 3) / 4 < most ? (rows + 3) / 4 : most);
    a->split = p->grid;
    p->groups = 2 * p->grid;
  }
  return MIVOS_OK;
}

static int rotary_check(const mivos_rotary *d, bool grad, const char *what) {
  if (!d || !dtype_ok(d->dtype) || d->batch < 0 || d->tokens < 0 || d->dim < 2 || d->dim > 512 || d->pairs < 1 || 2 * d->pairs > d->dim || !d->freq || !d->axis)
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "%s: bad shape (rows of 2 to 512 channels, at most half as many pairs)", what);
  if ((int64_t)d->batch * d->tokens > (1ll << 30)) return fail(MIVOS_ERR_INVALID_ARGUMENT, "%s: too many tokens", what);
  if ((int64_t)d->batch * d->tokens == 0) return MIVOS_OK;
  if (!d->positions) return fail(MIVOS_ERR_INVALID_ARGUMENT, "%s: null positions", what);
  for (int k = 0; k < 2; ++k) {
    const mivos_rotary_rows &r = d->rows[k];
    if (r.heads < 0 || r.heads > 4096 || (k == 0 && r.heads == 0)) return fail(MIVOS_ERR_INVALID_ARGUMENT, "%s: %d heads", what, r.heads);
    if (r.heads && (!r.x || !r.y || (grad && !r.g) || ((grad || d->eps >= 0.f) && !r.weight))) return fail(MIVOS_ERR_INVALID_ARGUMENT, "%s: null rows", what);
  }
  return MIVOS_OK;
}

template <typename T, bool GRAD>
static void rotary_launch(const RotaryArgs &a, const RotaryPlan &p, hipStream_t s) {
  if (!p.rows) { rotary_any_kernel<T, GRAD><<<p.grid, 256, 0, s>>>(a); return; }
  if constexpr (GRAD) {
    if (a.interleaved) rotary_rows_kernel<T, true, false, true><<<p.grid, 256, p.lds, s>>>(a, p.lanes);
    else rotary_rows_kernel<T, false, false, true><<<p.grid, 256, p.lds, s>>>(a, p.lanes);
  } else if (a.norm) {
    if (a.interleaved) rotary_rows_kernel<T, true, true, false><<<p.grid, 256, p.lds, s>>>(a, p.lanes);
    else rotary_rows_kernel<T, false, true, false><<<p.grid, 256, p.lds, s>>>(a, p.lanes);
  } else {
    if (a.interleaved) rotary_rows_kernel<T, true, false, false><<<p.grid, 256, p.lds, s>>>(a, p.lanes);
    else rotary_rows_kernel<T, false, false, false><<<p.grid, 256, p.lds, s>>>(a, p.lanes);
  }
}

}  // namespace mivos

using namespace mivos;

extern "C" int mivos_rotary_axes(const mivos_rotary *d, void *stream) {
  if (int rc = rotary_check(d, false, "rotary_axes")) return rc;
  if ((int64_t)d->batch * d->tokens == 0) return MIVOS_OK;
  RotaryArgs a{};
  RotaryPlan p{};
  rotary_plan(d, &a, &p, false);
  hipStream_t s = (hipStream_t)stream;
  if (d->dtype == MIVOS_F32) rotary_launch<float, false>(a, p, s);
  else if (d->dtype == MIVOS_F16) rotary_launch<_Float16, false>(a, p, s);
  else rotary_launch<__bf16, false>(a, p, s);
  return check_launch("rotary_axes");
}

extern "C" int64_t mivos_norm_rotary_grad_workspace_bytes(int dim) { return ((int64_t)ROTARY_GRAD_GROUPS + 1) * 2 * dim * 4; }

extern "C" int mivos_norm_rotary_grad(const mivos_rotary *d, float *dq_weight, float *dk_weight, void *stream) {
  if (int rc = rotary_check(d, true, "norm_rotary_grad")) return rc;
  if (d->eps < 0.f || !dq_weight || (d->rows[1].heads && !dk_weight)) return fail(MIVOS_ERR_INVALID_ARGUMENT, "norm_rotary_grad: bad argument");
  hipStream_t s = (hipStream_t)stream;
  RotaryArgs a{};
  RotaryPlan p{};
  if ((int64_t)d->batch * d->tokens) {
    if (!d->workspace || d->workspace_bytes < mivos_norm_rotary_grad_workspace_bytes(d->dim)) return fail(MIVOS_ERR_INVALID_ARGUMENT, "norm_rotary_grad: workspace");
    rotary_plan(d, &a, &p, true);
    if (d->dtype == MIVOS_F32) rotary_launch<float, true>(a, p, s);
    else if (d->dtype == MIVOS_F16) rotary_launch<_Float16, true>(a, p, s);
    else rotary_launch<__bf16, true>(a, p, s);
  }
  rotary_weight_sum_kernel<<<dim3(cdiv(d->dim, 16), dk_weight ? 2 : 1), 256, 0, s>>>(a.partial, a.split, p.groups, d->dim, dq_weight, dk_weight);
  return check_launch("norm_rotary_grad");
}
