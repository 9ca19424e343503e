// Memory bank in 4 bits: append (quantise + store), values (read back), evict (keep the slots with the most attention weight).
// All three move bytes: append reads a row once and writes 17/64 of its bf16 size, values the reverse, evict reads 4 bytes a slot for the
// choice and moves the kept rows once.  The attention read over the bank is bank4_read.hip.
#include "bank4.h"

namespace mivos {

// ---------------------------------------------------------------------------------------------- append
// One thread quantises 8 channels, four neighbours make up a block of 32: they share the block's largest magnitude by two lane
// exchanges, so a row is read once and nothing is staged.  scale = the smallest power of two 2^e with max |x| <= 6 * 2^e: nothing
// saturates (the floor(log2) rule of the microscaling formats clips up to a quarter off a block's largest value).  A workgroup's threads
// keep their place in the row; rows (token, head) go by 256 / units.  13 us for 8160 x 3 fp32 rows of 640 channels (5.3 TB/s; two and four rows in
// flight a thread: 15 and 16).
template <typename T>
__global__ __launch_bounds__(256) void bank4_append_kernel(mivos_bank4 bank, const T *__restrict__ keys, int64_t kb, int64_t kt, int64_t kh,
                                                           const T *__restrict__ values, int64_t vb, int64_t vt, int64_t vh, int vec,
                                                           const int32_t *at, const int32_t *__restrict__ count, int tokens, int units) {
  const int b = blockIdx.y, rows = 256 / units, r = threadIdx.x / units;       // units = (key_dim + value_dim) / 8, a multiple of 4
  int u = threadIdx.x - r * units;
  const int64_t start = at[b];
  int n = count ? count[b] : tokens;
  n = n < 0 ? 0 : n > tokens ? tokens : n;
  const int ku = bank.key_dim / 8;
  const bool is_key = u < ku, first = u == 0;
  u = is_key ? u : u - ku;
  const T *src = (is_key ? keys + b * kb : values + b * vb) + u * 8;
  const int64_t st = is_key ? kt : vt, sh = is_key ? kh : vh;
  const int dim = is_key ? bank.key_dim : bank.value_dim;
  uint32_t *codes = reinterpret_cast<uint32_t *>(is_key ? bank.key_codes : bank.value_codes) + u;
  uint8_t *scales = (is_key ? bank.key_scales : bank.value_scales) + (u >> 2);
  const uint32_t total = (uint32_t)n * bank.heads;
  bool lost = false;
  for (uint32_t i = blockIdx.x * rows + r; r < rows && i < total; i += gridDim.x * rows) {
    const uint32_t t = i / (uint32_t)bank.heads, h = i - t * bank.heads;
    const int64_t slot = start + t;
    if (slot < 0 || slot >= bank.slots) { lost = true; continue; }      // (the four lanes of a block share the branch)
    const int64_t row = ((int64_t)b * bank.heads + h) * bank.slots + slot;
    const f32x8 x = load8(src + t * st + h * sh, vec);
    if (first) bank.weight[row] = 0.f;
    float top = 0.f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float m = __builtin_fabsf(x[j]);
      bad |= !(m < INFINITY);
      top = fmaxf(top, m);
    }
    if (bad) top = INFINITY;
    top = fmaxf(top, __shfl_xor(top, 1, 4));
    top = fmaxf(top, __shfl_xor(top, 2, 4));
    const uint32_t bits = __float_as_uint(top);
    // top = 1.f * 2^(E - 127): the smallest e with top <= 6 * 2^e = 1.5 * 2^(e + 2) is E - 129, one more where 1.f > 1.5
    int e = (int)(bits >> 23) - 129 + ((bits & 0x7fffffu) > 0x400000u);
    e = e < -120 ? -120 : e > 125 ? 125 : e;
    uint32_t packed = 0, byte = kBank4NanScale;
    if (top < INFINITY) {
      byte = (uint32_t)(e + 127);
      const float scale = __uint_as_float(byte << 23);
      packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, x[0], x[1], scale, 0);
      packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, x[2], x[3], scale, 1);
      packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, x[4], x[5], scale, 2);
      packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, x[6], x[7], scale, 3);
    }
    codes[row * (dim / 8)] = packed;
    if ((u & 3) == 0) scales[row * (dim / 32)] = (uint8_t)byte;
  }
  if (lost) atomicOr(reinterpret_cast<unsigned int *>(bank.status), 1u);
  // the new length; where `at` is the length itself, the last workgroup of the stream to have read it writes it
  int64_t end = start + n;
  end = end < 0 ? 0 : end > bank.slots ? bank.slots : end;
  if (at != bank.lens) {
    if (blockIdx.x == 0 && threadIdx.x == 0) bank.lens[b] = (int32_t)end;
    return;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const int32_t seen = atomicAdd(bank.status + 1 + b, 1);
    if (seen == (int32_t)gridDim.x - 1) {
      bank.status[1 + b] = 0;
      bank.lens[b] = (int32_t)end;
    }
  }
}

// ---------------------------------------------------------------------------------------------- values
// Rows as in append, four in flight a thread: 84 us for 32 x 24 576 rows of 256 channels to bf16 (6.1 TB/s,
// nine tenths of it written; one in flight: 131).
constexpr int VALUES_DEEP = 4;

template <typename T>
__global__ __launch_bounds__(256) void bank4_values_kernel(mivos_bank4 bank, const int32_t *__restrict__ first, int count, T *__restrict__ key_out,
                                                           T *__restrict__ value_out) {
  const int bh = blockIdx.y, b = bh / bank.heads;
  const int ku = bank.key_dim / 8, units = ku + bank.value_dim / 8, rows = 256 / units, r = threadIdx.x / units;
  if (r >= rows) return;
  int u = threadIdx.x - r * units;
  const bool is_key = u < ku;
  u = is_key ? u : u - ku;
  const int dim = is_key ? bank.key_dim : bank.value_dim;
  const int64_t start = first ? first[b] : 0;
  int64_t len = bank.lens[b];
  len = len > bank.slots ? bank.slots : len;
  const uint32_t *codes = reinterpret_cast<const uint32_t *>(is_key ? bank.key_codes : bank.value_codes) + (int64_t)bh * bank.slots * (dim / 8) + u;
  const uint8_t *scales = (is_key ? bank.key_scales : bank.value_scales) + (int64_t)bh * bank.slots * (dim / 32) + (u >> 2);
  T *out = (is_key ? key_out : value_out) + (int64_t)bh * count * dim + u * 8;
  for (int64_t j0 = (int64_t)blockIdx.x * VALUES_DEEP * rows + r; j0 < count; j0 += (int64_t)gridDim.x * VALUES_DEEP * rows) {
    uint32_t c[VALUES_DEEP], s[VALUES_DEEP];
#pragma unroll
    for (int k = 0; k < VALUES_DEEP; ++k) {
      const int64_t slot = start + j0 + k * rows;
      c[k] = 0u;
      s[k] = 127u;
      if (slot >= 0 && slot < len) { c[k] = codes[slot * (dim / 8)]; s[k] = scales[slot * (dim / 32)]; }
    }
#pragma unroll
    for (int k = 0; k < VALUES_DEEP; ++k) {
      if (j0 + k * rows >= count) break;
      const bf16x8 w = bank4_unpack8(c[k], bank4_scale(s[k]));
      if constexpr (sizeof(T) == 2) *reinterpret_cast<bf16x8 *>(out + (j0 + k * rows) * dim) = w;
      else {
        f32x8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)w[i];
        store8(out + (j0 + k * rows) * dim, v);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- evict
// Order of the weights as unsigned integers: larger weight, larger key; NaN lowest; -0 = +0.  From 1 (NaN) to 0xff800000 (infinity): 0 is left
// for what is no slot, KEY_STAYS for what is protected.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 1u;
  const uint32_t b = __float_as_uint(w + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t KEY_STAYS = 0xffffffffu;

constexpr int EVICT_THREADS = 1024, EVICT_WAVES = EVICT_THREADS / 64, EVICT_BINS = 2048, EVICT_COPIES = 4;
// Keys a lane holds: banks of up to 32 768 slots are read once, larger ones again in each pass (a call that keeps 64 rows: 32 768 slots 21 us, 32 769
// 42, 100 000 104, 400 000 377).
constexpr int EVICT_KEYS = 32;

__device__ __forceinline__ uint32_t waves_before(const uint32_t *v, int wave) {      // the sum over the waves before, all 16 read at once
  uint32_t sum = 0;
#pragma unroll
  for (int i = 0; i < EVICT_WAVES / 4; ++i) {
    const u32x4 x = reinterpret_cast<const u32x4 *>(v)[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += 4 * i + j < wave ? x[j] : 0u;
  }
  return sum;
}

// Which slots of one (stream, head) stay: a radix select of the keep-th largest key (protected slots have the largest), 11 + 11 + 10 bits, the
// counts in LDS (four of each bin, by lane: most weights of a bank share a few exponents, and increments of one address are serial; one of each
// takes 20 us instead of 18, the keys in LDS instead of registers no less), then one ordered pass that writes the kept slots ascending.  Equal weights: the lowest slots stay.  A wave owns a run of slots, so a slot's place follows from ballots
// of its wave and one sum over the waves before: (larger keys before it) + min(equal ones before it, equal ones that stay).
// One workgroup a (stream, head): bound by latency, 12 barriers and three passes of LDS counts (18 us at 21 060 slots; slots visited one
// 1024-wide row at a time with a scan each, and 8-bit digits, took 49 us).
template <bool REGS>
__global__ __launch_bounds__(EVICT_THREADS) void bank4_select_kernel(const float *__restrict__ weight, const int32_t *__restrict__ lens, int heads, int64_t slots,
                                                                    int keep, int first, int recent, int32_t *__restrict__ slots_out,
                                                                    int32_t *__restrict__ lens_out) {
  __shared__ __align__(16) uint32_t hist[EVICT_BINS][EVICT_COPIES];
  __shared__ uint32_t chosen[2];
  __shared__ __align__(16) uint32_t sums[EVICT_WAVES], larger[EVICT_WAVES], equal[EVICT_WAVES];
  const int bh = blockIdx.x, b = bh / heads, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t n64 = lens[b];
  const int n = (int)(n64 < 0 ? 0 : n64 > slots ? slots : n64);
  const float *w = weight + (int64_t)bh * slots;
  int32_t *out = slots_out + (int64_t)bh * keep;
  const int fresh = n < keep ? n : keep;
  if (tid == 0 && bh % heads == 0) lens_out[b] = fresh;
  if (n <= keep) {
    for (int i = tid; i < keep; i += EVICT_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const int hi = n - recent;                                         // slots [0, first) and [hi, n) are protected; first + recent <= keep < n
  int want = keep;
  const int rounds = (n + EVICT_THREADS - 1) / EVICT_THREADS, run = rounds * 64, base = wave * run + lane;     // the wave's slots: base + 64 j, j < rounds
  uint32_t held[REGS ? EVICT_KEYS : 1];
  auto slot_weight = [&](int j) { const int i = base + j * 64; return w[i < n ? i : n - 1]; };      // (no branch: all loads go out together)
  auto slot_key = [&](int j, float x) {
    const int i = base + j * 64;
    return i >= n ? 0u : i < first || i >= hi ? KEY_STAYS : weight_key(x);
  };
  if constexpr (REGS) {
    float x[EVICT_KEYS];
#pragma unroll
    for (int j = 0; j < EVICT_KEYS; ++j) x[j] = slot_weight(j < rounds ? j : 0);
#pragma unroll
    for (int j = 0; j < EVICT_KEYS; ++j) held[j] = slot_key(j, x[j]);
  }
  auto each = [&](auto &&use) {      // use(slot, key) for the wave's slots in order; every lane takes part in every call
    if constexpr (REGS) {
#pragma unroll
      for (int j = 0; j < EVICT_KEYS; ++j)
        if (j < rounds) use(base + j * 64, held[j]);
    } else {
      for (int j = 0; j < rounds; j += 8) {
        float x[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) x[c] = slot_weight(j + c < rounds ? j + c : 0);
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (j + c < rounds) use(base + (j + c) * 64, slot_key(j + c, x[c]));
      }
    }
  };
  uint32_t prefix = 0, mask = 0;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < EVICT_BINS; i += EVICT_THREADS) *reinterpret_cast<u32x4 *>(hist[i]) = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    each([&](int i, uint32_t k) {
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)][lane % EVICT_COPIES], 1u);
    });
    __syncthreads();
    // thread t: bins 2 t, 2 t + 1 counted from the top
    uint32_t c[2], sum = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int bin = bins - 1 - (2 * tid + j);
      const u32x4 v = *reinterpret_cast<const u32x4 *>(hist[bin >= 0 ? bin : 0]);
      c[j] = bin >= 0 ? v[0] + v[1] + v[2] + v[3] : 0u;
      sum += c[j];
    }
    uint32_t before = sum;
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(before, d);
      if (lane >= d) before += o;
    }
    if (lane == 63) sums[wave] = before;
    __syncthreads();
    before += waves_before(sums, wave) - sum;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (before < (uint32_t)want && (uint32_t)want <= before + c[j]) { chosen[0] = bins - 1 - (2 * tid + j); chosen[1] = before; }
      before += c[j];
    }
    __syncthreads();
    prefix |= chosen[0] << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    want -= (int)chosen[1];
  }
  // now: keys above `prefix` stay, and the first `want` of those equal to it
  int n_larger = 0, n_equal = 0;
  each([&](int, uint32_t k) {
    n_larger += __popcll(__ballot(k > prefix));
    n_equal += __popcll(__ballot(k == prefix));
  });
  if (lane == 0) { larger[wave] = n_larger; equal[wave] = n_equal; }
  __syncthreads();
  n_larger = (int)waves_before(larger, wave);
  n_equal = (int)waves_before(equal, wave);
  each([&](int i, uint32_t k) {
    const uint64_t ba = __ballot(k > prefix), bt = __ballot(k == prefix);
    const int ties = n_equal + __builtin_amdgcn_mbcnt_hi((uint32_t)(bt >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bt, 0));
    const int place = n_larger + __builtin_amdgcn_mbcnt_hi((uint32_t)(ba >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ba, 0)) + (ties < want ? ties : want);
    if (k > prefix || (k == prefix && ties < want)) out[place] = i;
    n_larger += __popcll(ba);
    n_equal += __popcll(bt);
  });
}

// Moves the kept rows: a thread a block of 32 channels, 16 bytes of codes; every fourth the scales of four blocks (WIDE: both rows have a
// multiple of 128 channels; else each its own), the first the weight.  56 us for 32 x 24 576 of 32 768 rows of 256 channels
// (3.9 TB/s of what is kept; stores among the loads: 67; a second row in flight a thread gains nothing).
template <bool WIDE>
__global__ __launch_bounds__(256) void bank4_move_kernel(mivos_bank4 from, mivos_bank4 to, int keep, const int32_t *__restrict__ slots) {
  const int bh = blockIdx.y;
  const int kb = from.key_dim / 32, vb = from.value_dim / 32, units = kb + vb, rows = 256 / units;      // units <= 64
  const int u = threadIdx.x % units, r = threadIdx.x / units;
  if (r >= rows) return;
  const bool is_key = u < kb;
  const int blk = is_key ? u : u - kb, nb = is_key ? kb : vb;
  const u32x4 *sc = reinterpret_cast<const u32x4 *>(is_key ? from.key_codes : from.value_codes) + (int64_t)bh * from.slots * nb + blk;
  const uint8_t *ss = (is_key ? from.key_scales : from.value_scales) + (int64_t)bh * from.slots * nb + blk;
  u32x4 *dc = reinterpret_cast<u32x4 *>(is_key ? to.key_codes : to.value_codes) + (int64_t)bh * to.slots * nb + blk;
  uint8_t *ds = (is_key ? to.key_scales : to.value_scales) + (int64_t)bh * to.slots * nb + blk;
  const int32_t *from_slot = slots + (int64_t)bh * keep;
  for (int64_t j = (int64_t)blockIdx.x * rows + r; j < keep; j += (int64_t)gridDim.x * rows) {
    const int64_t slot = from_slot[j];
    if (slot < 0) continue;
    const u32x4 codes = sc[slot * nb];                 // (all loads ahead of the stores)
    const bool scales = !WIDE || (blk & 3) == 0;
    uint32_t scale = 0;
    float w = 0.f;
    if (scales) scale = WIDE ? *reinterpret_cast<const uint32_t *>(ss + slot * nb) : ss[slot * nb];
    if (u == 0) w = from.weight[(int64_t)bh * from.slots + slot];
    dc[j * nb] = codes;
    if (WIDE && scales) *reinterpret_cast<uint32_t *>(ds + j * nb) = scale;
    else if (!WIDE) ds[j * nb] = (uint8_t)scale;
    if (u == 0) to.weight[(int64_t)bh * to.slots + j] = w;
  }
}

// Workgroups a stream (or a head of it) of `at_once` rows each, up to `most`.  Values and moves take one a row group (a launch that goes round
// 16 a CU instead: 97 and 61 us instead of 84 and 56, at the sizes above), append up to 16 a CU, each of which reads the length and counts itself out.
static int grid_x(int64_t rows, int at_once, int64_t most) {
  const int64_t n = (rows + at_once - 1) / at_once;
  return (int)(n < 1 ? 1 : n > most ? most : n);
}
constexpr int64_t GRID_MOST = 1 << 20;

}  // namespace mivos

using namespace mivos;

extern "C" int mivos_bank4_append(const mivos_bank4 *bank, const void *keys, int64_t kb, int64_t kt, int64_t kh, const void *values, int64_t vb,
                                  int64_t vt, int64_t vh, int dtype, const int32_t *at, const int32_t *count, int tokens, void *stream) {
  if (int rc = bank4_check(bank, "bank4_append")) return rc;
  if (!dtype_ok(dtype) || tokens < 0 || !at || (tokens && (!keys || !values))) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_append: bad argument");
  const Span lens(bank->lens, (int64_t)bank->batch * 4);
  if ((at != bank->lens && lens.meets(Span(at, (int64_t)bank->batch * 4))) || (count && lens.meets(Span(count, (int64_t)bank->batch * 4))))
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_append: at or count overlaps the bank's lengths");
  if ((int64_t)tokens * bank->heads > 0x7fffffff) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_append: %d tokens x %d heads", tokens, bank->heads);
  const int units = (bank->key_dim + bank->value_dim) / 8, es = dtype_bytes(dtype);
  const int64_t all = kb | kt | kh | vb | vt | vh;
  const int vec = ((all * es) & 15) == 0 && (((uintptr_t)keys | (uintptr_t)values) & 15) == 0;
  const dim3 grid(grid_x((int64_t)tokens * bank->heads, 256 / units, 256 * 16 / bank->batch + 1), bank->batch);
  hipStream_t s = (hipStream_t)stream;
#define GO(T) bank4_append_kernel<T><<<grid, 256, 0, s>>>(*bank, (const T *)keys, kb, kt, kh, (const T *)values, vb, vt, vh, vec, at, count, tokens, units)
  if (dtype == MIVOS_F32) GO(float);
  else if (dtype == MIVOS_F16) GO(_Float16);
  else GO(__bf16);
#undef GO
  return check_launch("bank4_append");
}

extern "C" int mivos_bank4_values(const mivos_bank4 *bank, const int32_t *first, int64_t count, void *key_out, void *value_out, int dtype, void *stream) {
  if (int rc = bank4_check(bank, "bank4_values")) return rc;
  if ((dtype != MIVOS_F32 && dtype != MIVOS_BF16) || count < 0 || count > bank->slots || (count && (!key_out || !value_out)))
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_values: bad argument");
  if (count == 0) return MIVOS_OK;
  const int rows = bank->batch * bank->heads, units = (bank->key_dim + bank->value_dim) / 8;
  const dim3 grid(grid_x(count, VALUES_DEEP * (256 / units), GRID_MOST), rows);
  if (dtype == MIVOS_F32) bank4_values_kernel<float><<<grid, 256, 0, (hipStream_t)stream>>>(*bank, first, (int)count, (float *)key_out, (float *)value_out);
  else bank4_values_kernel<__bf16><<<grid, 256, 0, (hipStream_t)stream>>>(*bank, first, (int)count, (__bf16 *)key_out, (__bf16 *)value_out);
  return check_launch("bank4_values");
}

extern "C" int mivos_bank4_evict(const mivos_bank4 *bank, const mivos_bank4 *out, int64_t keep, int64_t first, int64_t recent, int32_t *slots_out,
                                 void *stream) {
  if (int rc = bank4_check(bank, "bank4_evict")) return rc;
  if (int rc = bank4_check(out, "bank4_evict")) return rc;
  if (out->batch != bank->batch || out->heads != bank->heads || out->key_dim != bank->key_dim || out->value_dim != bank->value_dim)
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_evict: the two banks differ in streams, heads or channels");
  if (bank4_meet(*bank, *out)) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_evict: the banks share memory");
  if (keep < 1 || keep > out->slots || first < 0 || recent < 0 || first + recent > keep || !slots_out)
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_evict: keep %lld of %lld slots, first %lld, recent %lld", (long long)keep, (long long)out->slots,
                (long long)first, (long long)recent);
  const int rows = bank->batch * bank->heads, a_row = 256 / ((bank->key_dim + bank->value_dim) / 32);
  hipStream_t s = (hipStream_t)stream;
  if (bank->slots <= EVICT_THREADS * EVICT_KEYS)
    bank4_select_kernel<true><<<rows, EVICT_THREADS, 0, s>>>(bank->weight, bank->lens, bank->heads, bank->slots, (int)keep, (int)first, (int)recent, slots_out, out->lens);
  else
    bank4_select_kernel<false><<<rows, EVICT_THREADS, 0, s>>>(bank->weight, bank->lens, bank->heads, bank->slots, (int)keep, (int)first, (int)recent, slots_out, out->lens);
  if (int rc = check_launch("bank4_evict")) return rc;
  const dim3 grid(grid_x(keep, a_row, GRID_MOST), rows);
  if (bank->key_dim % 128 == 0 && bank->value_dim % 128 == 0) bank4_move_kernel<true><<<grid, 256, 0, s>>>(*bank, *out, (int)keep, slots_out);
  else bank4_move_kernel<false><<<grid, 256, 0, s>>>(*bank, *out, (int)keep, slots_out);
  return check_launch("bank4_evict");
}
