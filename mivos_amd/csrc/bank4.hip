// Memory bank in 4 bits: append (quantise + store), values (read back), evict (keep the slots with the most attention weight).
// All three move bytes: append reads a row once and writes 17/64 of its bf16 size, values the reverse, evict reads 4 bytes a slot for the
// choice and moves the kept rows once.  The attention read over the bank is bank4_read.hip.
#include "bank4.h"

namespace mivos {

// ---------------------------------------------------------------------------------------------- append
// One thread quantises 8 channels, four neighbours make up a block of 32: they share the block's largest magnitude by two lane
// exchanges, so a row is read once and nothing is staged.  scale = the smallest power of two 2^e with max |x| <= 6 * 2^e: nothing
// saturates (the floor(log2) rule of the microscaling formats clips up to a quarter off a block's largest value).
template <typename T>
__global__ __launch_bounds__(256) void bank4_append_kernel(mivos_bank4 bank, const T *__restrict__ keys, int64_t kb, int64_t kt, int64_t kh,
                                                           const T *__restrict__ values, int64_t vb, int64_t vt, int64_t vh, int vec,
                                                           const int32_t *at, const int32_t *__restrict__ count, int tokens, int units) {
  const int b = blockIdx.y;
  const int64_t total = (int64_t)tokens * bank.heads * units;       // units = (key_dim + value_dim) / 8, a multiple of 4
  const int64_t start = at[b];
  int n = count ? count[b] : tokens;
  n = n < 0 ? 0 : n > tokens ? tokens : n;
  bool lost = false;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const uint32_t th = (uint32_t)(i / units);
    int u = (int)(i - (int64_t)th * units);
    const int t = th / (uint32_t)bank.heads, h = th - t * bank.heads;
    const int64_t slot = start + t;
    if (t >= n) continue;                                            // (the four lanes of a block share t, h and the branch)
    if (slot < 0 || slot >= bank.slots) { lost = true; continue; }
    const int64_t row = ((int64_t)b * bank.heads + h) * bank.slots + slot;
    if (u == 0) bank.weight[row] = 0.f;
    const int ku = bank.key_dim / 8;
    const bool is_key = u < ku;
    const T *src = is_key ? keys + b * kb + t * kt + h * kh : values + b * vb + t * vt + h * vh;
    uint8_t *codes = is_key ? bank.key_codes : bank.value_codes, *scales = is_key ? bank.key_scales : bank.value_scales;
    const int dim = is_key ? bank.key_dim : bank.value_dim;
    u = is_key ? u : u - ku;
    const f32x8 x = load8(src + u * 8, vec);
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
    reinterpret_cast<uint32_t *>(codes + row * (dim / 2))[u] = packed;
    if ((u & 3) == 0) scales[row * (dim / 32) + (u >> 2)] = (uint8_t)byte;
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
template <typename T>
__global__ __launch_bounds__(256) void bank4_values_kernel(mivos_bank4 bank, const int32_t *__restrict__ first, int count, T *__restrict__ key_out,
                                                           T *__restrict__ value_out) {
  const int bh = blockIdx.y, b = bh / bank.heads;
  const int ku = bank.key_dim / 8, units = ku + bank.value_dim / 8;
  const int64_t start = first ? first[b] : 0;
  int64_t len = bank.lens[b];
  len = len > bank.slots ? bank.slots : len;
  const int64_t total = (int64_t)count * units;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const uint32_t j = (uint32_t)(i / units);
    int u = (int)(i - (int64_t)j * units);
    const bool is_key = u < ku;
    u = is_key ? u : u - ku;
    const int dim = is_key ? bank.key_dim : bank.value_dim;
    const int64_t slot = start + j, row = (int64_t)bh * bank.slots + slot;
    f32x8 v;
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = 0.f;
    if (slot >= 0 && slot < len) {
      const uint32_t codes = reinterpret_cast<const uint32_t *>((is_key ? bank.key_codes : bank.value_codes) + row * (dim / 2))[u];
      const bf16x8 w = bank4_unpack8(codes, bank4_scale((is_key ? bank.key_scales : bank.value_scales)[row * (dim / 32) + (u >> 2)]));
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = (float)w[c];
    }
    store8((is_key ? key_out : value_out) + ((int64_t)bh * count + j) * dim + u * 8, v);
  }
}

// ---------------------------------------------------------------------------------------------- evict
// Order of the weights as unsigned integers: larger weight, larger key; NaN lowest; -0 = +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int EVICT_THREADS = 1024;

// Which slots of one (stream, head) stay: a radix select of the keep-th largest key among the unprotected slots (four passes of
// 8 bits, the counts in LDS), then one ordered pass that writes the kept slots ascending.  Equal weights: the lowest slots stay.
__global__ __launch_bounds__(EVICT_THREADS) void bank4_select_kernel(const float *__restrict__ weight, const int32_t *__restrict__ lens, int heads, int64_t slots,
                                                                    int keep, int first, int recent, int32_t *__restrict__ slots_out,
                                                                    int32_t *__restrict__ lens_out) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t chosen[2];
  __shared__ int base[2];
  __shared__ int wave_kept[EVICT_THREADS / 64], wave_ties[EVICT_THREADS / 64];
  const int bh = blockIdx.x, b = bh / heads, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t n64 = lens[b];
  const int n = (int)(n64 < 0 ? 0 : n64 > slots ? slots : n64);
  const float *w = weight + (int64_t)bh * slots;
  int32_t *out = slots_out + (int64_t)bh * keep;
  const int fresh = n < keep ? n : keep;
  if (tid == 0 && bh % heads == 0) lens_out[b] = fresh;
  if (n <= keep) {
    for (int i = tid; i < keep; i += EVICT_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const int lo = first, hi = n - recent;                             // unprotected slots [lo, hi); first + recent <= keep < n
  int want = keep - first - recent;                                  // of which this many stay
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    for (int i = tid; i < 256; i += EVICT_THREADS) hist[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += EVICT_THREADS) {
      const uint32_t k = weight_key(w[i]);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid < 64) {                                                  // lane l: bins 255 - 4l .. 252 - 4l, from the top
      uint32_t c[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += c[j] = hist[255 - 4 * tid - j];
      uint32_t before = sum;
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(before, d);
        if (tid >= d) before += o;
      }
      before -= sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (before < (uint32_t)want && (uint32_t)want <= before + c[j]) { chosen[0] = 255 - 4 * tid - j; chosen[1] = before; }
        before += c[j];
      }
    }
    __syncthreads();
    prefix |= chosen[0] << shift;
    mask |= 255u << shift;
    want -= (int)chosen[1];
    __syncthreads();
  }
  // now: keys above `prefix` stay, and the first `want` of those equal to it
  const bool any = keep - first - recent > 0;
  if (tid == 0) base[0] = base[1] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += EVICT_THREADS) {
    const int i = i0 + tid;
    bool stays = false, tie = false;
    if (i < n) {
      if (i < lo || i >= hi) stays = true;
      else if (any) {
        const uint32_t k = weight_key(w[i]);
        stays = k > prefix;
        tie = k == prefix;
      }
    }
    const uint64_t below = (1ull << lane) - 1;
    const uint64_t ties = __ballot(tie);
    if (lane == 0) wave_ties[wave] = __popcll(ties);
    __syncthreads();
    int tie_rank = base[1] + __popcll(ties & below);
    for (int v = 0; v < wave; ++v) tie_rank += wave_ties[v];
    stays |= tie && tie_rank < want;
    const uint64_t kept = __ballot(stays);
    if (lane == 0) wave_kept[wave] = __popcll(kept);
    __syncthreads();
    int rank = base[0] + __popcll(kept & below);
    for (int v = 0; v < wave; ++v) rank += wave_kept[v];
    if (stays) out[rank] = i;
    __syncthreads();
    if (tid == 0)
      for (int v = 0; v < EVICT_THREADS / 64; ++v) { base[0] += wave_kept[v]; base[1] += wave_ties[v]; }
    __syncthreads();
  }
}

// Moves the kept rows: one thread a 4-byte word of codes; the scales and the weight go with the row's first threads.
__global__ __launch_bounds__(256) void bank4_move_kernel(mivos_bank4 from, mivos_bank4 to, int keep, const int32_t *__restrict__ slots) {
  const int bh = blockIdx.y;
  const int ku = from.key_dim / 8, units = ku + from.value_dim / 8;
  const int64_t total = (int64_t)keep * units;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const uint32_t j = (uint32_t)(i / units);
    int u = (int)(i - (int64_t)j * units);
    const int32_t slot = slots[(int64_t)bh * keep + j];
    if (slot < 0) continue;
    const int64_t src = (int64_t)bh * from.slots + slot, dst = (int64_t)bh * to.slots + j;
    if (u == 0) to.weight[dst] = from.weight[src];
    const bool is_key = u < ku;
    u = is_key ? u : u - ku;
    const int dim = is_key ? from.key_dim : from.value_dim;
    const uint8_t *sc = is_key ? from.key_codes : from.value_codes, *ss = is_key ? from.key_scales : from.value_scales;
    uint8_t *dc = is_key ? to.key_codes : to.value_codes, *ds = is_key ? to.key_scales : to.value_scales;
    reinterpret_cast<uint32_t *>(dc + dst * (dim / 2))[u] = reinterpret_cast<const uint32_t *>(sc + src * (dim / 2))[u];
    if ((u & 3) == 0) ds[dst * (dim / 32) + (u >> 2)] = ss[src * (dim / 32) + (u >> 2)];
  }
}

static int grid_x(int64_t threads, int rows) {     // workgroups of 256 a (stream, head): all of them, up to 16 a CU over the launch
  int64_t n = (threads + 255) / 256, most = 256 * 16 / rows + 1;
  return (int)(n < 1 ? 1 : n > most ? most : n);
}

}  // namespace mivos

using namespace mivos;

extern "C" int mivos_bank4_append(const mivos_bank4 *bank, const void *keys, int64_t kb, int64_t kt, int64_t kh, const void *values, int64_t vb,
                                  int64_t vt, int64_t vh, int dtype, const int32_t *at, const int32_t *count, int tokens, void *stream) {
  if (int rc = bank4_check(bank, "bank4_append")) return rc;
  if (!dtype_ok(dtype) || tokens < 0 || !at || (tokens && (!keys || !values))) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_append: bad argument");
  if ((int64_t)tokens * bank->heads > 0x7fffffff) return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_append: %d tokens x %d heads", tokens, bank->heads);
  const int units = (bank->key_dim + bank->value_dim) / 8, es = dtype_bytes(dtype);
  const int64_t all = kb | kt | kh | vb | vt | vh;
  const int vec = ((all * es) & 15) == 0 && (((uintptr_t)keys | (uintptr_t)values) & 15) == 0;
  const dim3 grid(grid_x((int64_t)tokens * bank->heads * units, bank->batch), bank->batch);
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
  const dim3 grid(grid_x(count * units, rows), rows);
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
  if (out->key_codes == bank->key_codes || out->value_codes == bank->value_codes || out->weight == bank->weight || out->lens == bank->lens)
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_evict: the banks share memory");
  if (keep < 1 || keep > out->slots || first < 0 || recent < 0 || first + recent > keep || !slots_out)
    return fail(MIVOS_ERR_INVALID_ARGUMENT, "bank4_evict: keep %lld of %lld slots, first %lld, recent %lld", (long long)keep, (long long)out->slots,
                (long long)first, (long long)recent);
  const int rows = bank->batch * bank->heads, units = (bank->key_dim + bank->value_dim) / 8;
  hipStream_t s = (hipStream_t)stream;
  bank4_select_kernel<<<rows, EVICT_THREADS, 0, s>>>(bank->weight, bank->lens, bank->heads, bank->slots, (int)keep, (int)first, (int)recent, slots_out, out->lens);
  if (int rc = check_launch("bank4_evict")) return rc;
  bank4_move_kernel<<<dim3(grid_x(keep * units, rows), rows), 256, 0, s>>>(*bank, *out, (int)keep, slots_out);
  return check_launch("bank4_evict");
}
