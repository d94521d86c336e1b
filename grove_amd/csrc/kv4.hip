// The paged 4-bit key / value cache (layout: grove_hip.h): quantise into pages, read back, attend.
#include "common.h"

namespace {

// Where channel c of the row `r` of a page is held: the byte within the (page, head) plane, and which nibble of it.
template <int HD>
__device__ __forceinline__ int key_byte(int r, int c, int& hi) {
  const int t = c >> 5, h = (c >> 3) & 3, i = c & 7, nib = (i & 1) * 4 + (i >> 1);
  hi = nib & 1;
  return r * (HD / 2) + (h * (HD / 32) + t) * 4 + (nib >> 1);
}
template <int HD>
__device__ __forceinline__ int value_byte(int r, int c, int& hi) {
  const int tp = (r >> 1) & 1, par = r & 1, j = c >> 4, m = c & 15;
  hi = j & 1;
  const int quad = (r >> 2) * (2 * HD) + m * (HD / 8);
  if constexpr (HD == 32) return quad + par * 2 + tp;
  return quad + ((j >> 2) * 2 + tp) * 4 + par * 2 + ((j >> 1) & 1);
}

__device__ __forceinline__ bool slot_of(const int* slots, int row, int page, int pages, int& pg, int& at) {
  const int s = slots[row];
  if (s < 0 || s >= (int64_t)pages * page) return false;
  pg = s / page;
  at = s - pg * page;
  return true;
}

// One wave per (row, head, keys or values).
template <int HD>
__global__ __launch_bounds__(64) void kv4_append_kernel(const grove_kv4_append_params p) {
  __shared__ unsigned char code[HD];
  const int lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y, which = blockIdx.z;
  int pg, at;
  if (!slot_of(p.slots, row, p.page, p.pages, pg, at)) return;
  const bf16_raw* x = which ? (const bf16_raw*)p.v + row * p.sv_row + head * p.sv_head : (const bf16_raw*)p.k + row * p.sk_row + head * p.sk_head;
  float v[(HD + 63) / 64], lo = INFINITY, hi = -INFINITY;
  bool bad = false;
  for (int i = 0, c = lane; c < HD; c += 64, ++i) {
    v[i] = bf2f(x[c]);
    bad |= !(fabsf(v[i]) < INFINITY);
    lo = fminf(lo, v[i]);
    hi = fmaxf(hi, v[i]);
  }
  lo = -wave_max(-lo);
  hi = wave_max(hi);
  const float span = hi - lo;
  bad = __any(bad) || !(span < INFINITY);
  bf16_raw sb = span < 0x1p-100f ? 0 : f2bf(span / 15.f), mb = f2bf(lo);
  if (bad) sb = mb = 0x7fc0;
  const float s = bf2f(sb);
  for (int i = 0, c = lane; c < HD; c += 64, ++i)
    code[c] = (bad || s == 0.f) ? 0 : (unsigned char)fminf(fmaxf(rintf((v[i] - lo) / s), 0.f), 15.f);
  __syncthreads();
  const int64_t plane = ((int64_t)pg * 2 + which) * p.kv + head;
  unsigned char* out = (unsigned char*)p.codes + plane * p.page * (HD / 2);
  for (int c = lane; c < HD; c += 64) {
    int up;
    const int byte = which ? value_byte<HD>(at, c, up) : key_byte<HD>(at, c, up);
    const int pair = which ? c + 16 : c + 2;  // the channel in the upper nibble of the same byte
    if (!up) out[byte] = code[c] | (code[pair] << 4);
  }
  if (lane == 0) ((unsigned*)p.scales)[plane * p.page + at] = sb | ((unsigned)mb << 16);
}

template <int HD, typename T>
__global__ __launch_bounds__(64) void kv4_read_kernel(const grove_kv4_read_params p) {
  const int lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y, which = blockIdx.z;
  int pg = 0, at = 0;
  const bool ok = slot_of(p.slots, row, p.page, p.pages, pg, at);
  const int64_t plane = ((int64_t)pg * 2 + which) * p.kv + head;
  const unsigned char* in = (const unsigned char*)p.codes + plane * p.page * (HD / 2);
  T* y = (T*)(which ? p.v : p.k) + ((int64_t)row * p.kv + head) * HD;
  const unsigned sm = ok ? ((const unsigned*)p.scales)[plane * p.page + at] : 0;
  for (int c = lane; c < HD; c += 64) {
    int up;
    const int byte = which ? value_byte<HD>(at, c, up) : key_byte<HD>(at, c, up);
    const int code = ok ? (in[byte] >> (4 * up)) & 15 : 0;
    const float v = fmaf((float)code, bf_lo(sm), bf_hi(sm));
    if constexpr (sizeof(T) == 4) y[c] = v; else y[c] = f2bf(v);
  }
}

// One wave per (row, query head): 64 keys at a time, a lane each for the scores; then a lane per channel for the values.
template <int HD>
__global__ __launch_bounds__(64) void kv4_attn_simple_kernel(const grove_kv4_attn_params p) {
  __shared__ float q[HD], pr[64];
  __shared__ int pages[64];
  const int lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y, kvh = head / (p.heads / p.kv);
  int b = -1;
  for (int i = 0; i < p.requests; ++i)
    if (row >= p.cu_q[i] && row < p.cu_q[i + 1]) b = i;
  if (b < 0) return;
  const int n = p.cu_q[b + 1] - p.cu_q[b], len = p.kv_len[b];
  const int64_t room = (int64_t)p.max_pages * p.page;
  const int seen = (int)min(room, (int64_t)len - n + (row - p.cu_q[b]) + 1);
  const bf16_raw* x = (const bf16_raw*)p.q + row * p.sq_row + head * p.sq_head;
  for (int c = lane; c < HD; c += 64) q[c] = bf2f(x[c]);
  constexpr int NC = (HD + 63) / 64;
  float acc[NC] = {}, mx = -INFINITY, sum = 0.f;
  for (int t0 = 0; t0 < seen; t0 += 64) {
    __syncthreads();
    const int t = t0 + lane;
    const int pg = t < seen ? p.table[b * p.ld_table + t / p.page] : -1;
    pages[lane] = pg;
    float z = -INFINITY;
    if (pg >= 0 && pg < p.pages) {
      const int64_t plane = (int64_t)pg * 2 * p.kv + kvh;
      const unsigned char* in = (const unsigned char*)p.codes + plane * p.page * (HD / 2);
      const unsigned sm = ((const unsigned*)p.scales)[plane * p.page + t % p.page];
      z = 0.f;
      for (int c = 0; c < HD; ++c) {
        int up;
        const int byte = key_byte<HD>(t % p.page, c, up);
        z = fmaf(q[c], fmaf((float)((in[byte] >> (4 * up)) & 15), bf_lo(sm), bf_hi(sm)), z);
      }
      z *= p.alpha;
    }
    const float top = fmaxf(mx, wave_max(z)), ref = top == -INFINITY ? 0.f : top;
    const float e = z == -INFINITY ? 0.f : expf(z - ref), keep = mx == -INFINITY ? 0.f : expf(mx - ref);
    mx = top;
    sum = sum * keep + wave_sum(e);
    pr[lane] = e;
    __syncthreads();
    for (int i = 0; i < NC; ++i) acc[i] *= keep;
    for (int k = 0; k < 64; ++k) {
      const int pk = pages[k];
      if (pk < 0 || pk >= p.pages) continue;
      const int64_t plane = ((int64_t)pk * 2 + 1) * p.kv + kvh;
      const unsigned char* in = (const unsigned char*)p.codes + plane * p.page * (HD / 2);
      const int at = (t0 + k) % p.page;
      const unsigned sm = ((const unsigned*)p.scales)[plane * p.page + at];
      for (int i = 0, c = lane; c < HD; c += 64, ++i) {
        int up;
        const int byte = value_byte<HD>(at, c, up);
        acc[i] = fmaf(pr[k], fmaf((float)((in[byte] >> (4 * up)) & 15), bf_lo(sm), bf_hi(sm)), acc[i]);
      }
    }
  }
  bf16_raw* y = (bf16_raw*)p.out + row * p.so_row + (int64_t)head * HD;
  for (int i = 0, c = lane; c < HD; c += 64, ++i) y[c] = f2bf(sum > 0.f || sum != sum ? acc[i] / sum : 0.f);
}

bool page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128 || page == 256; }
bool hd_ok(int hd) { return hd == 32 || hd == 64 || hd == 128 || hd == 256; }

}  // namespace

#define KV4_SHAPE(p, what)                                                                                                                   \
  GROVE_CHECK(hd_ok((p)->hd) && page_ok((p)->page), GROVE_E_SHAPE, what ": the head size must be 32, 64, 128 or 256, the page 16, 32, 64, 128 or 256"); \
  GROVE_CHECK((p)->pages > 0 && (int64_t)(p)->pages * (p)->page <= 0x7fffffff, GROVE_E_SHAPE, what ": bad number of pages")
#define KV4_HD(hd, LAUNCH)      \
  switch (hd) {                 \
    case 32: LAUNCH(32); break; \
    case 64: LAUNCH(64); break; \
    case 128: LAUNCH(128); break; \
    default: LAUNCH(256);       \
  }

extern "C" int grove_kv4_append(const grove_kv4_append_params* p, void* stream) {
  GROVE_CHECK(p && p->rows >= 0 && p->kv > 0 && p->kv <= 65535, GROVE_E_SHAPE, "kv4_append: bad shape");
  KV4_SHAPE(p, "kv4_append");
  if (p->rows == 0) return GROVE_OK;
  GROVE_CHECK(p->k && p->v && p->codes && p->scales && p->slots, GROVE_E_SHAPE, "kv4_append: null pointer");
  GROVE_CHECK(((uintptr_t)p->codes & 15) == 0 && ((uintptr_t)p->scales & 15) == 0, GROVE_E_ALIGN, "kv4_append: the cache must be 16-byte aligned");
#define LAUNCH(HD) hipLaunchKernelGGL(kv4_append_kernel<HD>, dim3((unsigned)p->rows, (unsigned)p->kv, 2), dim3(64), 0, (hipStream_t)stream, *p)
  KV4_HD(p->hd, LAUNCH)
#undef LAUNCH
  GROVE_LAUNCH_CHECK();
  return GROVE_OK;
}

extern "C" int grove_kv4_read(const grove_kv4_read_params* p, void* stream) {
  GROVE_CHECK(p && p->rows >= 0 && p->kv > 0 && p->kv <= 65535, GROVE_E_SHAPE, "kv4_read: bad shape");
  KV4_SHAPE(p, "kv4_read");
  if (p->rows == 0) return GROVE_OK;
  GROVE_CHECK(p->k && p->v && p->codes && p->scales && p->slots, GROVE_E_SHAPE, "kv4_read: null pointer");
  GROVE_CHECK(((uintptr_t)p->codes & 15) == 0 && ((uintptr_t)p->scales & 15) == 0, GROVE_E_ALIGN, "kv4_read: the cache must be 16-byte aligned");
  const dim3 grid((unsigned)p->rows, (unsigned)p->kv, 2);
#define LAUNCH(HD)                                                                                                     \
  if (p->f32) hipLaunchKernelGGL((kv4_read_kernel<HD, float>), grid, dim3(64), 0, (hipStream_t)stream, *p);            \
  else hipLaunchKernelGGL((kv4_read_kernel<HD, bf16_raw>), grid, dim3(64), 0, (hipStream_t)stream, *p)
  KV4_HD(p->hd, LAUNCH)
#undef LAUNCH
  GROVE_LAUNCH_CHECK();
  return GROVE_OK;
}

extern "C" int grove_kv4_attn(const grove_kv4_attn_params* p, void* stream) {
  GROVE_CHECK(p && p->requests >= 0 && p->requests <= 65535 && p->rows >= 0 && p->kv > 0 && p->heads > 0 && p->heads % p->kv == 0 && p->heads <= 65535 &&
              p->max_pages > 0 && p->ld_table >= p->max_pages && p->max_q >= 0, GROVE_E_SHAPE, "kv4_attn: bad shape (heads must be a multiple of kv)");
  KV4_SHAPE(p, "kv4_attn");
  if (p->rows == 0 || p->requests == 0 || p->max_q == 0) return GROVE_OK;
  GROVE_CHECK(p->q && p->codes && p->scales && p->table && p->kv_len && p->cu_q && p->out, GROVE_E_SHAPE, "kv4_attn: null pointer");
  GROVE_CHECK(((uintptr_t)p->codes & 15) == 0 && ((uintptr_t)p->scales & 15) == 0, GROVE_E_ALIGN, "kv4_attn: the cache must be 16-byte aligned");
#define LAUNCH(HD) hipLaunchKernelGGL(kv4_attn_simple_kernel<HD>, dim3((unsigned)p->rows, (unsigned)p->heads), dim3(64), 0, (hipStream_t)stream, *p)
  KV4_HD(p->hd, LAUNCH)
#undef LAUNCH
  GROVE_LAUNCH_CHECK();
  return GROVE_OK;
}
