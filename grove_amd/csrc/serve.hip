// The bookkeeping around a paged cache: rotary positions in both layouts, page tables from lengths, verification of drafted tokens.
#include "common.h"

namespace {

template <typename T> __device__ __forceinline__ float ld1(const T* p);
template <> __device__ __forceinline__ float ld1<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float ld1<bf16_raw>(const bf16_raw* p) { return bf2f(*p); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(bf16_raw* p, float v) { *p = f2bf(v); }

// ---------------------------------------------------------------- rotary positions
// The angle in turns, reduced to [-1/2, 1/2] in fp64 before it becomes a float: at position 1e6 a float angle is off by 0.03 radians.
__device__ __forceinline__ void turn(int pos, double freq, float& s, float& c) {
  const double t = (double)pos * (freq * 0.15915494309189533577);
  sincospif((float)(2.0 * (t - rint(t))), &s, &c);
}

// One thread per pair; the channels behind `rot` are copied by the threads behind the pairs.
template <typename T>
__global__ __launch_bounds__(256) void rotary_kernel(const grove_rotary_params p) {
  const int half = p.rot >> 1, per = half + (p.x == p.y ? 0 : p.hd - p.rot);
  const int64_t n = (int64_t)p.rows * p.heads * per;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    const int i = (int)(e % per);
    const int64_t rh = e / per;
    const int h = (int)(rh % p.heads), r = (int)(rh / p.heads);
    const T* x = (const T*)p.x + r * p.sx_row + h * p.sx_head;
    T* y = (T*)p.y + r * p.sy_row + h * p.sy_head;
    if (i >= half) {
      y[p.rot + i - half] = x[p.rot + i - half];
      continue;
    }
    float s, c;
    turn(p.pos[r], p.freq[i], s, c);
    c *= p.mscale;
    s *= p.backward ? -p.mscale : p.mscale;
    const int ia = p.interleaved ? 2 * i : i, ib = p.interleaved ? 2 * i + 1 : i + half;
    const float a = ld1(x + ia), b = ld1(x + ib);
    st1(y + ia, a * c - b * s);
    st1(y + ib, b * c + a * s);
  }
}

// ---------------------------------------------------------------- page tables
constexpr int PT_THREADS = 256, PT_MAX_REQ = 4096;

// Largest b with pre[b] <= v (pre ascending from 0, n entries and the total behind them, v < total): requests without rows are passed over.
__device__ __forceinline__ int owner(const int* pre, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (pre[m] <= v) lo = m; else hi = m;
  }
  return lo;
}

// Every block forms both prefix sums for itself (a few words per request, from L2), so the entries can be dealt to all blocks of ONE
// launch; a page that this launch hands out is taken from the free list again where a slot needs it, never from the table.
__global__ __launch_bounds__(PT_THREADS) void page_tables_kernel(const grove_page_tables_params p, const int shift) {
  extern __shared__ int lds[];
  int* cu = lds;                        // [requests + 1] rows before
  int* start = lds + p.requests + 1;    // [requests + 1] pages before
  __shared__ long long wsum[2][PT_THREADS / 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, B = p.requests;
  const int per = (B + PT_THREADS - 1) / PT_THREADS, b0 = min(B, tid * per), b1 = min(B, b0 + per);
  auto lengths = [&](int b, int& ctx, int& nw, int& held, int& need) {
    ctx = max(0, p.ctx_len[b]);
    nw = max(0, p.new_len[b]);
    held = max(0, p.held[b]);
    const long long pages = ((long long)ctx + nw + (1 << shift) - 1) >> shift;
    need = (int)max(0LL, min(pages, (long long)p.max_pages) - held);
  };
  long long rows = 0, pages = 0;
  for (int b = b0; b < b1; ++b) {
    int c, nw, h, need;
    lengths(b, c, nw, h, need);
    rows += nw;
    pages += need;
  }
  long long ir = rows, ip = pages;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long a = __shfl_up(ir, o, 64), c = __shfl_up(ip, o, 64);
    if (lane >= o) { ir += a; ip += c; }
  }
  if (lane == 63) { wsum[0][w] = ir; wsum[1][w] = ip; }
  __syncthreads();
  for (int i = 0; i < w; ++i) { ir += wsum[0][i]; ip += wsum[1][i]; }
  rows = ir - rows;
  pages = ip - pages;
  const bool first = blockIdx.x == 0;
  auto cap = [](long long v) { return (int)min(v, 0x7fffffffLL); };
  for (int b = b0; b < b1; ++b) {
    int c, nw, h, need;
    lengths(b, c, nw, h, need);
    cu[b] = cap(rows);
    start[b] = cap(pages);
    if (first) {
      p.kv_len[b] = cap((long long)c + nw);
      p.cu_q[b] = cap(rows);
      p.held_out[b] = h + (int)max(0LL, min((long long)need, p.n_free - pages));
    }
    rows += nw;
    pages += need;
  }
  if (tid == PT_THREADS - 1) {
    cu[B] = cap(rows);
    start[B] = cap(pages);
    if (first) { p.cu_q[B] = cap(rows); p.taken[0] = cap(pages); }
  }
  __syncthreads();
  const int g = blockIdx.x * PT_THREADS + tid, step = gridDim.x * PT_THREADS;
  for (int64_t e = g; e < start[B]; e += step) {
    const int b = owner(start, B, (int)e);
    const int i = max(0, p.held[b]) + (int)e - start[b];
    if (i < p.max_pages) p.table[(int64_t)b * p.ld_table + i] = e < p.n_free ? p.free_pages[e] : -1;
  }
  for (int64_t r = g; r < p.rows; r += step) {
    int slot = -1, pos = 0;
    if (r < cu[B]) {
      const int b = owner(cu, B, (int)r);
      const long long t = (long long)max(0, p.ctx_len[b]) + ((int)r - cu[b]);
      pos = cap(t);
      const long long pi = t >> shift;
      const int held = max(0, p.held[b]);
      if (pi < p.max_pages) {
        const long long e = start[b] + (pi - held);
        const int page = pi < held ? p.table[(int64_t)b * p.ld_table + pi] : e < p.n_free ? p.free_pages[e] : -1;
        const long long at = ((long long)page << shift) + (t & ((1 << shift) - 1));
        if (page >= 0 && at <= 0x7fffffffLL) slot = (int)at;
      }
    }
    p.slots[r] = slot;
    p.pos[r] = pos;
  }
}

// ---------------------------------------------------------------- verification of drafted tokens
constexpr int VD_THREADS = 1024, VD_WAVES = VD_THREADS / 64;

// Inclusive sum over the block in fp64; `total` = the block's. Two barriers.
__device__ __forceinline__ double block_scan(double v, double* wsum, double& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double a = __shfl_up(v, o, 64);
    if (lane >= o) v += a;
  }
  __syncthreads();
  if (lane == 63) wsum[w] = v;
  __syncthreads();
  double before = 0;
  total = 0;
  for (int i = 0; i < VD_WAVES; ++i) {
    if (i == w) before = total;
    total += wsum[i];
  }
  return before + v;
}

// One block per request: the drafts are tested side by side, then the row where they end is summed by chunks (at most 1024), the chunk
// that holds the threshold is found by a scan over the chunk sums and searched element by element.
template <typename T>
__global__ __launch_bounds__(VD_THREADS) void verify_drafts_kernel(const grove_verify_drafts_params p) {
  __shared__ double sums[VD_THREADS], wsum[VD_WAVES];
  __shared__ int s_a, s_min, s_max;
  __shared__ double s_carry;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, b = blockIdx.x, V = p.vocab;
  const int n = p.count ? max(0, min(p.count[b], p.drafts)) : p.drafts;
  const T* P = (const T*)p.p + b * p.sp_req;
  const T* Q = p.q ? (const T*)p.q + b * p.sq_req : nullptr;
  const int* draft = p.draft + (int64_t)b * p.drafts;
  if (tid == 0) s_a = n;
  __syncthreads();
  for (int i = tid; i < n; i += VD_THREADS) {
    const int x = draft[i];
    bool ok = x >= 0 && x < V;
    if (ok) {
      const double q = Q ? (double)ld1(Q + i * p.sq_row + x) : 1.0;
      ok = (double)p.u[(int64_t)b * p.drafts + i] * q < (double)ld1(P + i * p.sp_row + x);
    }
    if (!ok) atomicMin(&s_a, i);
  }
  __syncthreads();
  const int a = s_a;
  P += a * p.sp_row;
  if (Q) Q += a * p.sq_row;
  const int sure = a < n && !Q ? draft[a] : -1;  // a certain drafter's refused token: its mass is what is taken off
  const int per = (V + VD_THREADS * 1024 - 1) / (VD_THREADS * 1024), chunk = 1024 * per, nchunk = (V + chunk - 1) / chunk;
  int token = -1;
  for (int mode = a < n ? 0 : 1; mode < 2; ++mode) {  // 0: what the drafter left over, 1: the target itself
    auto rest = [&](int j) -> double {
      double r = (double)ld1(P + j);
      if (mode == 0) {
        if (Q) r -= (double)ld1(Q + j);
        else if (j == sure) r -= 1.0;
      }
      return r > 0 ? r : 0.0;
    };
    for (int c = w; c < nchunk; c += VD_WAVES) {
      double s = 0;
      for (int j = c * chunk + lane; j < min(V, (c + 1) * chunk); j += 64) s += rest(j);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
      if (lane == 0) sums[c] = s;
    }
    if (tid == 0) { s_min = V; s_max = -1; }
    __syncthreads();
    const double own = tid < nchunk ? sums[tid] : 0.0;
    double total;
    const double inc = block_scan(own, wsum, total);
    if (!(total > 0)) { __syncthreads(); continue; }
    const double thr = (double)p.pick[b] * total;
    if (tid < nchunk && own > 0) {
      if (inc > thr) atomicMin(&s_min, tid);
      atomicMax(&s_max, tid);
    }
    __syncthreads();
    const int c = s_min < V ? s_min : s_max;
    if (tid == c) s_carry = inc - own;
    __syncthreads();
    double carry = s_carry;
    if (tid == 0) { s_min = V; s_max = -1; }
    __syncthreads();
    for (int j0 = c * chunk; j0 < min(V, (c + 1) * chunk); j0 += VD_THREADS) {
      const int j = j0 + tid;
      const double r = j < V ? rest(j) : 0.0;
      double sub;
      const double cdf = carry + block_scan(r, wsum, sub);
      if (r > 0) {
        if (cdf > thr) atomicMin(&s_min, j);
        atomicMax(&s_max, j);
      }
      carry += sub;
    }
    __syncthreads();
    token = s_min < V ? s_min : s_max;
    break;
  }
  for (int i = tid; i <= p.drafts; i += VD_THREADS) p.tokens[(int64_t)b * (p.drafts + 1) + i] = i < a ? draft[i] : i == a ? token : -1;
  if (tid == 0) p.accepted[b] = a;
}

}  // namespace

extern "C" int grove_rotary(const grove_rotary_params* p, void* stream) {
  GROVE_CHECK(p && p->rows >= 0 && p->heads >= 0 && p->hd > 0 && p->rot >= 0 && p->rot <= p->hd && (p->rot & 1) == 0, GROVE_E_SHAPE, "rotary: bad shape");
  if (p->rows == 0 || p->heads == 0) return GROVE_OK;
  GROVE_CHECK(p->x && p->y && p->pos && (p->freq || p->rot == 0), GROVE_E_SHAPE, "rotary: null pointer");
  GROVE_CHECK(p->x != p->y || (p->sx_row == p->sy_row && p->sx_head == p->sy_head), GROVE_E_SHAPE, "rotary: in place needs equal strides");
  const int64_t n = (int64_t)p->rows * p->heads * p->hd;
  const unsigned blocks = (unsigned)((n + 255) / 256 > 65536 ? 65536 : (n + 255) / 256);
  if (p->f32) hipLaunchKernelGGL(rotary_kernel<float>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, *p);
  else hipLaunchKernelGGL(rotary_kernel<bf16_raw>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, *p);
  GROVE_LAUNCH_CHECK();
  return GROVE_OK;
}

extern "C" int grove_page_tables(const grove_page_tables_params* p, void* stream) {
  GROVE_CHECK(p && p->requests > 0 && p->requests <= PT_MAX_REQ && p->max_pages > 0 && p->rows >= 0 && p->n_free >= 0 && p->ld_table >= p->max_pages,
              GROVE_E_SHAPE, "page_tables: bad shape (1 to %d requests)", PT_MAX_REQ);
  GROVE_CHECK(p->page >= 1 && (p->page & (p->page - 1)) == 0, GROVE_E_SHAPE, "page_tables: the page size must be a power of two");
  GROVE_CHECK(p->ctx_len && p->new_len && p->held && (p->free_pages || p->n_free == 0) && p->table && p->kv_len && p->cu_q &&
              ((p->slots && p->pos) || p->rows == 0) && p->held_out && p->taken && p->held_out != p->held && p->kv_len != p->ctx_len &&
              p->kv_len != p->new_len, GROVE_E_SHAPE, "page_tables: null pointer, or an output is an input");
  const int64_t rows = p->rows > p->requests ? p->rows : p->requests;
  const unsigned blocks = (unsigned)((rows + PT_THREADS - 1) / PT_THREADS > 256 ? 256 : (rows + PT_THREADS - 1) / PT_THREADS);
  hipLaunchKernelGGL(page_tables_kernel, dim3(blocks), dim3(PT_THREADS), (size_t)8 * (p->requests + 1), (hipStream_t)stream, *p, __builtin_ctz((unsigned)p->page));
  GROVE_LAUNCH_CHECK();
  return GROVE_OK;
}

extern "C" int grove_verify_drafts(const grove_verify_drafts_params* p, void* stream) {
  GROVE_CHECK(p && p->requests >= 0 && p->drafts >= 0 && p->vocab > 0 && p->vocab <= (1 << 30), GROVE_E_SHAPE, "verify_drafts: bad shape");
  if (p->requests == 0) return GROVE_OK;
  GROVE_CHECK(p->p && p->pick && p->tokens && p->accepted && ((p->draft && p->u) || p->drafts == 0), GROVE_E_SHAPE, "verify_drafts: null pointer");
  if (p->bf16) hipLaunchKernelGGL(verify_drafts_kernel<bf16_raw>, dim3((unsigned)p->requests), dim3(VD_THREADS), 0, (hipStream_t)stream, *p);
  else hipLaunchKernelGGL(verify_drafts_kernel<float>, dim3((unsigned)p->requests), dim3(VD_THREADS), 0, (hipStream_t)stream, *p);
  GROVE_LAUNCH_CHECK();
  return GROVE_OK;
}
