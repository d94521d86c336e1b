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

// A block makes cos and sin of its rows once, in LDS (fp64 reduction and sincospif are some 60 instructions a pair, and every head of a row shares
// them), then streams the heads: each thread takes E channels of a pair's first member and, in the half layout, the E of its second (16 bytes each
// where everything is aligned; E = 1 pair otherwise). Bound by memory: everything is read once and written once.
constexpr int ROT_THREADS = 256, ROT_TABLE = 2048;  // pairs that a block's table holds

__device__ __forceinline__ void rot_ld(const float* p, float (&v)[4]) {
  const f32x4_t x = *(const f32x4_t*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = x[i];
}
__device__ __forceinline__ void rot_ld(const bf16_raw* p, float (&v)[8]) {
  const u32x4_t x = *(const u32x4_t*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = bf_lo(x[i]); v[2 * i + 1] = bf_hi(x[i]); }
}
__device__ __forceinline__ void rot_st(float* p, const float (&v)[4]) { *(f32x4_t*)p = (f32x4_t){v[0], v[1], v[2], v[3]}; }
__device__ __forceinline__ void rot_st(bf16_raw* p, const float (&v)[8]) {
  *(u32x4_t*)p = (u32x4_t){pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7])};
}
template <typename T> __device__ __forceinline__ void rot_ld(const T* p, float (&v)[1]) { v[0] = ld1(p); }
template <typename T> __device__ __forceinline__ void rot_st(T* p, const float (&v)[1]) { st1(p, v[0]); }

// rpb rows and hpb heads per block; grid (row groups, head groups).
template <typename T, int E, bool INTERLEAVED>
__global__ __launch_bounds__(ROT_THREADS) void rotary_kernel(const grove_rotary_params p, const int rpb, const int hpb) {
  __shared__ __attribute__((aligned(16))) float s_c[ROT_TABLE], s_s[ROT_TABLE];
  const int tid = threadIdx.x, half = p.rot >> 1, row0 = blockIdx.x * rpb, nr = min(rpb, p.rows - row0), h0 = blockIdx.y * hpb, nh = min(hpb, p.heads - h0);
  const float sign = p.backward ? -p.mscale : p.mscale;
  for (int e = tid; e < nr * half; e += ROT_THREADS) {
    const int r = e / half, i = e - r * half;
    float s, c;
    turn(p.pos[row0 + r], p.freq[i], s, c);
    s_c[e] = c * p.mscale;
    s_s[e] = s * sign;
  }
  __syncthreads();
  // items of a (row, head): the rotated ones, then the ones that pass through (nothing to do in place)
  constexpr int STEP = INTERLEAVED && E == 1 ? 2 : E;  // channels of an item, and of an item's first member in the half layout
  const int turned = INTERLEAVED ? p.rot / STEP : half / STEP, per = turned + (p.x == p.y ? 0 : (p.hd - p.rot) / E), n = nr * nh * per;
  for (int e = tid; e < n; e += ROT_THREADS) {
    const int rh = e / per, i = e - rh * per, r = rh / nh, h = h0 + rh - r * nh;
    const T* x = (const T*)p.x + (row0 + r) * p.sx_row + h * p.sx_head;
    T* y = (T*)p.y + (row0 + r) * p.sy_row + h * p.sy_head;
    float a[E], b[E];
    if (i >= turned) {
      const int c = p.rot + (i - turned) * E;
      rot_ld(x + c, a);
      rot_st(y + c, a);
    } else if constexpr (INTERLEAVED && E > 1) {
      rot_ld(x + i * E, a);
      const int t = r * half + i * (E / 2);
#pragma unroll
      for (int k = 0; k < E; k += 2) {
        const float c = s_c[t + k / 2], s = s_s[t + k / 2];
        b[k] = a[k] * c - a[k + 1] * s;
        b[k + 1] = a[k + 1] * c + a[k] * s;
      }
      rot_st(y + i * E, b);
    } else {
      const int ia = INTERLEAVED ? 2 * i : i * E, ib = INTERLEAVED ? 2 * i + 1 : i * E + half, t = r * half + i * E;
      rot_ld(x + ia, a);
      rot_ld(x + ib, b);
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float c = s_c[t + k], s = s_s[t + k], u = a[k] * c - b[k] * s;
        b[k] = b[k] * c + a[k] * s;
        a[k] = u;
      }
      rot_st(y + ia, a);
      rot_st(y + ib, b);
    }
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
  GROVE_CHECK(p && p->rows >= 0 && p->heads >= 0 && p->hd > 0 && p->rot >= 0 && p->rot <= p->hd && (p->rot & 1) == 0 && (int64_t)p->heads * p->hd < (1 << 28),
              GROVE_E_SHAPE, "rotary: bad shape");
  if (p->rows == 0 || p->heads == 0) return GROVE_OK;
  GROVE_CHECK(p->x && p->y && p->pos && (p->freq || p->rot == 0), GROVE_E_SHAPE, "rotary: null pointer");
  GROVE_CHECK(p->x != p->y || (p->sx_row == p->sy_row && p->sx_head == p->sy_head), GROVE_E_SHAPE, "rotary: in place needs equal strides");
  // 16 bytes at a time where every piece of a (row, head) starts at a multiple of 16 bytes: the pairs' second members and what passes through too
  const int es = p->f32 ? 4 : 2, E = 16 / es;
  auto whole = [&](int64_t v) { return v % E == 0; };
  const bool vec = (((uintptr_t)p->x | (uintptr_t)p->y) & 15) == 0 && whole(p->sx_row) && whole(p->sx_head) && whole(p->sy_row) && whole(p->sy_head) &&
                   whole(p->interleaved ? p->rot : p->rot / 2) && whole(p->hd - p->rot);
  const int half = p->rot / 2;
  GROVE_CHECK(half <= ROT_TABLE, GROVE_E_SHAPE, "rotary: at most %d rotated channels", 2 * ROT_TABLE);
  // A block per row and half a dozen heads while there are few rows (their latency counts), rows whole once they fill the chip, and several rows a
  // block while its items would not keep 256 threads busy.
  const int items = p->hd / (vec ? E : 1);
  int rpb = 1, hpb = p->heads;
  while (hpb > 1 && (int64_t)p->rows * ((p->heads + hpb - 1) / hpb) < 512 && hpb * items > 2 * ROT_THREADS) hpb = (hpb + 1) / 2;
  while (hpb == p->heads && 2 * rpb * (half ? half : 1) <= ROT_TABLE && rpb * p->heads * items < 8 * ROT_THREADS && p->rows / rpb > 2048) rpb *= 2;
  const dim3 grid((unsigned)((p->rows + rpb - 1) / rpb), (unsigned)((p->heads + hpb - 1) / hpb));
#define LAUNCH(T, E, I) hipLaunchKernelGGL((rotary_kernel<T, E, I>), grid, dim3(ROT_THREADS), 0, (hipStream_t)stream, *p, rpb, hpb)
#define LAUNCH2(T, E) do { if (p->interleaved) LAUNCH(T, E, true); else LAUNCH(T, E, false); } while (0)
  if (p->f32) { if (vec) LAUNCH2(float, 4); else LAUNCH2(float, 1); }
  else { if (vec) LAUNCH2(bf16_raw, 8); else LAUNCH2(bf16_raw, 1); }
#undef LAUNCH2
#undef LAUNCH
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
