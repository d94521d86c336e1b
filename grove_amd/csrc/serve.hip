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
// where everything is aligned; E = 1 pair otherwise). Bound by memory: everything is read once and written once. 16384 rows x 40 heads x 128 in bf16:
// 68 us, 4.9 TB/s, what a large copy reaches (a thread per pair with its own fp64 angle: 207 us); 8 rows x 64 heads: 2.5 us, a launch.
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
// launch; a page that this launch hands out is taken from the free list again where a slot needs it, never from the table. Bound by the chain lengths ->
// sums -> entries: 3.5 us for 8 requests, 5.3 us for 512 with 19932 rows.
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
constexpr int VD_THREADS = 256, VD_WAVES = VD_THREADS / 64;

// Inclusive sum over the block in fp64; `total`: of all. Two barriers.
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

// Four consecutive values; `vec`: the row starts at a multiple of four values' bytes.
__device__ __forceinline__ void ld4(const float* p, bool vec, float (&v)[4]) {
  if (vec) {
    const f32x4_t x = *(const f32x4_t*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x[i];
  } else
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = p[i];
}
__device__ __forceinline__ void ld4(const bf16_raw* p, bool vec, float (&v)[4]) {
  if (vec) {
    const u32x2_t x = *(const u32x2_t*)p;
#pragma unroll
    for (int i = 0; i < 2; ++i) { v[2 * i] = bf_lo(x[i]); v[2 * i + 1] = bf_hi(x[i]); }
  } else
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = bf2f(p[i]);
}

__device__ __forceinline__ int drafts_of(const grove_verify_drafts_params& p, int b) { return p.count ? max(0, min(p.count[b], p.drafts)) : p.drafts; }

// The first refused draft of request b (n: none), for all threads of the block; s_a in LDS. One wave tests 64 drafts side by side.
template <typename T>
__device__ __forceinline__ int accept(const grove_verify_drafts_params& p, int b, int n, int* s_a) {
  if (threadIdx.x < 64) {
    const T* P = (const T*)p.p + b * p.sp_req;
    const T* Q = p.q ? (const T*)p.q + b * p.sq_req : nullptr;
    int a = n;
    for (int i0 = 0; i0 < n && a == n; i0 += 64) {
      const int i = i0 + threadIdx.x;
      bool refused = false;
      if (i < n) {
        const int x = p.draft[(int64_t)b * p.drafts + i];
        const float u = p.u[(int64_t)b * p.drafts + i];
        refused = x < 0 || x >= p.vocab;
        if (!refused) {
          const double q = Q ? (double)ld1(Q + i * p.sq_row + x) : 1.0;
          refused = !((double)u * q < (double)ld1(P + i * p.sp_row + x));
        }
      }
      const unsigned long long any = __ballot(refused);
      if (any) a = i0 + __builtin_ctzll(any);
    }
    if (threadIdx.x == 0) *s_a = a;
  }
  __syncthreads();
  return *s_a;
}

// What request b's last token is drawn from: r = max(p - q, 0) of the refused draft's row, or p itself (plain).
template <typename T>
struct rest_row {
  const T *P, *Q;
  int sure;  // a certain drafter's refused token: its mass is what is taken off
  bool vp, vq;
  __device__ rest_row(const grove_verify_drafts_params& p, int b, int a, bool plain) {
    P = (const T*)p.p + b * p.sp_req + a * p.sp_row;
    Q = !plain && p.q ? (const T*)p.q + b * p.sq_req + a * p.sq_row : nullptr;
    sure = !plain && !p.q ? p.draft[(int64_t)b * p.drafts + a] : -1;
    vp = ((uintptr_t)P & (4 * sizeof(T) - 1)) == 0;
    vq = ((uintptr_t)Q & (4 * sizeof(T) - 1)) == 0;
  }
  __device__ double one(int j) const {
    double r = (double)ld1(P + j);
    if (Q) r -= (double)ld1(Q + j);
    else if (j == sure) r -= 1.0;
    return r > 0 ? r : 0.0;
  }
  // the sum of [j0, j1), by a wave
  __device__ double sum(int j0, int j1) const {
    double s = 0;
    for (int base = j0; base < j1; base += 1024) {
      const int lane = threadIdx.x & 63;
      if (base + 1024 <= j1) {
        float x[4][4], y[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = base + 256 * k + 4 * lane;
          ld4(P + j, vp, x[k]);
          if (Q) ld4(Q + j, vq, y[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            double r = (double)x[k][i];
            if (Q) r -= (double)y[k][i];
            else if (base + 256 * k + 4 * lane + i == sure) r -= 1.0;
            s += r > 0 ? r : 0.0;
          }
      } else
        for (int j = base + lane; j < j1; j += 64) s += one(j);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    return s;
  }
};
__host__ __device__ inline int vd_chunk(int V) { return 1024 * ((V + (1 << 20) - 1) >> 20); }  // at most 1024 chunks
__host__ __device__ inline int vd_chunks(int V) { return (V + vd_chunk(V) - 1) / vd_chunk(V); }

// The token at `pick` of a row whose chunk sums are in LDS: the chunk by a scan over the sums, then element by element. -1: the row holds nothing.
struct draw_lds {
  double sums[1024], wsum[VD_WAVES], before;
  int low[VD_WAVES], last[VD_WAVES];
};
// Of 4 x 256 weights, 4 consecutive ones a thread: the first whose running sum (from `carry`) passes thr, else the last that is not 0, else -1; by
// ballots (atomics on one LDS word take their lanes one after the other). `sum`: of all; s.before, after a barrier: the sum before the one found.
// pick >= 0: thr becomes that part of the sum first.
__device__ int search(const double (&r)[4], double carry, float pick, double& thr, draw_lds& s, double& sum, bool& passed) {
  const int tid = threadIdx.x, w = tid >> 6;
  const double own = (r[0] + r[1]) + (r[2] + r[3]), before = carry + (block_scan(own, s.wsum, sum) - own);
  if (pick >= 0.f) thr = (double)pick * sum;
  int low = 4, last = -1;
  double c[5];
  c[0] = before;
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i + 1] = c[i] + r[i];
#pragma unroll
  for (int i = 3; i >= 0; --i)
    if (r[i] > 0) {
      if (last < 0) last = i;
      if (c[i + 1] > thr) low = i;
    }
  const unsigned long long lows = __ballot(low < 4), some = __ballot(last >= 0);
  const int l0 = lows ? __builtin_ctzll(lows) : 0, l1 = some ? 63 - __builtin_clzll(some) : 0;
  const int low_i = __shfl(low, l0, 64), last_i = __shfl(last, l1, 64);
  if ((tid & 63) == 0) {
    s.low[w] = lows ? (w * 64 + l0) * 4 + low_i : 1024;
    s.last[w] = some ? (w * 64 + l1) * 4 + last_i : -1;
  }
  __syncthreads();
  int lo = s.low[0], la = s.last[0];
#pragma unroll
  for (int i = 1; i < VD_WAVES; ++i) { lo = min(lo, s.low[i]); la = max(la, s.last[i]); }
  passed = lo < 1024;
  const int at = passed ? lo : la;
  if (at >= 0 && tid == at >> 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i == (at & 3)) s.before = c[i];
  }
  return at;
}
template <typename T>
__device__ int draw(const rest_row<T>& row, int V, float pick, draw_lds& s) {
  const int tid = threadIdx.x, chunk = vd_chunk(V), nchunk = vd_chunks(V);
  __syncthreads();  // the sums are there
  double r[4], total, part, thr = 0;
  bool passed;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = 4 * tid + i < nchunk ? s.sums[4 * tid + i] : 0.0;
  const int c = search(r, 0.0, pick, thr, s, total, passed);
  if (c < 0) return -1;
  __syncthreads();
  double carry = s.before;
  int last = -1;
  for (int j0 = c * chunk; j0 < min(V, (c + 1) * chunk); j0 += 1024) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = j0 + 4 * tid + i < V ? row.one(j0 + 4 * tid + i) : 0.0;
    const int at = search(r, carry, -1.f, thr, s, part, passed);
    if (at >= 0) last = j0 + at;
    if (passed) return last;
    carry += part;
    __syncthreads();
  }
  return last;
}

// Bound by memory for many requests (128 x 7 drafts over 128000: 27 us for 115 MB), by the chain drafts -> row -> chunk -> token for few (8 x 4 over 32008:
// 8.7 us in two launches; 16.5 us in one, where a CU reads the row).
// One block per request. SUMMED: the chunk sums and the number of accepted drafts come from verify_sums_kernel. Otherwise the block forms them; and in
// either case those of the target alone where the difference leaves nothing.
template <typename T, bool SUMMED>
__global__ __launch_bounds__(VD_THREADS) void verify_drafts_kernel(const grove_verify_drafts_params p) {
  __shared__ draw_lds s;
  __shared__ int s_a;
  const int tid = threadIdx.x, b = blockIdx.x, V = p.vocab, n = drafts_of(p, b), nchunk = vd_chunks(V), chunk = vd_chunk(V);
  const int a = SUMMED ? p.accepted[b] : accept<T>(p, b, n, &s_a);
  bool ready = SUMMED;
  if (SUMMED)
    for (int c = tid; c < nchunk; c += VD_THREADS) s.sums[c] = p.partial[(int64_t)b * nchunk + c];
  int token = -1;
  for (int plain = a < n ? 0 : 1; plain < 2 && token < 0; ++plain) {
    const rest_row<T> row(p, b, a, plain);
    if (!ready) {
      __syncthreads();
      for (int c = tid >> 6; c < nchunk; c += VD_WAVES) {
        const double sum = row.sum(c * chunk, min(V, (c + 1) * chunk));
        if ((tid & 63) == 0) s.sums[c] = sum;
      }
    }
    ready = false;
    token = draw(row, V, p.pick[b], s);
  }
  const int* draft = p.draft + (int64_t)b * p.drafts;
  for (int i = tid; i <= p.drafts; i += VD_THREADS) p.tokens[(int64_t)b * (p.drafts + 1) + i] = i < a ? draft[i] : i == a ? token : -1;
  if (!SUMMED && tid == 0) p.accepted[b] = a;
}

// A few blocks per request form the chunk sums (a CU reads some 22 GB/s, so one block takes 12 us over a vocabulary of 32008): each tests the drafts for
// itself, then a wave takes a chunk at a time.
template <typename T>
__global__ __launch_bounds__(256) void verify_sums_kernel(const grove_verify_drafts_params p, const int per) {
  __shared__ int s_a;
  const int b = blockIdx.y, V = p.vocab, n = drafts_of(p, b), nchunk = vd_chunks(V), chunk = vd_chunk(V);
  const int a = accept<T>(p, b, n, &s_a);
  const rest_row<T> row(p, b, a, a == n);
  for (int c = blockIdx.x * per + (threadIdx.x >> 6); c < min(nchunk, ((int)blockIdx.x + 1) * per); c += 4) {
    const double sum = row.sum(c * chunk, min(V, (c + 1) * chunk));
    if ((threadIdx.x & 63) == 0) p.partial[(int64_t)b * nchunk + c] = sum;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.accepted[b] = a;
}

}  // namespace

extern "C" int grove_rotary(const grove_rotary_params* p, void* stream) {
  GROVE_CHECK(p && p->rows >= 0 && p->rows <= 1 << 30 && p->heads >= 0 && p->hd > 0 && p->rot >= 0 && p->rot <= p->hd && (p->rot & 1) == 0 && (int64_t)p->heads * p->hd < (1 << 28),
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
  const dim3 grid((unsigned)p->requests);
  if (p->partial) {
    // a chunk for each wave of a block, several once that makes more than 2048 blocks
    GROVE_CHECK(p->requests <= 65535, GROVE_E_SHAPE, "verify_drafts: at most 65535 requests with a workspace");
    const int nchunk = vd_chunks(p->vocab);
    const int64_t want = ((int64_t)nchunk * p->requests + 2047) / 2048;
    const int per = want <= 4 ? 4 : (int)(want + 3) / 4 * 4;
    const dim3 parts((unsigned)((nchunk + per - 1) / per), (unsigned)p->requests);
    if (p->bf16) hipLaunchKernelGGL(verify_sums_kernel<bf16_raw>, parts, dim3(256), 0, (hipStream_t)stream, *p, per);
    else hipLaunchKernelGGL(verify_sums_kernel<float>, parts, dim3(256), 0, (hipStream_t)stream, *p, per);
    GROVE_LAUNCH_CHECK();
    if (p->bf16) hipLaunchKernelGGL((verify_drafts_kernel<bf16_raw, true>), grid, dim3(VD_THREADS), 0, (hipStream_t)stream, *p);
    else hipLaunchKernelGGL((verify_drafts_kernel<float, true>), grid, dim3(VD_THREADS), 0, (hipStream_t)stream, *p);
  } else {
    if (p->bf16) hipLaunchKernelGGL((verify_drafts_kernel<bf16_raw, false>), grid, dim3(VD_THREADS), 0, (hipStream_t)stream, *p);
    else hipLaunchKernelGGL((verify_drafts_kernel<float, false>), grid, dim3(VD_THREADS), 0, (hipStream_t)stream, *p);
  }
  GROVE_LAUNCH_CHECK();
  return GROVE_OK;
}
