// The paged 4-bit key / value cache (layout: grove_hip.h): quantise into pages, read back, attend.
#include "common.h"
#include <type_traits>

namespace {

__device__ __forceinline__ bool slot_of(const int* slots, int row, int rows, int page, int pages, int& pg, int& at) {
  const int s = row < rows ? slots[row] : -1;
  if (s < 0 || s >= (int64_t)pages * page) return false;
  pg = s / page;
  at = s - pg * page;
  return true;
}

// ---------------------------------------------------------------- into the pages and out of them
// HD / 8 lanes take one row of one head, 8 channels (16 bytes) each, so a wave holds 512 / HD consecutive rows: of a key row a lane's channels are one
// word of the cache, of a value row one nibble of eight places, and four lanes exchange bytes to have all the nibbles of two places each. Bound by
// memory for many rows (16387 rows x 8 heads x 128: in 23 us, 84 MB; out 17 us), by the chain slot -> row -> page for few (40 rows x 32 heads: 2 x 2.6 us).

// lane g's word holds the nibbles of channels 8 g + 0..7 (g = 2 j + half of the 16 places): a 4 x 4 transpose of bytes over the lanes j = 4 jq + 0..3
template <int CTRL> __device__ __forceinline__ int lanes(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }
constexpr int XOR1 = 0xB1, XOR2 = 0x4E, XOR3 = 0x1B, XOR7 = 0x141, XOR15 = 0x140;  // data-parallel moves within 16 lanes: no trip through LDS
__device__ __forceinline__ unsigned byte_transpose(unsigned w, int g) {
  unsigned t = lanes<XOR2>(w);
  w = (g & 2) ? __builtin_amdgcn_perm(t, w, 0x03070105) : __builtin_amdgcn_perm(t, w, 0x06020400);
  t = lanes<XOR3>(lanes<XOR7>(w));
  return (g & 4) ? __builtin_amdgcn_perm(t, w, 0x03020706) : __builtin_amdgcn_perm(t, w, 0x05040100);
}
__device__ __forceinline__ unsigned low_nibbles(unsigned w) {  // the low nibbles of the four bytes side by side
  w &= 0x0f0f0f0fu;
  w = (w | w >> 4) & 0x00ff00ffu;
  return (w | w >> 8) & 0xffffu;
}
__device__ __forceinline__ unsigned spread_nibbles(unsigned w) {  // and back
  w = (w | w << 8) & 0x00ff00ffu;
  return (w | w << 4) & 0x0f0f0f0fu;
}

// The eight codes of a lane, nibble i = channel i; and the row's scale and minimum. G lanes share the row.
// Minimum and maximum run on the bf16 bits as ordered integers (sign and magnitude -> two's complement), two at a time; infinities and NaN are the
// values outside +-0x7f7f. Quotients x / y: an approximate one, its exact remainder, one correction: right where x / y has few bits, as the ties of
// both roundings have (a bf16 of 8 bits times 15, a bf16 times k + 1/2), and off by no more than its last bit elsewhere.
template <int G>
__device__ __forceinline__ unsigned quantise(const u32x4_t x, unsigned& scale_min) {
  typedef __attribute__((ext_vector_type(2))) short s16x2_t;
  auto ordered = [](unsigned b) {
    const s16x2_t a = __builtin_bit_cast(s16x2_t, b);
    return a ^ ((a >> 15) & (s16x2_t){0x7fff, 0x7fff});
  };
  s16x2_t lo2 = ordered(x[0]), hi2 = lo2;
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    const s16x2_t o = ordered(x[i]);
    lo2 = __builtin_elementwise_min(lo2, o);
    hi2 = __builtin_elementwise_max(hi2, o);
  }
  int lo = min((int)lo2[0], (int)lo2[1]), hi = max((int)hi2[0], (int)hi2[1]);
  lo = min(lo, lanes<XOR1>(lo));
  hi = max(hi, lanes<XOR1>(hi));
  lo = min(lo, lanes<XOR2>(lo));
  hi = max(hi, lanes<XOR2>(hi));
  if constexpr (G >= 8) { lo = min(lo, lanes<XOR7>(lo)); hi = max(hi, lanes<XOR7>(hi)); }
  if constexpr (G >= 16) { lo = min(lo, lanes<XOR15>(lo)); hi = max(hi, lanes<XOR15>(hi)); }
  if constexpr (G >= 32) { lo = min(lo, __shfl_xor(lo, 16, 64)); hi = max(hi, __shfl_xor(hi, 16, 64)); }
  const unsigned lob = (unsigned)(lo ^ ((lo >> 15) & 0x7fff)) & 0xffffu, hib = (unsigned)(hi ^ ((hi >> 15) & 0x7fff)) & 0xffffu;
  const float lof = bf_lo(lob), span = bf_lo(hib) - lof;
  const bool none = hi >= 0x7f80 || lo <= (int)(short)0x807f || !(span < INFINITY);
  float q15 = span * (1.f / 15.f);
  q15 = fmaf(fmaf(-q15, 15.f, span), 1.f / 15.f, q15);
  const bf16_raw sb = none ? 0x7fc0 : span < 0x1p-100f ? 0 : f2bf(q15), mb = none ? 0x7fc0 : (bf16_raw)lob;
  scale_min = sb | ((unsigned)mb << 16);
  const float s = bf2f(sb), r = __builtin_amdgcn_rcpf(s);
  unsigned w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = ((i & 1) ? bf_hi(x[i >> 1]) : bf_lo(x[i >> 1])) - lof;
    float q = d * r;
    q = fmaf(fmaf(-q, s, d), r, q);
    w += __float_as_uint(fminf(q, 15.f) + 0x1p23f) << (4 * i);  // rounded to an integer in the last bits of 2^23 + c
  }
  unsigned off = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) off += 0x4b000000u << (4 * i);
  return (none || sb == 0) ? 0u : w - off;
}

template <int HD>
__global__ __launch_bounds__(256) void kv4_append_kernel(const grove_kv4_append_params p, const int vec) {
  constexpr int G = HD / 8, R = 64 / G;
  const int lane = threadIdx.x & 63, g = lane & (G - 1);
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // (rows of a wave, head), heads side by side
  const int head = (int)(unit % p.kv), row = (int)(unit / p.kv) * R + lane / G;
  if ((unit / p.kv) * R >= p.rows) return;
  int pg = 0, at = 0;
  const bool ok = slot_of(p.slots, row, p.rows, p.page, p.pages, pg, at);
  const int r = ok ? row : 0;
  u32x4_t x[2];
  const bf16_raw* kp = (const bf16_raw*)p.k + r * p.sk_row + head * p.sk_head + 8 * g;
  const bf16_raw* vp = (const bf16_raw*)p.v + r * p.sv_row + head * p.sv_head + 8 * g;
  if (vec) {
    x[0] = *(const u32x4_t*)kp;
    x[1] = *(const u32x4_t*)vp;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[0][i] = kp[2 * i] | ((unsigned)kp[2 * i + 1] << 16);
      x[1][i] = vp[2 * i] | ((unsigned)vp[2 * i + 1] << 16);
    }
  }
  unsigned sm[2];
  const unsigned wk = quantise<G>(x[0], sm[0]), wv = quantise<G>(x[1], sm[1]);
  const int64_t plane = (int64_t)pg * 2 * p.kv + head;
  unsigned char* kc = (unsigned char*)p.codes + plane * p.page * (HD / 2);
  unsigned char* vc = kc + (int64_t)p.kv * p.page * (HD / 2) + (at >> 2) * (2 * HD);
  if (ok) {
    // channels 0, 2, 4, 6 in the low half, 1, 3, 5, 7 in the high half
    unsigned e = wk & 0x0f0f0f0fu, o = (wk >> 4) & 0x0f0f0f0fu;
    e = (e | e >> 4) & 0x00ff00ffu;
    o = (o | o >> 4) & 0x00ff00ffu;
    const unsigned word = ((e | e >> 8) & 0xffffu) | (o | o >> 8) << 16;
    *(unsigned*)(kc + at * (HD / 2) + ((g & 3) * (HD / 32) + (g >> 2)) * 4) = word;
    if (g == 0) {
      ((unsigned*)p.scales)[plane * p.page + at] = sm[0];
      ((unsigned*)p.scales)[(plane + p.kv) * p.page + at] = sm[1];
    }
  }
  const int tp = (at >> 1) & 1, par = at & 1;
  if constexpr (HD == 32) {
    const unsigned t = lanes<XOR2>(wv), a = (g & 2) ? t >> 16 : wv, b = (g & 2) ? wv >> 16 : t;  // j = 0 and 1 of this lane's four places
    if (ok)
#pragma unroll
      for (int i = 0; i < 4; ++i) vc[(8 * (g & 1) + 2 * (g & 2) + i) * 4 + par * 2 + tp] = (unsigned char)((a >> (4 * i) & 15) | (b >> (4 * i) & 15) << 4);
  } else {
    const unsigned w = byte_transpose(wv, g);
    const int m = 8 * (g & 1) + (g & 6), jq = g >> 3;
    bf16_raw* y = (bf16_raw*)(vc + m * (HD / 8) + (jq * 2 + tp) * 4 + par * 2);
    if (ok) {
      y[0] = (bf16_raw)low_nibbles(w);
      y[HD / 16] = (bf16_raw)low_nibbles(w >> 4);
    }
  }
}

template <int HD, typename T>
__global__ __launch_bounds__(256) void kv4_read_kernel(const grove_kv4_read_params p) {
  constexpr int G = HD / 8, R = 64 / G;
  const int lane = threadIdx.x & 63, g = lane & (G - 1);
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int head = (int)(unit % p.kv), row = (int)(unit / p.kv) * R + lane / G;
  if ((unit / p.kv) * R >= p.rows) return;
  int pg = 0, at = 0;
  const bool ok = slot_of(p.slots, row, p.rows, p.page, p.pages, pg, at);
  const int64_t plane = (int64_t)pg * 2 * p.kv + head;
  const unsigned char* kc = (const unsigned char*)p.codes + plane * p.page * (HD / 2);
  const unsigned char* vc = kc + (int64_t)p.kv * p.page * (HD / 2) + (at >> 2) * (2 * HD);
  const unsigned sk = ((const unsigned*)p.scales)[plane * p.page + at], sv = ((const unsigned*)p.scales)[(plane + p.kv) * p.page + at];
  const unsigned word = *(const unsigned*)(kc + at * (HD / 2) + ((g & 3) * (HD / 32) + (g >> 2)) * 4);
  const unsigned wk = spread_nibbles(word & 0xffffu) | spread_nibbles(word >> 16) << 4;
  const int tp = (at >> 1) & 1, par = at & 1;
  unsigned wv = 0;
  if constexpr (HD == 32) {
    unsigned a = 0, b = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned c = vc[(8 * (g & 1) + 2 * (g & 2) + i) * 4 + par * 2 + tp];
      a |= (c & 15) << (4 * i);
      b |= (c >> 4) << (4 * i);
    }
    const unsigned give = (g & 2) ? a : b, t = lanes<XOR2>(give);  // j = 0 goes to the lane with j = 0, j = 1 to the other
    wv = (g & 2) ? t | b << 16 : a | t << 16;
  } else {
    const int m = 8 * (g & 1) + (g & 6), jq = g >> 3;
    const bf16_raw* y = (const bf16_raw*)(vc + m * (HD / 8) + (jq * 2 + tp) * 4 + par * 2);
    wv = byte_transpose(spread_nibbles(y[0]) | spread_nibbles(y[HD / 16]) << 4, g);
  }
  if (row >= p.rows) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const unsigned w = which ? wv : wk, sm = which ? sv : sk;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = ok ? fmaf((float)(w >> (4 * i) & 15), bf_lo(sm), bf_hi(sm)) : 0.f;
    T* y = (T*)(which ? p.v : p.k) + ((int64_t)row * p.kv + head) * HD + 8 * g;
    if constexpr (sizeof(T) == 4) {
      *(f32x4_t*)y = (f32x4_t){v[0], v[1], v[2], v[3]};
      *(f32x4_t*)(y + 4) = (f32x4_t){v[4], v[5], v[6], v[7]};
    } else {
      *(u32x4_t*)y = (u32x4_t){pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7])};
    }
  }
}

// ---------------------------------------------------------------- attention over 4-bit pages
// A block of four waves takes one (request, key / value head, range of keys) and up to 16 CT query columns: the group's query heads of the
// request's new tokens side by side (column = token * group + head). 32 keys at a time and wave, from two 16-key parts of a page:
//   S^T[key, col] = sum_c K[key, c] q[col, c]   A = keys (16) x 32 channels, B = columns: the codes go to the matrix unit as bf16 16 + c, which a
//     shift and one and-or make of a nibble pair (exact; the offset is taken off with the row's minimum), so a key costs no multiply for its scale:
//     z = (alpha' s) raw + (m - 16 s) (alpha' sum q), in units of log2.
//   O^T[c, col] += sum_key V[key, c] (P s)[key, col]   A = channels (16) x 32 keys, B = the scores' own registers: the accumulator of S^T holds keys
//     4 h + i of either part in lane (col, h), and the values' four-token order gives the A operand the same keys. P s goes in as two bf16 parts
//     (hi + lo, 2^-17), the minimum's share sum P (m - 16 s) is one number per column.
// Bound, at hd 128: 32 contexts of up to 32768 keys under 4 heads a group, one token each (607 MB): 123 us and 4 for the join, 4.8 TB/s, what a large
// copy reaches. 32 columns and more: by ragged lengths and by the chain product, softmax, product of a tile with a wave or two on a SIMD (64 requests x 8
// tokens x 4 heads over up to 4096 keys: 71 us for 167 MB, of which a wave lives half; vector units 37 % busy, matrix units 15; even lengths: 46 us).
// hd 64 and 32: by the work per tile, at half and a quarter of the bytes (53 us for 168 MB, 45 for 93; vector units 57 %). Few short contexts: by the chain
// lengths -> page -> tile -> output, 5 us, 7 with two column tiles, and 3 for the join (one context of 703 keys, 32 heads: 7.7 us in 8 blocks a head).
// The tiles travel global -> LDS (LDS-DMA) into a ring of kv4_slots slots per wave: several tiles per wave are in flight without a register held
// for them. At hd 128 and 256 every lane takes back the bytes that it asked for, side by side in lane order: no bank conflicts. No barriers: a wave
// reads only its own ring. Waits are counted: a tile is kv4_ops vector memory operations.
constexpr int kv4_part(int hd) { return 64 * (hd / 8); }              // bytes of 16 keys' codes
constexpr int kv4_bytes(int hd) { return 4 * kv4_part(hd) + 256; }    // of a tile: two parts of keys, two of values, scales
constexpr int kv4_ops(int hd) { return hd / 32 + 1; }
constexpr int kv4_slots(int hd, int ct) { return hd == 256 ? (ct == 1 ? 2 : 4) : hd == 128 ? (ct == 2 ? 4 : 3) : 4; }

template <int HD>
struct kv4_tile {
  unsigned k[2][HD / 32], v[2][HD / 32];
  u32x4_t ks[2], vs[2];
};

__device__ __forceinline__ void dma16(const void* g, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
__device__ __forceinline__ void dma4(const void* g, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)lds, 4, 0, 0);
}
// Two parts' codes and their scales from the ring, waited for in place (the compiler would wait for every load in flight). O: offset of the codes
// within the tile, OS: of the scales.
template <int HD, int O, int OS>
__device__ __forceinline__ void ring_read(unsigned a, unsigned as, unsigned (&w)[2][HD / 32], u32x4_t (&s)[2]) {
  if constexpr (HD == 32) {
    asm volatile("ds_read_b32 %0, %4 offset:%6\n\tds_read_b32 %1, %4 offset:%7\n\tds_read_b128 %2, %5 offset:%8\n\tds_read_b128 %3, %5 offset:%9\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(w[0][0]), "=&v"(w[1][0]), "=&v"(s[0]), "=&v"(s[1])
                 : "v"(a), "v"(as), "n"(O), "n"(O + 256), "n"(OS), "n"(OS + 64) : "memory");
  } else if constexpr (HD == 64) {
    u32x2_t x[2];
    asm volatile("ds_read_b64 %0, %4 offset:%6\n\tds_read_b64 %1, %4 offset:%7\n\tds_read_b128 %2, %5 offset:%8\n\tds_read_b128 %3, %5 offset:%9\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(s[0]), "=&v"(s[1])
                 : "v"(a), "v"(as), "n"(O), "n"(O + 512), "n"(OS), "n"(OS + 64) : "memory");
#pragma unroll
    for (int u = 0; u < 2; ++u) { w[u][0] = x[u][0]; w[u][1] = x[u][1]; }
  } else {
    constexpr int N = HD / 128;
    u32x4_t x[2][N];
    if constexpr (N == 1) {
      asm volatile("ds_read_b128 %0, %4 offset:%6\n\tds_read_b128 %1, %4 offset:%7\n\tds_read_b128 %2, %5 offset:%8\n\tds_read_b128 %3, %5 offset:%9\n\t"
                   "s_waitcnt lgkmcnt(0)"
                   : "=&v"(x[0][0]), "=&v"(x[1][0]), "=&v"(s[0]), "=&v"(s[1])
                   : "v"(a), "v"(as), "n"(O), "n"(O + 1024), "n"(OS), "n"(OS + 64) : "memory");
    } else {
      asm volatile("ds_read_b128 %0, %6 offset:%8\n\tds_read_b128 %1, %6 offset:%9\n\tds_read_b128 %2, %6 offset:%10\n\tds_read_b128 %3, %6 offset:%11\n\t"
                   "ds_read_b128 %4, %7 offset:%12\n\tds_read_b128 %5, %7 offset:%13\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(x[0][0]), "=&v"(x[0][N - 1]), "=&v"(x[1][0]), "=&v"(x[1][N - 1]), "=&v"(s[0]), "=&v"(s[1])
                   : "v"(a), "v"(as), "n"(O), "n"(O + 1024), "n"(O + 2 * 1024), "n"(O + 3 * 1024), "n"(OS), "n"(OS + 64) : "memory");
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) w[u][i] = x[u][i / 4][i % 4];
  }
}

// Nibble j of either half of a word as a pair of bf16 16 + c: the nibble on mantissa bits 3..6 below the exponent of 16. The two constants come
// from registers that the compiler cannot look into: as literals they would not fit into one v_and_or_b32, and take two instructions.
struct code_consts { unsigned mask, base; };
__device__ __forceinline__ code_consts get_code_consts() {
  code_consts k;
  asm("s_mov_b32 %0, 0x780078" : "=s"(k.mask));
  asm("v_mov_b32 %0, 0x41804180" : "=v"(k.base));
  return k;
}
__device__ __forceinline__ unsigned code_pair(unsigned w, int j, const code_consts k) {
  const unsigned x = j == 0 ? w << 3 : w >> (4 * j - 3);
  return (x & k.mask) | k.base;
}
__device__ __forceinline__ bf16x8_t frag(unsigned a, unsigned b, unsigned c, unsigned d) { return __builtin_bit_cast(bf16x8_t, (u32x4_t){a, b, c, d}); }

constexpr float NEG = -INFINITY;

constexpr int kv4_waves(int hd, int ct) { return hd * ct <= 128 ? 3 : hd == 256 && ct == 2 ? 1 : 2; }  // a SIMD's, which their registers have to leave room for
// With 64 columns of 128 the queries stay in LDS, in the operand's order, and are read per tile: in registers they cost the second wave of a SIMD
// (64 requests x 5 tokens x 8 heads a group over 2048 keys: 85 us, in LDS 67). At 256 x 32 a single wave with its queries in registers and twice the
// ring is the faster one (72 us against 84).
constexpr bool kv4_q_lds(int hd, int ct) { return hd == 128 && ct == 4; }
constexpr int kv4_lds(int hd, int ct) { return 4 * kv4_slots(hd, ct) * kv4_bytes(hd) + (kv4_q_lds(hd, ct) ? 32 * hd * ct + 64 * ct : 0); }

template <int HD, int CT>
__global__ __launch_bounds__(256, kv4_waves(HD, CT)) void kv4_attn_kernel(const grove_kv4_attn_params p, const int shift) {
  constexpr int NK = HD / 32, NJ = HD / 16, CG = HD == 256 || CT < 2 ? 1 : 2;  // CG tiles of columns hand their outputs through LDS at a time
  constexpr bool QL = kv4_q_lds(HD, CT);
  constexpr int S = kv4_slots(HD, CT), BYTES = kv4_bytes(HD), OPS = kv4_ops(HD), PART = kv4_part(HD);
  static_assert(kv4_lds(HD, CT) >= (int)sizeof(float) * 4 * 16 * CG * (HD + 4), "the outputs pass through the rings' memory");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  __shared__ float s_m[4][16 * CT], s_l[4][16 * CT], s_c[4][16 * CT];
  float(*s_o)[16 * CG][HD + 4] = (float(*)[16 * CG][HD + 4])smem;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, h = lane >> 4;
  const int G = p.heads / p.kv, chunks = gridDim.y / p.kv, hk = blockIdx.y / chunks, cc = blockIdx.y - hk * chunks, b = blockIdx.z, sp = blockIdx.x;
  typedef const __attribute__((address_space(4))) int* scalar_ints;  // scalar loads: of inputs that nothing writes meanwhile
  const scalar_ints cu_q = (scalar_ints)(uintptr_t)p.cu_q;
  const int q_lo = cu_q[b], q_hi = cu_q[b + 1], kv_len = ((scalar_ints)(uintptr_t)p.kv_len)[b];
  if (p.fresh && p.n_split == 1 && b == 0 && cc == 0) {  // a new result's rows of no request
    const int r0 = max(0, min(p.cu_q[0], p.rows)), r1 = max(r0, min(p.cu_q[p.requests], p.rows));
    for (int64_t e = tid; e < (int64_t)(r0 + p.rows - r1) * G * HD; e += 256) {
      const int r = (int)(e / (G * HD));
      ((bf16_raw*)p.out)[(r < r0 ? r : r1 + r - r0) * p.so_row + (int64_t)hk * G * HD + e % (G * HD)] = 0;
    }
  }
  const int t0 = max(0, min(q_lo, p.rows)), t1 = max(t0, min(q_hi, p.rows)), n = t1 - t0;
  const int cols = min(n, p.max_q) * G, col0 = cc * 16 * CT;
  if (n > p.max_q && cc == chunks - 1) {  // more new tokens than the call allows for: NaN, not what the memory held
    for (int e = tid; e < (n - p.max_q) * G; e += 256) {
      const int64_t row = t0 + p.max_q + e / G, head = hk * G + e % G;
      if (p.n_split > 1) {
        float* ml = p.partial + (int64_t)p.rows * p.heads * p.n_split * HD + ((row * p.heads + head) * p.n_split + sp) * 2;
        ml[0] = 0.f;
        ml[1] = NAN;
      } else
        for (int c = 0; c < HD / 2; ++c) ((unsigned*)((bf16_raw*)p.out + row * p.so_row + head * HD))[c] = 0x7fc07fc0u;
    }
  }
  if (col0 >= cols) return;
  const int64_t room = (int64_t)p.max_pages << shift;
  const int base = (int)min((int64_t)max(kv_len, 0), room) - (q_hi - t0) + 1;  // token i sees base + i keys (of all its new tokens, also those past `rows`)
  const int seen_all = max(0, base + col0 / G), seen_any = max(0, base + (min(cols, col0 + 16 * CT) - 1) / G);
  const int tiles = (seen_any + 31) >> 5, per = (tiles + p.n_split - 1) / p.n_split, tile0 = sp * per, tile1 = min(tiles, tile0 + per);

  // the columns' queries: asked for after the page numbers and before the first tiles, used when those are on their way
  bf16x8_t q[QL ? 1 : CT][NK];  // (QL: of the column tile that this wave puts into LDS)
  auto ask_q = [&]() {
#pragma unroll
    for (int ct = 0; ct < (QL ? 1 : CT); ++ct) {
      const int c = col0 + (QL ? w : ct) * 16 + n16, i = c / G;
      const bf16_raw* x = (const bf16_raw*)p.q + (t0 + i) * p.sq_row + (int64_t)(hk * G + c - i * G) * p.sq_head + 8 * h;
#pragma unroll
      for (int t = 0; t < NK; ++t) {
        u32x4_t r = {0, 0, 0, 0};
        if (c < cols) r = *(const u32x4_t*)(x + 32 * t);
        q[ct][t] = __builtin_bit_cast(bf16x8_t, r);
      }
    }
  };
  float qs[QL ? 1 : CT], ref[CT], l[CT], cst[CT];  // ref: taken off the scores, -inf before the column's first key
  const float a2 = p.alpha * 1.44269504088896340736f;
  char* q_lds = smem + 4 * S * BYTES;
  auto use_q = [&]() {
#pragma unroll
    for (int ct = 0; ct < (QL ? 1 : CT); ++ct) {
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < NK; ++t) {
        const u32x4_t r = __builtin_bit_cast(u32x4_t, q[ct][t]);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += bf_lo(r[e]) + bf_hi(r[e]);
        if (QL && w < CT) *(u32x4_t*)(q_lds + ((w * NK + t) * 64 + lane) * 16) = r;
      }
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      qs[ct] = sum * a2;
      if (QL && w < CT && h == 0) ((float*)(q_lds + CT * NK * 1024))[w * 16 + n16] = qs[ct];
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) ref[ct] = NEG;
    if constexpr (QL) __syncthreads();
  };
  const unsigned q_at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)q_lds + lane * 16;
  const unsigned qs_at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)q_lds + CT * NK * 1024 + n16 * 4;
  auto q_of = [&](int ct, bf16x8_t (&f)[NK], float& sum) {
    const unsigned at = q_at + ct * NK * 1024;
    static_assert(!QL || NK == 4, "four operands a column tile");
    asm volatile("ds_read_b128 %0, %5 offset:%7\n\tds_read_b128 %1, %5 offset:%8\n\tds_read_b128 %2, %5 offset:%9\n\tds_read_b128 %3, %5 offset:%10\n\t"
                 "ds_read_b32 %4, %6\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1 % NK]), "=&v"(f[2 % NK]), "=&v"(f[3 % NK]), "=&v"(sum)
                 : "v"(at), "v"(qs_at + ct * 64), "n"(0), "n"(1024), "n"(2 * 1024), "n"(3 * 1024) : "memory");
  };
  // page numbers by scalar loads (the constant address space), asked for one tile ahead of their use
  const scalar_ints row = (scalar_ints)(uintptr_t)(p.table + b * p.ld_table);
  const int P = 1 << shift;
  const int64_t page_rows = (int64_t)2 * p.kv << shift, v_rows = (int64_t)p.kv << shift;  // cache rows of a page, and from its keys to its values
  const unsigned char* codes = (const unsigned char*)p.codes + ((int64_t)hk << shift) * (HD / 2);
  const unsigned* scales = (const unsigned*)p.scales + ((int64_t)hk << shift);
  const code_consts kc = get_code_consts();
  const int k_off = n16 * (HD / 2) + h * (HD / 8), v_off = h * (2 * HD) + n16 * (HD / 8);
  char* ring = smem + w * S * BYTES;
  const unsigned ring_at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)ring;
  int ask[2], ahead, to;  // the tile to be asked for next, and its slot
  unsigned bad = 0;                       // two bits a slot: a part whose page is not one of the cache (its keys are masked, its loads go to page 0)
  auto ask_pages = [&]() {
#pragma unroll
    for (int u = 0; u < 2; ++u) ask[u] = row[min((ahead * 32 + 16 * u) >> shift, p.max_pages - 1)];
  };
  auto issue = [&]() {
    char* slot = ring + to * BYTES;
    int64_t at[2];
    unsigned miss = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bool ok = (ask[u] >= 0) & (ask[u] < p.pages);
      miss |= ok ? 0u : 1u << u;
      at[u] = (int64_t)(ok ? ask[u] : 0) * page_rows + ((ahead * 32 + 16 * u) & (P - 1));
    }
    if constexpr (HD >= 128) {  // a lane's pieces for itself: 16 bytes of each part's keys and values
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < HD / 128; ++i) {
          dma16(codes + at[u] * (HD / 2) + k_off + 16 * i, slot + u * PART + 1024 * i);
          dma16(codes + (at[u] + v_rows) * (HD / 2) + v_off + 16 * i, slot + (2 + u) * PART + 1024 * i);
        }
    } else if constexpr (HD == 64) {  // both parts' 512 bytes in one load, in memory's order
      const int64_t mine = lane < 32 ? at[0] : at[1];
      dma16(codes + mine * 32 + (lane & 31) * 16, slot);
      dma16(codes + (mine + v_rows) * 32 + (lane & 31) * 16, slot + 2 * PART);
    } else {  // all four parts' 256 bytes
      dma16(codes + (((h & 1) ? at[1] : at[0]) + (h >= 2 ? v_rows : 0)) * 16 + n16 * 16, slot);
    }
    dma4(scales + ((h & 1) ? at[1] : at[0]) + (h >= 2 ? v_rows : 0) + n16, slot + 4 * PART);  // keys' parts 0, 1, values' parts 0, 1
    bad = (bad & ~(3u << (2 * to))) | miss << (2 * to);
    to = to == S - 1 ? 0 : to + 1;
    ahead += 4;
    ask_pages();
  };
  kv4_tile<HD> T;

  // A wave's tiles. A column's reference is the maximum of its first keys; the accumulators are never rescaled: where a later score passes it by 24
  // (P <= 2^24 loses nothing in fp32) the wave starts again with that score's reference. Scores that far above a wave's first 32 keys' are rare, and
  // rescaling in the loop costs a second set of registers for the accumulators (57 of them at CT = 2) or a copy of each per tile. The second start
  // reads the keys alone, for the references that hold to the end: scores that climb along the context cost three passes, not one per climb (8
  // requests of 8192 keys that climb by 0.32 a key: 73 us -> 38, with 5 tokens each 218 -> 59, against 23 and 36 without a climb; the test costs 1 %).
  f32x4_t acc[CT][NJ];
  int tile, from;
  bool keys_only = false;
  float z[CT][8], top[CT];
  auto raise = [&]() -> bool {  // new references for the columns whose scores passed theirs; true: something was summed with an old one
    bool again = false;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float t = fmaxf(top[ct], __shfl_xor(top[ct], 16, 64));
      t = fmaxf(t, __shfl_xor(t, 32, 64));
      const bool up = t - 24.f > ref[ct];
      again |= up && ref[ct] != NEG;  // (a column's first keys leave nothing to do again)
      ref[ct] = up ? t : ref[ct];
    }
    return __any(again);
  };
  auto run = [&]() -> int {  // 0: done, 1: to be started again, 2: left at a tile for new references
    while (tile < tile1) {
      if (ahead - tile == 4 * (S - 1)) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(OPS * (S - 2)) : "memory");  // the tiles behind this one may be on their way
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                                                  // the last ones
      const unsigned slot = ring_at + from * BYTES, at_scales = slot + 16 * h;
      const unsigned at_keys = slot + (HD < 128 ? n16 * (HD / 2) + h * (HD / 8) : lane * 16), at_values = slot + lane * (HD < 128 ? HD / 8 : 16);
      ring_read<HD, 0, 4 * PART>(at_keys, at_scales, T.k, T.ks);
      // One part's operands at a time, both where there is one column tile: unpacked all at once they would take the registers of another wave. The
      // products of different tiles take turns, so that none waits for the one before it.
      constexpr int UG = CT == 1 && HD <= 128 ? 2 : 1;
#pragma unroll
      for (int u0 = 0; u0 < 2; u0 += UG) {
        __builtin_amdgcn_sched_barrier(0);
        bf16x8_t kf[UG][NK];
#pragma unroll
        for (int u = 0; u < UG; ++u)
#pragma unroll
          for (int t = 0; t < NK; ++t) {
            const unsigned x = T.k[u0 + u][t];
            kf[u][t] = frag(code_pair(x, 0, kc), code_pair(x, 1, kc), code_pair(x, 2, kc), code_pair(x, 3, kc));
          }
        auto score = [&](int ct, int u, const f32x4_t raw, float qsum) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float s = bf_lo(T.ks[u][i]), mn = bf_hi(T.ks[u][i]);
            z[ct][4 * u + i] = fmaf(raw[i], a2 * s, fmaf(-16.f, s, mn) * qsum);
          }
        };
        if constexpr (QL) {
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            bf16x8_t qf[NK];
            float qsum;
            q_of(ct, qf, qsum);
            f32x4_t raw = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < NK; ++t) raw = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[0][t], qf[t], raw, 0, 0, 0);
            score(ct, u0, raw, qsum);
          }
        } else {
          f32x4_t raw[UG][CT];
#pragma unroll
          for (int t = 0; t < NK; ++t)
#pragma unroll
            for (int u = 0; u < UG; ++u)
#pragma unroll
              for (int ct = 0; ct < CT; ++ct)
                raw[u][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[u][t], q[ct][t], t ? raw[u][ct] : (f32x4_t){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
          for (int u = 0; u < UG; ++u)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) score(ct, u0 + u, raw[u][ct], qs[ct]);
        }
      }
      const unsigned miss = bad >> (2 * from) & 3;
      const bool masked = ((tile + 1) * 32 > seen_all) | (miss != 0);
      auto limit = [&](int ct) {  // of keys that a column sees
        const int c = col0 + ct * 16 + n16;
        return c < cols ? base + c / G : 0;
      };
      auto sees = [&](int lim, int i) { return (tile * 32 + 16 * (i >> 2) + 4 * h + (i & 3) < lim) & ((miss >> (i >> 2) & 1) == 0); };
      if (masked) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const int lim = limit(ct);
#pragma unroll
          for (int i = 0; i < 8; ++i) z[ct][i] = sees(lim, i) ? z[ct][i] : NEG;
        }
      }
      bool grow = false;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        top[ct] = z[ct][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top[ct] = fmaxf(top[ct], z[ct][i]);
        grow |= top[ct] - 24.f > ref[ct];
      }
      if (__any(grow)) {
        if constexpr (HD * CT >= 512) return 2;  // (outside of the loop: inside it the paths' joined registers do not fit)
        if (raise() && !keys_only) return 1;
      }
      if (ahead < tile1) issue();
      if (keys_only) {
        tile += 4;
        from = from == S - 1 ? 0 : from + 1;
        continue;
      }
      ring_read<HD, 2 * PART, 4 * PART + 128>(at_values, at_scales, T.v, T.vs);
      if (masked) {  // 0 times a minimum that is no number would reach the columns that do not see its row: it goes, and those that see it become NaN
        unsigned odd = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned sm = T.vs[i >> 2][i & 3];
          const bool is = !(fabsf(fmaf(-16.f, bf_lo(sm), bf_hi(sm))) < INFINITY);  // (what is used below: a finite scale of 2^124 overflows it)
          odd |= is ? 1u << i : 0u;
          T.vs[i >> 2][i & 3] = is ? 0u : sm;
        }
        if (__any(odd != 0)) {
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            const int lim = limit(ct);
#pragma unroll
            for (int i = 0; i < 8; ++i) l[ct] = ((odd >> i & 1) != 0) & sees(lim, i) ? NAN : l[ct];
          }
        }
      }
      bf16x8_t hi[CT], lo[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const float off = ref[ct] == NEG ? 0.f : ref[ct];
        unsigned a[4], c[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float ps[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = __builtin_amdgcn_exp2f(z[ct][4 * u + i] - off);
            const float s = bf_lo(T.vs[u][i]), mn = fmaf(-16.f, s, bf_hi(T.vs[u][i]));
            l[ct] += e;
            ps[i] = e * s;
            cst[ct] = fmaf(e, mn, cst[ct]);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            a[2 * u + i] = pack2bf(ps[2 * i], ps[2 * i + 1]);
            c[2 * u + i] = pack2bf(ps[2 * i] - bf_lo(a[2 * u + i]), ps[2 * i + 1] - bf_hi(a[2 * u + i]));
          }
        }
        hi[ct] = frag(a[0], a[1], a[2], a[3]);
        lo[ct] = frag(c[0], c[1], c[2], c[3]);
      }
#pragma unroll
      for (int j = 0; j < NJ; j += 2) {
        __builtin_amdgcn_sched_barrier(0);
        bf16x8_t vf[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if constexpr (HD == 32) vf[k] = frag(code_pair(T.v[0][0], k, kc), code_pair(T.v[0][0], k + 2, kc), code_pair(T.v[1][0], k, kc), code_pair(T.v[1][0], k + 2, kc));
          else {
            const int o = (j >> 2) * 2, jn = (j & 3) + k;
            vf[k] = frag(code_pair(T.v[0][o], jn, kc), code_pair(T.v[0][o + 1], jn, kc), code_pair(T.v[1][o], jn, kc), code_pair(T.v[1][o + 1], jn, kc));
          }
        }
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) acc[ct][j + k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[k], part ? lo[ct] : hi[ct], acc[ct][j + k], 0, 0, 0);
      }
      tile += 4;
      from = from == S - 1 ? 0 : from + 1;
    }
    return 0;
  };
  auto start = [&]() {
    tile = ahead = tile0 + w;
    to = from = 0;
    bad = 0;
    if (ahead < tile1) ask_pages();
  };
  auto fill = [&]() {  // (rolled: what a block runs once is fetched cold, and its length counts)
#pragma unroll 1
    for (int i = 0; i < S - 1 && ahead < tile1; ++i) issue();
  };
  start();
  ask_q();
  fill();
  use_q();
  for (int starts = 0;; ++starts) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      l[ct] = cst[ct] = 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[ct][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    int left;
    keys_only = starts == 2;
    while ((left = run()) == 2 && (!raise() || keys_only)) {
    }
    if (left == 0 && !keys_only) break;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the tiles in flight land before their slots are asked for again
    start();
    fill();
  }

  // the four waves' results: one maximum per column, the outputs through LDS
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] += __shfl_xor(l[ct], 16, 64);
    l[ct] += __shfl_xor(l[ct], 32, 64);
    cst[ct] += __shfl_xor(cst[ct], 16, 64);
    cst[ct] += __shfl_xor(cst[ct], 32, 64);
    if (h == 0) {
      s_m[w][ct * 16 + n16] = ref[ct];
      s_l[w][ct * 16 + n16] = l[ct];
      s_c[w][ct * 16 + n16] = cst[ct];
    }
  }
  __syncthreads();  // (the rings are read, nothing is in flight: their memory takes the outputs)
  auto joint = [&](int col) { return fmaxf(fmaxf(s_m[0][col], s_m[1][col]), fmaxf(s_m[2][col], s_m[3][col])); };
  auto part = [&](float mw, float M) { return mw == NEG ? 0.f : __builtin_amdgcn_exp2f(mw - M); };
  constexpr int EL = HD / 16;  // 16 threads a column
  const int och = (tid & 15) * EL;
#pragma unroll
  for (int g0 = 0; g0 < CT; g0 += CG) {
    if (g0) __syncthreads();
#pragma unroll
    for (int ct = g0; ct < g0 + CG; ++ct) {
      const float f = part(s_m[w][ct * 16 + n16], joint(ct * 16 + n16));
#pragma unroll
      for (int j = 0; j < NJ; ++j) *(f32x4_t*)&s_o[w][(ct - g0) * 16 + n16][16 * j + 4 * h] = acc[ct][j] * f;
    }
    __syncthreads();
#pragma unroll 1
    for (int oc = tid >> 4; oc < 16 * CG; oc += 16) {
      const int col = g0 * 16 + oc, c = col0 + col, i = c / G;
      if (c >= cols) break;
      const float M = joint(col);
      float L = 0.f, C = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float fk = part(s_m[k][col], M);
        L += fk * s_l[k][col];
        C += fk * s_c[k][col];
      }
      float o[EL];
#pragma unroll
      for (int e = 0; e < EL; ++e) o[e] = C + ((s_o[0][oc][och + e] + s_o[1][oc][och + e]) + (s_o[2][oc][och + e] + s_o[3][oc][och + e]));
      if (p.n_split > 1) {
        const int64_t unit = (int64_t)(t0 + i) * p.heads + hk * G + (c - i * G), at = unit * p.n_split + sp;
        if ((tid & 15) == 0) {
          float* ml = p.partial + (int64_t)p.rows * p.heads * p.n_split * HD + at * 2;
          ml[0] = M;
          ml[1] = L;
        }
        float* y = p.partial + at * HD + och;
#pragma unroll
        for (int e = 0; e < EL; ++e) y[e] = o[e];
      } else {
        unsigned* y = (unsigned*)((bf16_raw*)p.out + (t0 + i) * p.so_row + (int64_t)(hk * G + c - i * G) * HD + och);
        const bool some = L > 0.f || L != L;
        const float r = 1.f / L;
#pragma unroll
        for (int e = 0; e < EL / 2; ++e) y[e] = some ? pack2bf(o[2 * e] * r, o[2 * e + 1] * r) : 0u;
      }
    }
  }
}

// Joins the partial results of at most 64 splits: a lane per split for the weights, then WAVES waves over the splits of one (row, query head), eight
// partial outputs in flight. One wave each where the splits are few.
template <int HD, int WAVES>
__global__ __launch_bounds__(256) void kv4_join_kernel(const grove_kv4_attn_params p) {
  constexpr int NC = HD < 64 ? 1 : HD / 64;
  __shared__ float s_o[4][HD];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, S = p.n_split;
  const int64_t unit = WAVES == 1 ? (int64_t)blockIdx.x * 4 + w : (int64_t)blockIdx.x;
  if (unit >= (int64_t)p.rows * p.heads) return;
  const int row = (int)(unit / p.heads), head = (int)(unit - (int64_t)row * p.heads);
  // (everything is asked for at once: the partial results are there to read whether or not the row is a request's)
  const float* ml = p.partial + (int64_t)p.rows * p.heads * S * HD + unit * S * 2;
  const float* part = p.partial + unit * S * HD + min(lane, HD - 1);
  const int r0 = p.cu_q[0], r1 = p.cu_q[p.requests];
  const float m_in = ml[2 * min(lane, S - 1)], l_in = ml[2 * min(lane, S - 1) + 1];
  float x[8][NC];
  auto ask = [&](int s0) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int i = 0; i < NC; ++i) x[k][i] = part[(int64_t)min(s0 + k * WAVES, S - 1) * HD + 64 * i];
  };
  int s0 = WAVES == 1 ? 0 : w;
  ask(s0);
  const bool mine = row >= r0 && row < r1;
  if (!mine && !p.fresh) return;
  bf16_raw* y = (bf16_raw*)p.out + row * p.so_row + (int64_t)head * HD;
  float o[NC] = {}, L = 0.f;
  if (mine) {
    const bool live = lane < S && l_in != 0.f;  // a split without keys wrote no output
    const float ms = live ? m_in : NEG, ls = live ? l_in : 0.f;
    const float M = wave_max(ms), f = ms == NEG ? 0.f : __builtin_amdgcn_exp2f(ms - M);
    L = wave_sum(live ? f * ls : 0.f);
    const unsigned long long alive = __ballot(live);
    while (true) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int s = s0 + k * WAVES;
        const float fs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), min(s, 63)));
        if (s < S && (alive >> s & 1))
#pragma unroll
          for (int i = 0; i < NC; ++i) o[i] += fs * x[k][i];
      }
      s0 += 8 * WAVES;
      if (s0 >= S) break;
      ask(s0);
    }
  }
  if constexpr (WAVES > 1) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (HD >= 64 || lane < HD) s_o[w][lane + 64 * i] = o[i];
    __syncthreads();
    if (w > 0) return;
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (HD >= 64 || lane < HD) o[i] = (s_o[0][lane + 64 * i] + s_o[1][lane + 64 * i]) + (s_o[2][lane + 64 * i] + s_o[3][lane + 64 * i]);
  }
  const bool some = L > 0.f || L != L;
#pragma unroll
  for (int i = 0; i < NC; ++i)
    if (HD >= 64 || lane < HD) y[lane + 64 * i] = some ? f2bf(o[i] / L) : (bf16_raw)0;
}

// blocks of four waves for every (rows of a wave, head)
int64_t kv4_units(int rows, int kv, int hd) { return (((int64_t)rows + 512 / hd - 1) / (512 / hd) * kv + 3) / 4; }
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
  GROVE_CHECK(p && p->rows >= 0 && p->rows <= 1 << 30 && p->kv > 0 && p->kv <= 65535, GROVE_E_SHAPE, "kv4_append: bad shape");
  KV4_SHAPE(p, "kv4_append");
  if (p->rows == 0) return GROVE_OK;
  GROVE_CHECK(p->k && p->v && p->codes && p->scales && p->slots, GROVE_E_SHAPE, "kv4_append: null pointer");
  GROVE_CHECK(((uintptr_t)p->codes & 15) == 0 && ((uintptr_t)p->scales & 15) == 0, GROVE_E_ALIGN, "kv4_append: the cache must be 16-byte aligned");
  GROVE_CHECK(kv4_units(p->rows, p->kv, p->hd) <= 0x7fffffff, GROVE_E_SHAPE, "kv4_append: too many rows");
  const dim3 grid((unsigned)kv4_units(p->rows, p->kv, p->hd));
  const int vec = (((uintptr_t)p->k | (uintptr_t)p->v) & 15) == 0 && p->sk_row % 8 == 0 && p->sk_head % 8 == 0 && p->sv_row % 8 == 0 && p->sv_head % 8 == 0;
#define LAUNCH(HD) hipLaunchKernelGGL(kv4_append_kernel<HD>, grid, dim3(256), 0, (hipStream_t)stream, *p, vec)
  KV4_HD(p->hd, LAUNCH)
#undef LAUNCH
  GROVE_LAUNCH_CHECK();
  return GROVE_OK;
}

extern "C" int grove_kv4_read(const grove_kv4_read_params* p, void* stream) {
  GROVE_CHECK(p && p->rows >= 0 && p->rows <= 1 << 30 && p->kv > 0 && p->kv <= 65535, GROVE_E_SHAPE, "kv4_read: bad shape");
  KV4_SHAPE(p, "kv4_read");
  if (p->rows == 0) return GROVE_OK;
  GROVE_CHECK(p->k && p->v && p->codes && p->scales && p->slots, GROVE_E_SHAPE, "kv4_read: null pointer");
  GROVE_CHECK((((uintptr_t)p->codes | (uintptr_t)p->scales | (uintptr_t)p->k | (uintptr_t)p->v) & 15) == 0, GROVE_E_ALIGN,
              "kv4_read: the cache and the outputs must be 16-byte aligned");
  GROVE_CHECK(kv4_units(p->rows, p->kv, p->hd) <= 0x7fffffff, GROVE_E_SHAPE, "kv4_read: too many rows");
  const dim3 grid((unsigned)kv4_units(p->rows, p->kv, p->hd));
#define LAUNCH(HD)                                                                                              \
  if (p->f32) hipLaunchKernelGGL((kv4_read_kernel<HD, float>), grid, dim3(256), 0, (hipStream_t)stream, *p);    \
  else hipLaunchKernelGGL((kv4_read_kernel<HD, bf16_raw>), grid, dim3(256), 0, (hipStream_t)stream, *p)
  KV4_HD(p->hd, LAUNCH)
#undef LAUNCH
  GROVE_LAUNCH_CHECK();
  return GROVE_OK;
}

extern "C" int grove_kv4_attn(const grove_kv4_attn_params* p, void* stream) {
  GROVE_CHECK(p && p->requests >= 0 && p->requests <= 65535 && p->rows >= 0 && p->kv > 0 && p->heads > 0 && p->heads % p->kv == 0 && p->heads <= 65535 &&
              p->max_pages > 0 && p->ld_table >= 0 && p->max_q >= 0, GROVE_E_SHAPE, "kv4_attn: bad shape (heads must be a multiple of kv)");
  KV4_SHAPE(p, "kv4_attn");
  if (p->rows == 0 || p->requests == 0 || p->max_q == 0) return GROVE_OK;
  GROVE_CHECK(p->q && p->codes && p->scales && p->table && p->kv_len && p->cu_q && p->out, GROVE_E_SHAPE, "kv4_attn: null pointer");
  GROVE_CHECK(((uintptr_t)p->codes & 15) == 0 && ((uintptr_t)p->scales & 15) == 0, GROVE_E_ALIGN, "kv4_attn: the cache must be 16-byte aligned");
  GROVE_CHECK(p->n_split >= 1 && p->n_split <= 64 && (p->n_split == 1 || p->partial), GROVE_E_WORKSPACE, "kv4_attn: 1 to 64 splits, more than one with a workspace");
  GROVE_CHECK((int64_t)p->max_pages * p->page <= 1 << 30, GROVE_E_SHAPE, "kv4_attn: a row of the table holds more than 2^30 tokens");
  const int shift = __builtin_ctz((unsigned)p->page);
  GROVE_CHECK(((uintptr_t)p->q & 15) == 0 && p->sq_row % 8 == 0 && p->sq_head % 8 == 0 && ((uintptr_t)p->out & 3) == 0 && p->so_row % 2 == 0, GROVE_E_ALIGN,
              "kv4_attn: q must be aligned to 16 bytes and out to 4, their strides too");
  // columns that one pass over a key can serve: as few tiles of 16 as hold them, at most 64 (32 at hd 256, whose outputs fill the registers)
  const int64_t cols = (int64_t)(p->max_q < p->rows ? p->max_q : p->rows) * (p->heads / p->kv);
  const int ct = cols <= 16 ? 1 : cols <= 32 || p->hd == 256 ? 2 : 4;
  const int64_t chunks = (cols + 16 * ct - 1) / (16 * ct), units = (int64_t)p->rows * p->heads;
  GROVE_CHECK(units <= 1 << 30 && (p->n_split <= 8 || units < 1 << 24), GROVE_E_SHAPE, "kv4_attn: too many rows");
  GROVE_CHECK(chunks * p->kv <= 65535, GROVE_E_SHAPE, "kv4_attn: too many new tokens in a request (%lld columns)", (long long)cols);
  const dim3 grid((unsigned)p->n_split, (unsigned)(chunks * p->kv), (unsigned)p->requests);
#define RUN(HD, CT)                                                                                                                  \
  do {                                                                                                                               \
    constexpr int lds = kv4_lds(HD, CT);                                                                                             \
    if (lds > 64 * 1024) hipFuncSetAttribute((const void*)kv4_attn_kernel<HD, CT>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);                      \
    hipLaunchKernelGGL((kv4_attn_kernel<HD, CT>), grid, dim3(256), lds, (hipStream_t)stream, *p, shift);               \
  } while (0)
#define LAUNCH(HD)                       \
  if (ct == 1) RUN(HD, 1);               \
  else if (ct == 2) RUN(HD, 2);          \
  else RUN((HD < 256 ? HD : 128), 4)
  KV4_HD(p->hd, LAUNCH)
#undef LAUNCH
#undef RUN
  GROVE_LAUNCH_CHECK();
  if (p->n_split > 1) {
#define LAUNCH(HD)                                                                                                                                  \
  if (p->n_split > 8) hipLaunchKernelGGL((kv4_join_kernel<HD, 4>), dim3((unsigned)units), dim3(256), 0, (hipStream_t)stream, *p);                   \
  else hipLaunchKernelGGL((kv4_join_kernel<HD, 1>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, (hipStream_t)stream, *p)
    KV4_HD(p->hd, LAUNCH)
#undef LAUNCH
    GROVE_LAUNCH_CHECK();
  }
  return GROVE_OK;
}
