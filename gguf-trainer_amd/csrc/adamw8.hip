// AdamW whose moments are held in 8 bits: the step of AdamWGpu (src/backend/adamw-gpu.ts:131-251, src/train/adam.ts:46-82)
// over a whole group, with 2 bytes of state per parameter instead of 8.
//
//   g' = g * scale;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2;  w -= lr (m / bc1 / (sqrt(v / bc2) + eps) + wd w)
//
// What is held. m and r = sqrt(v), each as an OCP e4m3 value times 2^e with one e per block of 256 elements of a tensor:
// the smallest e with |value| <= 448 * 2^e over the block. A power of two, so that decoding is exact and a value that does
// not change keeps its code whatever its neighbours do. The root of v rather than v: e4m3 spans 2^17.8, which as a range of
// gradients is enough for a block and as a range of their squares would not be.
//
// How they are rounded. Up or down at random, in proportion to what is left over. A step moves m by a tenth and r by a
// two-thousandth (b2 = 0.999) of what separates it from its target, far less than half of e4m3's steps of 6 to 12 percent:
// rounded to nearest both would stay where they are. The random bits of an element are a function of the step's seed, the
// number of its block in the group and its place in the block, 16 for each moment, so a step repeats bit for bit. An r that
// is there is not rounded to zero: m / (0 + eps) would follow. r is unbiased, so v = r^2 is high by r's variance: where v still
// grows by small steps up to 6 percent, half of that in the update's denominator.
// The update itself uses m and v before they are rounded. Moments that are not finite are held as e4m3's NaN, and their neighbours'
// exponent goes by the finite ones. r has no use for the sign: its positive NaN stands for infinity, a square that left FP32, whose weight is
// left to its decay as with moments of 32 bits, its negative one for NaN.
//
// Bound by memory: 16 bytes per element (g read, w read and written, two codes each way), 20 with the clip, whose norm has
// to be known before the first update. One wavefront to a block, four neighbouring elements to a lane, so that the block's
// largest moments are one exchange within the wavefront and no LDS is used. 63 vector operations per element: at
// twice that (library roots and divisions, float comparisons for the block's largest) they were as long as the memory's time.
#include <algorithm>
#include <exception>
#include <iterator>
#include <utility>
#include "optim.h"

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

#define BLK8 256
#define CHUNK8 1024                              // four blocks, one to a wavefront
#define NORM8_PER_CU 8                           // workgroups of the norm's kernel
#define NORM8_GROUPS 2048
#define SLICE8_CHUNKS (1 << 22)                  // chunks to a launch: a grid's threads are counted in 32 bits
#define FOLD8_CHUNKS 2048                        // up to here the update's workgroups add up the norm's sums themselves
// The chunk table's pointers come out of memory, where the compiler cannot see that they are global: without this its loads
// take the flat path, which also waits for LDS.
#define GLOBAL __attribute__((address_space(1)))
typedef GLOBAL float gfloat;
typedef GLOBAL v4f gv4f;
typedef GLOBAL unsigned char gbyte;

struct Adam8H { float b1, b2, omb1, omb2, eps, wd, lr, ibc1, rbc2; unsigned key; };

// The random bits: a multiply-xorshift mixer (shifts 16, 15, 15 and two factors published with the hash-prospector search, public domain), two
// rounds of it for a block's key and one from there for each element.
__host__ __device__ __forceinline__ unsigned mix1(unsigned x) {
  x ^= x >> 16;
  x *= 0x21F0AAADu;
  return x ^ (x >> 15);
}
__host__ __device__ __forceinline__ unsigned mix2(unsigned x) {
  x = mix1(x) * 0x735A2D97u;
  return x ^ (x >> 15);
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// The bits of a positive float with its leading one at bit 23, and the exponent that goes with them (denormals too).
__device__ __forceinline__ void normal_bits(unsigned b, int &e, unsigned &frac) {
  const int sh = b >> 23 ? 0 : __builtin_clz(b | 1u) - 8;
  e = sh ? 1 - sh : (int)(b >> 23);
  frac = (b << sh) & 0x7fffffu;
}
// smallest e >= -126 with top <= 448 * 2^e, 448 = 1.75 * 2^8; whole numbers only, so that it runs on the scalar unit
__device__ __forceinline__ int exponent_m(unsigned top) {
  int e;
  unsigned frac;
  normal_bits(top, e, frac);
  return top ? max(e - 127 - (frac <= 0x600000u ? 8 : 7), -126) : -126;
}
// the same for sqrt(top), e >= LEAST_R: top <= 448^2 * 4^e, 448^2 = 1.53125 * 2^17. With it every r is a multiple of 2^-74 of at most four bits,
// and its square an FP32 number: none is lost where the step forms it or in FP32 moments, though it were the last of the denormals.
#define LEAST_R -65
__device__ __forceinline__ int exponent_r(unsigned top) {
  int e;
  unsigned frac;
  normal_bits(top, e, frac);
  return top ? max((e - 127 - (frac <= 0x440000u ? 17 : 16) + 1) >> 1, LEAST_R) : -126;
}

// Largest of one word over the wavefront, as a scalar: four exchanges within each row of 16 lanes, the four rows on the
// scalar unit.
template <int CTRL> __device__ __forceinline__ unsigned dpp_max(unsigned v) {
  const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
  return v > o ? v : o;
}
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
  v = dpp_max<0xB1>(v);                          // neighbours
  v = dpp_max<0x4E>(v);                          // pairs
  v = dpp_max<0x141>(v);                         // halves of a row
  v = dpp_max<0x140>(v);                         // rows mirrored
  const unsigned a = __builtin_amdgcn_readlane((int)v, 0), b = __builtin_amdgcn_readlane((int)v, 16), c = __builtin_amdgcn_readlane((int)v, 32),
                 d = __builtin_amdgcn_readlane((int)v, 48);
  return max(max(a, b), max(c, d));
}

#define FINITE_BITS 0x7f800000u                  // bits of a finite magnitude are below this

// sqrt(v) to the last bit or next to it: the hardware's 1 / sqrt, which takes no denormals, and one Newton step. Zero stays zero, infinity and
// NaN give NaN.
__device__ __forceinline__ float root(float v) {
  const float y = __builtin_amdgcn_rsqf(__builtin_amdgcn_fmed3f(v, 1.17549435e-38f, __builtin_inff()));
  const float s = v * y;
  return __builtin_fmaf(__builtin_fmaf(-s, s, v), 0.5f * y, s);
}
// Of four. Denormals (a block that has had no gradient for a thousand steps) and infinity are rare, so they are looked for together: the former
// are taken as 2^64 v, the latter stays itself.
__device__ __forceinline__ void roots(const float (&v)[4], float (&r)[4]) {
  unsigned least = ~0u, most = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    r[j] = root(v[j]);
    least = min(least, __float_as_uint(v[j]) - 1u);            // zero is the largest here
    most = max(most, __float_as_uint(v[j]));
  }
  if (least < 0x7fffffu || most >= FINITE_BITS) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (v[j] < 1.17549435e-38f) r[j] = root(v[j] * 1.84467441e19f) * 2.32830644e-10f;
      if (__float_as_uint(v[j]) == FINITE_BITS) r[j] = v[j];
    }
  }
}

// Four codes, one to a byte, from the magnitudes of four values scaled so that e4m3's exponent is theirs: y = |value| * 2^(-e - 120). A y
// below 2^-126 is then a denormal exactly where e4m3's are, so one addition rounds both: the code is the y's bits from 20
// up, after 16 random bits are added to the 20 below them. `low` is the least y of each (its bits), NaN and infinity
// become the code 0x7f. The codes come back in the top seven bits but one of each word, for the caller to set the sign and gather.
__device__ __forceinline__ unsigned code_word(float y, unsigned low, unsigned bits, unsigned place) {
  const unsigned r = __builtin_amdgcn_perm(0u, bits, place);                 // the 16 random bits at 8..23
  const unsigned b = min(max(__float_as_uint(y), low), 0x07f00000u);
  return (b << 4) + r;
}
__device__ __forceinline__ unsigned gather(const unsigned (&t)[4]) {
  const unsigned lo = __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0703u), hi = __builtin_amdgcn_perm(t[3], t[2], 0x07030c0cu);
  return lo | hi;
}

__device__ __forceinline__ unsigned without_256(unsigned c) {
#pragma unroll
  for (int j = 0; j < 4; j++) if ((c >> (8 * j) & 0x7fu) == 0x78u) c -= 1u << (8 * j);
  return c;
}

#define INF_R 0x7fu                              // codes of an r that is infinite
#define NAN_R 0xffu                              // and of one that is no number

// Codes and exponents of a block's moments from their values and roots, four elements to a lane (elements past the tensor's
// end as zeros). bits: 16 random bits for m below 16 for r.
__device__ __forceinline__ void encode_block(const float (&m)[4], const float (&v)[4], const float (&r)[4], const unsigned (&bits)[4], unsigned &mc,
                                             unsigned &rc, int &em, int &er) {
  // magnitudes order as their bits do
  unsigned am[4], av[4];
#pragma unroll
  for (int j = 0; j < 4; j++) { am[j] = __float_as_uint(m[j]) & 0x7fffffffu; av[j] = __float_as_uint(v[j]); }
  unsigned tm = wave_umax(max(max(am[0], am[1]), max(am[2], am[3])));
  unsigned tv = wave_umax(max(max(av[0], av[1]), max(av[2], av[3])));
  const bool odd = max(tm, tv) >= FINITE_BITS;
  if (odd) {                                     // an infinity, a NaN, a second moment below zero: the exponents go by the others
    tm = tv = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (am[j] < FINITE_BITS) tm = max(tm, am[j]);
      if (av[j] < FINITE_BITS) tv = max(tv, av[j]);
    }
    tm = wave_umax(tm);
    tv = wave_umax(tv);
  }
  em = exponent_m(tm);
  er = exponent_r(tv);
  unsigned cm[4], cr[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const unsigned c = code_word(__builtin_ldexpf(__builtin_fabsf(m[j]), -120 - em), 0u, bits[j], 0x0c01000cu);
    cm[j] = (c & 0x7fffffffu) | (__float_as_uint(m[j]) & 0x80000000u);
    cr[j] = code_word(__builtin_ldexpf(r[j], -120 - er), v[j] > 0.f ? 1u << 20 : 0u, bits[j], 0x0c03020cu);
  }
  mc = gather(cm);
  rc = gather(cr);
  if (odd) {
#pragma unroll
    for (int j = 0; j < 4; j++) if (!(v[j] >= 0.f)) rc |= NAN_R << (8 * j);
  }
  // next to FP32's largest, 256 * 2^120 is past it as an m, and the square of 256 * 2^56 as an r: 240 of them are the most that is held
  if (em >= 120) mc = without_256(mc);
  if (er >= 56) rc = without_256(rc);
}
__device__ __forceinline__ void decode4(unsigned c, float s, float (&out)[4]) {
  const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  out[0] = lo[0] * s; out[1] = lo[1] * s; out[2] = hi[0] * s; out[3] = hi[1] * s;
}
__device__ __forceinline__ void decode_roots4(unsigned c, float s, float (&out)[4]) {
  decode4(c, s, out);
  if (((c & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) {       // a NaN among them
#pragma unroll
    for (int j = 0; j < 4; j++) if ((c >> (8 * j) & 0xffu) == INF_R) out[j] = __builtin_inff();
  }
}
// four neighbouring bytes of a block of n elements; zeros past its end
__device__ __forceinline__ unsigned load_codes(const gbyte *p, int i0, int n, bool whole) {
  if (whole) return __builtin_nontemporal_load((const GLOBAL unsigned *)(p + i0));
  unsigned c = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) if (i0 + j < n) c |= (unsigned)p[i0 + j] << (8 * j);
  return c;
}
__device__ __forceinline__ void store_codes(gbyte *p, int i0, int n, bool whole, unsigned c) {
  if (whole) { __builtin_nontemporal_store(c, (GLOBAL unsigned *)(p + i0)); return; }
#pragma unroll
  for (int j = 0; j < 4; j++) if (i0 + j < n) p[i0 + j] = (unsigned char)(c >> (8 * j));
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
  return v;
}
__device__ __forceinline__ double block_sum64(double v, double *sm) {
  v = wave_sum64(v);
  __syncthreads();
  if (threadIdx.x % WAVE == 0) sm[threadIdx.x / WAVE] = v;
  __syncthreads();
  return (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

// The clip scale and the norm from the partial sums, in every thread of a workgroup.
__device__ __forceinline__ float clip_scale(const double *__restrict__ sums, int nsums, double clip, double *sm, double &norm) {
  double t = 0;
  for (int i = threadIdx.x; i < nsums; i += 256) t += sums[i];
  norm = sqrt(block_sum64(t, sm));
  return norm > clip ? (float)(clip / (norm + 1e-12)) : 1.0f;
}

// A workgroup takes one chunk, a wavefront one block, and nothing is repeated: 1642 us for 642M parameters (6.26 TB/s, a large copy
// reaches 4.8 to 5.0 there), against 1770 with two blocks to a wavefront, 1848 with four and 2060 with as many workgroups as
// the card holds going through all chunks. Every array is touched once a step, so all accesses are streaming ones: 1956
// without (four blocks). nsums > 0: the clip scale is formed here from the partial sums instead of by adamw8_scale_k.
__global__ __launch_bounds__(256) void adamw8_update_k(const Chunk8 *__restrict__ chunks, const double *__restrict__ sums, int nsums, double clip,
                                                       float *__restrict__ scale, Adam8H h) {
#pragma clang fp contract(off)                   // m and v: every product is rounded before it is added, so that they are defined to the bit
  __shared__ double sm[4];
  float sc;
  if (nsums) {
    double norm;
    sc = clip_scale(sums, nsums, clip, sm, norm);
    if (blockIdx.x == 0 && threadIdx.x == 0) { scale[0] = sc; scale[1] = (float)norm; }
  } else {
    sc = scale[0];
  }
  const Chunk8 c = chunks[blockIdx.x];
  const int lane = threadIdx.x % WAVE, i0 = lane * 4, b = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int n = min(BLK8, c.len - b * BLK8);
  if (n <= 0) return;
  const bool whole = n == BLK8 && ((reinterpret_cast<uintptr_t>(c.w) | reinterpret_cast<uintptr_t>(c.g)) % 16 |
                                   (reinterpret_cast<uintptr_t>(c.m) | reinterpret_cast<uintptr_t>(c.r)) % 4) == 0;
  gfloat *w = (gfloat *)c.w + b * BLK8;
  const gfloat *g = (const gfloat *)c.g + b * BLK8;
  gbyte *mp = (gbyte *)c.m + b * BLK8, *rp = (gbyte *)c.r + b * BLK8;
  GLOBAL signed char *e = (GLOBAL signed char *)c.e + 2 * b;
  float gg[4] = {0, 0, 0, 0}, ww[4] = {0, 0, 0, 0}, m[4], v[4], r[4];
  if (whole) {
    const v4f a = __builtin_nontemporal_load((const gv4f *)g + lane), d = __builtin_nontemporal_load((const gv4f *)w + lane);
#pragma unroll
    for (int j = 0; j < 4; j++) { gg[j] = a[j]; ww[j] = d[j]; }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) if (i0 + j < n) { gg[j] = g[i0 + j]; ww[j] = w[i0 + j]; }
  }
  decode4(load_codes(mp, i0, n, whole), pow2(e[0]), m);
  decode_roots4(load_codes(rp, i0, n, whole), pow2(e[1]), v);
  const unsigned key = mix2((c.block + b) ^ h.key) + (unsigned)i0 * 0x9E3779B9u;
  unsigned bits[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float x = gg[j] * sc;
    m[j] = m[j] * h.b1 + x * h.omb1;
    v[j] = (v[j] * v[j]) * h.b2 + (x * h.omb2) * x;
  }
  roots(v, r);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    // 1 / x to the last bit but one: the update is a small part of the weight
    float upd = (m[j] * h.ibc1) * __builtin_amdgcn_rcpf(__builtin_fmaf(r[j], h.rbc2, h.eps));
    if (h.wd > 0.f) upd = __builtin_fmaf(h.wd, ww[j], upd);
    ww[j] = __builtin_fmaf(-h.lr, upd, ww[j]);
    bits[j] = mix1(key + (unsigned)j * 0x9E3779B9u);
  }
  unsigned mc, rc;
  int em, er;
  encode_block(m, v, r, bits, mc, rc, em, er);
  if (whole) __builtin_nontemporal_store(v4f{ww[0], ww[1], ww[2], ww[3]}, (gv4f *)w + lane);
  else
#pragma unroll
    for (int j = 0; j < 4; j++) if (i0 + j < n) w[i0 + j] = ww[j];
  store_codes(mp, i0, n, whole, mc);
  store_codes(rp, i0, n, whole, rc);
  if (lane == 0) *(GLOBAL unsigned short *)e = (unsigned short)((unsigned)(em & 0xff) | (unsigned)(er & 0xff) << 8);
}

// Sum of squares of every gradient in 64 bits: each workgroup its chunks in order, its sum to sums[workgroup]. 135M gradients in 84 us
// (6.4 TB/s) with eight workgroups to a CU, 120 with four, 187 with two.
__global__ __launch_bounds__(256) void adamw8_norm_k(const Chunk8 *__restrict__ chunks, int nchunks, double *__restrict__ sums) {
  __shared__ double sm[4];
  double s[4] = {0, 0, 0, 0};
  // four chunks at a time, so that each thread has four loads in flight
  for (int k = blockIdx.x * 4; k < nchunks; k += gridDim.x * 4) {
    bool all = k + 4 <= nchunks;
    for (int u = 0; u < 4 && all; u++) all = chunks[k + u].len == CHUNK8 && (uintptr_t)chunks[k + u].g % 16 == 0;
    if (all) {
      v4f x[4];
#pragma unroll
      for (int u = 0; u < 4; u++) x[u] = __builtin_nontemporal_load((const gv4f *)chunks[k + u].g + threadIdx.x);
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[j] = fma((double)x[u][j], (double)x[u][j], s[j]);
      continue;
    }
    for (int u = k; u < min(k + 4, nchunks); u++) {
      const gfloat *g = (const gfloat *)chunks[u].g;
      const int len = chunks[u].len;
      for (int i = threadIdx.x; i < len; i += 256) s[0] = fma((double)g[i], (double)g[i], s[0]);
    }
  }
  const double t = block_sum64((s[0] + s[1]) + (s[2] + s[3]), sm);
  if (threadIdx.x == 0) sums[blockIdx.x] = t;
}

__global__ __launch_bounds__(256) void adamw8_scale_k(const double *__restrict__ sums, int nsums, double clip, float *__restrict__ scale) {
  __shared__ double sm[4];
  double norm;
  const float sc = clip_scale(sums, nsums, clip, sm, norm);
  if (threadIdx.x == 0) { scale[0] = sc; scale[1] = (float)norm; }
}

// The moments of one tensor as FP32 values, and states from such values, rounded to the nearest (ties away from zero).
__global__ __launch_bounds__(256) void state8_read_k(int64_t size, const unsigned char *mp, const unsigned char *rp, const signed char *e, float *m,
                                                     float *v) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256) {
    const int64_t b = i / BLK8;
    if (m) m[i] = __builtin_amdgcn_cvt_f32_fp8((int)mp[i], 0) * pow2(e[2 * b]);
    if (v) {
      const float r = __builtin_amdgcn_cvt_f32_fp8((int)rp[i], 0) * pow2(e[2 * b + 1]);
      v[i] = rp[i] == INF_R ? __builtin_inff() : r * r;
    }
  }
}
__global__ __launch_bounds__(256) void state8_write_k(int64_t size, unsigned char *mp, unsigned char *rp, signed char *e, const float *m, const float *v) {
  const int lane = threadIdx.x % WAVE, i0 = lane * 4;
  const int64_t nb = (size + BLK8 - 1) / BLK8;
  for (int64_t b = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE; b < nb; b += (int64_t)gridDim.x * 4) {
    const int n = (int)min((int64_t)BLK8, size - b * BLK8);
    float mm[4] = {0, 0, 0, 0}, vv[4] = {0, 0, 0, 0}, rr[4];
    const unsigned half[4] = {0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
#pragma unroll
    for (int j = 0; j < 4; j++) if (i0 + j < n) { mm[j] = m[b * BLK8 + i0 + j]; vv[j] = v[b * BLK8 + i0 + j] + 0.f; }      // -0 becomes 0
    roots(vv, rr);
    unsigned mc, rc;
    int em, er;
    encode_block(mm, vv, rr, half, mc, rc, em, er);
    store_codes((gbyte *)mp + b * BLK8, i0, n, false, mc);
    store_codes((gbyte *)rp + b * BLK8, i0, n, false, rc);
    if (lane == 0) { e[2 * b] = (signed char)em; e[2 * b + 1] = (signed char)er; }
  }
}

extern "C" {

int gt_adamw8_create(gt_ctx *ctx, int n, const gt_buf *w, const gt_buf *g, const gt_buf *m, const gt_buf *r, const gt_buf *e, const int64_t *sizes,
                     double beta1, double beta2, double eps, double weight_decay, double clip, gt_adamw **out) {
  GT_ENTER(ctx);
  GT_REQUIRE(ctx, n >= 0 && out && (n == 0 || (w && g && m && r && e && sizes)), "gt_adamw8_create: bad arguments");
  int64_t blocks = 0, chunks = 0;
  for (int i = 0; i < n; i++) {
    GT_REQUIRE(ctx, w[i] && g[i] && m[i] && r[i] && e[i] && sizes[i] >= 0 && sizes[i] <= (int64_t)1 << 40,
               "gt_adamw8_create: tensor %d has a null buffer or a size that is negative or more than 2^40", i);
    GT_REQUIRE(ctx, (w[i] | g[i]) % 4 == 0 && e[i] % 2 == 0, "gt_adamw8_create: tensor %d: a buffer is not aligned to its elements", i);
    blocks += cdiv(sizes[i], BLK8);
    chunks += cdiv(sizes[i], CHUNK8);
  }
  GT_REQUIRE(ctx, blocks <= 0xffffffffll && chunks <= 0x7fffffffll, "gt_adamw8_create: %lld blocks are more than a group can number", (long long)blocks);
  // two tensors that share what a step writes would be stepped by two workgroups at once
  std::vector<std::pair<uint64_t, uint64_t>> spans;
  std::vector<Chunk8> ch;
  gt_adamw *o = nullptr;
  try {
    spans.reserve((size_t)n * 4);
    ch.reserve((size_t)chunks);
    o = new gt_adamw();
    o->tensors8.reserve((size_t)n);
  } catch (const std::exception &) {
    delete o;
    GT_FAIL(ctx, "gt_adamw8_create: no host memory for a table of %lld chunks", (long long)chunks);
  }
  for (int i = 0; i < n; i++)
    if (sizes[i]) {
      const uint64_t s = (uint64_t)sizes[i];
      for (auto p : {std::make_pair(w[i], s * 4), std::make_pair(m[i], s), std::make_pair(r[i], s), std::make_pair(e[i], (uint64_t)cdiv(sizes[i], BLK8) * 2)})
        spans.push_back({p.first, p.first + p.second});
    }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); i++)
    if (spans[i].first < spans[i - 1].second) {
      delete o;
      GT_FAIL(ctx, "gt_adamw8_create: two of the buffers that a step writes overlap (a tensor listed twice?)");
    }
  // and a gradient in what a step writes would be read by some workgroups before and by others after
  for (int i = 0; i < n; i++)
    if (sizes[i]) {
      const auto at = std::upper_bound(spans.begin(), spans.end(), std::make_pair(g[i], UINT64_MAX));
      if ((at != spans.begin() && std::prev(at)->second > g[i]) || (at != spans.end() && at->first < g[i] + (uint64_t)sizes[i] * 4)) {
        delete o;
        GT_FAIL(ctx, "gt_adamw8_create: the gradient of tensor %d and a buffer that a step writes overlap", i);
      }
    }
  o->bits8 = true;
  o->n = n; o->beta1 = beta1; o->beta2 = beta2; o->eps = eps; o->wd = weight_decay; o->clip = clip;
  unsigned block = 0;
  for (int i = 0; i < n; i++) {
    o->tensors8.push_back({P<unsigned char>(m[i]), P<unsigned char>(r[i]), P<signed char>(e[i]), sizes[i]});
    o->total_elems += (double)sizes[i];
    for (int64_t off = 0; off < sizes[i]; off += CHUNK8) {
      const int len = (int)std::min<int64_t>(CHUNK8, sizes[i] - off);
      ch.push_back({P<float>(w[i]) + off, P<const float>(g[i]) + off, P<unsigned char>(m[i]) + off, P<unsigned char>(r[i]) + off,
                    P<signed char>(e[i]) + off / BLK8 * 2, len, block});
      block += (unsigned)cdiv(len, BLK8);
    }
  }
  o->nchunks = (int)ch.size();
  // one allocation: scale and norm, the norm's partial sums, the chunk table
  const size_t head = 256 + NORM8_GROUPS * sizeof(double), bytes = head + ch.size() * sizeof(Chunk8);
  const float one[2] = {1.0f, 0.0f};
  hipError_t err = hipMalloc(&o->block8, bytes);
  if (err == hipSuccess) {
    char *at = static_cast<char *>(o->block8);
    o->scale = reinterpret_cast<float *>(at);
    o->sums8 = reinterpret_cast<double *>(at + 256);
    o->chunks8 = reinterpret_cast<Chunk8 *>(at + head);
    err = hipMemcpy(o->scale, one, sizeof one, hipMemcpyHostToDevice);
    if (err == hipSuccess && !ch.empty()) err = hipMemcpy(o->chunks8, ch.data(), ch.size() * sizeof(Chunk8), hipMemcpyHostToDevice);
  }
  if (err != hipSuccess) {
    (void)hipGetLastError();
    adamw_release(o);
    GT_FAIL(ctx, "gt_adamw8_create: setting up the chunk table failed: %s", hipGetErrorString(err));
  }
  ctx->adamws.insert(o);
  *out = o;
  return 0;
}

int gt_adamw8_step(gt_ctx *ctx, gt_adamw *o, double lr, double bc1, double bc2, uint64_t seed) {
  GT_ENTER(ctx);
  GT_REQUIRE(ctx, o && ctx->adamws.count(o), "gt_adamw8_step: not an optimizer of this context");
  GT_REQUIRE(ctx, o->bits8, "gt_adamw8_step: this group's states are held in 32 bits: use gt_adamw_step");
  GT_REQUIRE(ctx, bc1 > 0 && bc2 > 0, "gt_adamw8_step: bias corrections must be positive");
  if (o->nchunks == 0) return 0;
  ProfScope ps(ctx, "adamw8", o->total_elems * (o->clip > 0 ? 20.0 : 16.0));
  const int nsums = o->clip > 0 ? (int)std::min<int64_t>({cdiv(o->nchunks, 4), (int64_t)ctx->num_cu * NORM8_PER_CU, NORM8_GROUPS}) : 0;
  // While the update's workgroups fit the card at once each adds up the few KB of sums itself, which saves a launch: 61 chunks take
  // 11.9 us a step this way and 14.5 the other, 4770 chunks 26 both ways, 131000 chunks 685 against 467.
  const bool fold = o->nchunks <= FOLD8_CHUNKS;
  if (nsums) {
    hipLaunchKernelGGL(adamw8_norm_k, dim3((unsigned)nsums), dim3(256), 0, ctx->stream, o->chunks8, o->nchunks, o->sums8);
    GT_LAUNCHED(ctx);
  }
  // every constant is formed in f64 and rounded to f32 once
  Adam8H h{(float)o->beta1, (float)o->beta2, (float)(1.0 - o->beta1), (float)(1.0 - o->beta2), (float)o->eps, (float)o->wd,
           (float)lr, (float)(1.0 / bc1), (float)(1.0 / sqrt(bc2)), mix2((unsigned)seed ^ mix2((unsigned)(seed >> 32) + 0x9E3779B9u))};
  if (nsums && !fold) {
    hipLaunchKernelGGL(adamw8_scale_k, dim3(1), dim3(256), 0, ctx->stream, o->sums8, nsums, o->clip, o->scale);
    GT_LAUNCHED(ctx);
  }
  for (int k = 0; k < o->nchunks; k += SLICE8_CHUNKS) {
    const unsigned nb = (unsigned)std::min(SLICE8_CHUNKS, o->nchunks - k);
    hipLaunchKernelGGL(adamw8_update_k, dim3(nb), dim3(256), 0, ctx->stream, o->chunks8 + k, o->sums8, fold ? nsums : 0, o->clip, o->scale, h);
    GT_LAUNCHED(ctx);
  }
  return 0;
}

static int state8_of(gt_ctx *ctx, const char *who, gt_adamw *o, int i, const Tensor8 **t) {
  GT_REQUIRE(ctx, o && ctx->adamws.count(o), "%s: not an optimizer of this context", who);
  GT_REQUIRE(ctx, o->bits8, "%s: this group's states are held in 32 bits", who);
  GT_REQUIRE(ctx, i >= 0 && i < o->n, "%s: tensor %d of %d", who, i, o->n);
  *t = &o->tensors8[i];
  return 0;
}

static bool meet(gt_buf a, uint64_t na, const void *b, uint64_t nb) {
  const uint64_t at = reinterpret_cast<uint64_t>(b);
  return a && at && a < at + nb && at < a + na;
}
static bool meets_state(gt_buf a, const Tensor8 *t) {
  const uint64_t n = (uint64_t)t->size, na = n * 4;
  return meet(a, na, t->m, n) || meet(a, na, t->r, n) || meet(a, na, t->e, (uint64_t)cdiv(t->size, BLK8) * 2);
}

int gt_adamw8_read(gt_ctx *ctx, gt_adamw *o, int i, gt_buf m, gt_buf v) {
  GT_ENTER(ctx);
  const Tensor8 *t;
  if (state8_of(ctx, "gt_adamw8_read", o, i, &t)) return 1;
  GT_REQUIRE(ctx, (m | v) % 4 == 0, "gt_adamw8_read: a buffer is not aligned to its elements");
  if (t->size == 0 || (!m && !v)) return 0;
  GT_REQUIRE(ctx, !meets_state(m, t) && !meets_state(v, t) && !meet(m, (uint64_t)t->size * 4, P<void>(v), (uint64_t)t->size * 4),
             "gt_adamw8_read: the buffers overlap, each other or the tensor's states");
  const unsigned nb = (unsigned)std::min<int64_t>(cdiv(t->size, 256), (int64_t)ctx->num_cu * 16);
  hipLaunchKernelGGL(state8_read_k, dim3(nb), dim3(256), 0, ctx->stream, t->size, t->m, t->r, t->e, P<float>(m), P<float>(v));
  GT_LAUNCHED(ctx);
  return 0;
}

int gt_adamw8_write(gt_ctx *ctx, gt_adamw *o, int i, gt_buf m, gt_buf v) {
  GT_ENTER(ctx);
  const Tensor8 *t;
  if (state8_of(ctx, "gt_adamw8_write", o, i, &t)) return 1;
  GT_REQUIRE(ctx, m && v && (m | v) % 4 == 0, "gt_adamw8_write: a buffer is missing or not aligned to its elements");
  if (t->size == 0) return 0;
  GT_REQUIRE(ctx, !meets_state(m, t) && !meets_state(v, t), "gt_adamw8_write: a buffer and the tensor's states overlap");
  const unsigned nb = (unsigned)std::min<int64_t>(cdiv(t->size, 4 * BLK8), (int64_t)ctx->num_cu * 16);
  hipLaunchKernelGGL(state8_write_k, dim3(nb), dim3(256), 0, ctx->stream, t->size, t->m, t->r, t->e, P<const float>(m), P<const float>(v));
  GT_LAUNCHED(ctx);
  return 0;
}
}
