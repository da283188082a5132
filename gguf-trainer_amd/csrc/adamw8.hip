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
// is there is never rounded to zero: m / (0 + eps) would follow.
// The update itself uses m and v before they are rounded. A moment that is not finite is held as e4m3's NaN and its
// neighbours' exponent goes by the finite ones.
//
// Bound by memory: 16 bytes per element (g read, w read and written, two codes each way), 20 with the clip, whose norm has
// to be known before the first update. One wavefront to a block, four neighbouring elements to a lane, so that the block's
// largest moments are one exchange within the wavefront and no LDS is used.
#include <algorithm>
#include "optim.h"

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

#define BLK8 256
#define CHUNK8 4096                              // 16 blocks, four to a wavefront
#define SSQ8_MAX_GROUPS 4096

struct Adam8H { float b1, b2, omb1, omb2, eps, wd, lr, ibc1, ibc2; unsigned key; };

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
// smallest e >= -126 with top <= 448 * 2^e (448 = 0.875 * 2^9)
__device__ __forceinline__ int exponent_for(float top) {
  if (!(top > 0.f)) return -126;
  return max(__builtin_amdgcn_frexp_expf(top) - (__builtin_amdgcn_frexp_mantf(top) <= 0.875f ? 9 : 8), -126);
}
// code of y in [0, 448] (not finite: the NaN code): the lower e4m3 neighbour, or the upper one where the remainder plus
// r16 / 65536 of a step makes a step
__device__ __forceinline__ unsigned encode8(float y, unsigned r16) {
  const unsigned normal = min(((__float_as_uint(y) + (r16 << 4)) >> 20) - (120u << 3), 0x7fu);
  const unsigned small = (unsigned)(y * 512.f + (float)r16 * (1.f / 65536.f));
  return y < 0.015625f ? small : normal;
}
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.40282347e38f; }

// Codes and exponents of a block's moments from their values, four elements to a lane (elements past the tensor's end as
// zeros). bits: 16 random bits for m below 16 for r.
__device__ __forceinline__ void encode_block(const float (&m)[4], const float (&v)[4], const unsigned (&bits)[4], unsigned &mc, unsigned &rc,
                                             int &em, int &er) {
  float tm = 0.f, tv = 0.f;
#pragma unroll
  for (int j = 0; j < 4; j++) { tm = fmaxf(tm, fabsf(m[j])); tv = fmaxf(tv, v[j]); }      // NaN drops out
  tm = wave_max(tm);
  tv = wave_max(tv);
  if (!is_finite(tm) || !is_finite(tv)) {
    tm = tv = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (is_finite(m[j])) tm = fmaxf(tm, fabsf(m[j]));
      if (is_finite(v[j])) tv = fmaxf(tv, v[j]);
    }
    tm = wave_max(tm);
    tv = wave_max(tv);
  }
  em = exponent_for(tm);
  er = exponent_for(sqrtf(tv));
  const float sm = pow2(-em), sr = pow2(-er);
  mc = rc = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const unsigned cm = encode8(fabsf(m[j]) * sm, bits[j] & 0xffffu) | (__float_as_uint(m[j]) >> 31 << 7);
    const unsigned cr = max(encode8(sqrtf(v[j]) * sr, bits[j] >> 16), v[j] > 0.f ? 1u : 0u);
    mc |= cm << (8 * j);
    rc |= cr << (8 * j);
  }
}
__device__ __forceinline__ void decode4(unsigned c, float s, float (&out)[4]) {
  const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  out[0] = lo[0] * s; out[1] = lo[1] * s; out[2] = hi[0] * s; out[3] = hi[1] * s;
}
// four neighbouring bytes of a block of n elements; zeros past its end
__device__ __forceinline__ unsigned load_codes(const unsigned char *p, int i0, int n, bool whole) {
  if (whole) return *reinterpret_cast<const unsigned *>(p + i0);
  unsigned c = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) if (i0 + j < n) c |= (unsigned)p[i0 + j] << (8 * j);
  return c;
}
__device__ __forceinline__ void store_codes(unsigned char *p, int i0, int n, bool whole, unsigned c) {
  if (whole) { *reinterpret_cast<unsigned *>(p + i0) = c; return; }
#pragma unroll
  for (int j = 0; j < 4; j++) if (i0 + j < n) p[i0 + j] = (unsigned char)(c >> (8 * j));
}

__global__ __launch_bounds__(256) void adamw8_update_k(const Chunk8 *__restrict__ chunks, const float *__restrict__ scale, Adam8H h) {
#pragma clang fp contract(off)                   // every product is rounded before it is added: the moments are defined to the bit
  const Chunk8 c = chunks[blockIdx.x];
  const float sc = scale[0];
  const int lane = threadIdx.x % WAVE, i0 = lane * 4;
  const bool aligned = ((reinterpret_cast<uintptr_t>(c.w) | reinterpret_cast<uintptr_t>(c.g)) % 16 |
                        (reinterpret_cast<uintptr_t>(c.m) | reinterpret_cast<uintptr_t>(c.r)) % 4) == 0;
  for (int b = threadIdx.x / WAVE; b * BLK8 < c.len; b += 4) {
    const int n = min(BLK8, c.len - b * BLK8);
    const bool whole = aligned && n == BLK8;
    float *w = c.w + b * BLK8;
    const float *g = c.g + b * BLK8;
    unsigned char *mp = c.m + b * BLK8, *rp = c.r + b * BLK8;
    float gg[4] = {0, 0, 0, 0}, ww[4] = {0, 0, 0, 0}, m[4], v[4];
    if (whole) {
      const v4f a = reinterpret_cast<const v4f *>(g)[lane], d = reinterpret_cast<const v4f *>(w)[lane];
#pragma unroll
      for (int j = 0; j < 4; j++) { gg[j] = a[j]; ww[j] = d[j]; }
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) if (i0 + j < n) { gg[j] = g[i0 + j]; ww[j] = w[i0 + j]; }
    }
    decode4(load_codes(mp, i0, n, whole), pow2(c.e[2 * b]), m);
    decode4(load_codes(rp, i0, n, whole), pow2(c.e[2 * b + 1]), v);
    const unsigned key = mix2((c.block + b) ^ h.key);
    unsigned bits[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float x = gg[j] * sc;
      m[j] = m[j] * h.b1 + x * h.omb1;
      v[j] = (v[j] * v[j]) * h.b2 + (x * h.omb2) * x;
      float upd = (m[j] * h.ibc1) / (sqrtf(v[j] * h.ibc2) + h.eps);
      if (h.wd > 0.f) upd += h.wd * ww[j];
      ww[j] -= h.lr * upd;
      bits[j] = mix1(key + (unsigned)(i0 + j) * 0x9E3779B9u);
    }
    unsigned mc, rc;
    int em, er;
    encode_block(m, v, bits, mc, rc, em, er);
    if (whole) reinterpret_cast<v4f *>(w)[lane] = v4f{ww[0], ww[1], ww[2], ww[3]};
    else
#pragma unroll
      for (int j = 0; j < 4; j++) if (i0 + j < n) w[i0 + j] = ww[j];
    store_codes(mp, i0, n, whole, mc);
    store_codes(rp, i0, n, whole, rc);
    if (lane == 0) *reinterpret_cast<unsigned short *>(c.e + 2 * b) = (unsigned short)((unsigned)(em & 0xff) | (unsigned)(er & 0xff) << 8);
  }
}

// Sum of squares of every gradient in 64 bits: each workgroup its chunks, its sum to sums[workgroup]; the workgroup that
// comes last adds the sums in workgroup order and turns the norm into the clip scale. sums[SSQ8_MAX_GROUPS] counts.
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
__global__ __launch_bounds__(256) void adamw8_norm_k(const Chunk8 *__restrict__ chunks, int nchunks, double *sums, double clip, float *scale) {
  __shared__ double sm[4];
  __shared__ int last;
  double s = 0;
  for (int k = blockIdx.x; k < nchunks; k += gridDim.x) {
    const float *g = chunks[k].g;
    const int len = chunks[k].len;
    const int n4 = reinterpret_cast<uintptr_t>(g) % 16 == 0 ? len / 4 : 0;
    for (int i = threadIdx.x; i < n4; i += 256) {
      const v4f x = reinterpret_cast<const v4f *>(g)[i];
#pragma unroll
      for (int j = 0; j < 4; j++) s = fma((double)x[j], (double)x[j], s);
    }
    for (int i = n4 * 4 + threadIdx.x; i < len; i += 256) s = fma((double)g[i], (double)g[i], s);
  }
  s = block_sum64(s, sm);
  unsigned *count = reinterpret_cast<unsigned *>(sums + SSQ8_MAX_GROUPS);
  if (threadIdx.x == 0) {
    __hip_atomic_store(sums + blockIdx.x, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  double t = 0;
  for (unsigned i = threadIdx.x; i < gridDim.x; i += 256) t += __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  t = block_sum64(t, sm);
  if (threadIdx.x == 0) {
    const double norm = sqrt(t);
    scale[0] = norm > clip ? (float)(clip / (norm + 1e-12)) : 1.0f;
    scale[1] = (float)norm;
    __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// The moments of one tensor as FP32 values, and states from such values, rounded to the nearest (ties away from zero).
__global__ __launch_bounds__(256) void state8_read_k(int64_t size, const unsigned char *mp, const unsigned char *rp, const signed char *e, float *m,
                                                     float *v) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256) {
    const int64_t b = i / BLK8;
    if (m) m[i] = __builtin_amdgcn_cvt_f32_fp8((int)mp[i], 0) * pow2(e[2 * b]);
    if (v) {
      const float r = __builtin_amdgcn_cvt_f32_fp8((int)rp[i], 0) * pow2(e[2 * b + 1]);
      v[i] = r * r;
    }
  }
}
__global__ __launch_bounds__(256) void state8_write_k(int64_t size, unsigned char *mp, unsigned char *rp, signed char *e, const float *m, const float *v) {
  const int lane = threadIdx.x % WAVE, i0 = lane * 4;
  const int64_t nb = (size + BLK8 - 1) / BLK8;
  for (int64_t b = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE; b < nb; b += (int64_t)gridDim.x * 4) {
    const int n = (int)min((int64_t)BLK8, size - b * BLK8);
    float mm[4] = {0, 0, 0, 0}, vv[4] = {0, 0, 0, 0};
    const unsigned half[4] = {0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
#pragma unroll
    for (int j = 0; j < 4; j++) if (i0 + j < n) { mm[j] = m[b * BLK8 + i0 + j]; vv[j] = v[b * BLK8 + i0 + j]; }
    unsigned mc, rc;
    int em, er;
    encode_block(mm, vv, half, mc, rc, em, er);
    store_codes(mp + b * BLK8, i0, n, false, mc);
    store_codes(rp + b * BLK8, i0, n, false, rc);
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
    GT_REQUIRE(ctx, w[i] && g[i] && m[i] && r[i] && e[i] && sizes[i] >= 0, "gt_adamw8_create: tensor %d has a null buffer or a negative size", i);
    GT_REQUIRE(ctx, (w[i] | g[i]) % 4 == 0 && e[i] % 2 == 0, "gt_adamw8_create: tensor %d: a buffer is not aligned to its elements", i);
    blocks += cdiv(sizes[i], BLK8);
    chunks += cdiv(sizes[i], CHUNK8);
  }
  GT_REQUIRE(ctx, blocks <= 0xffffffffll && chunks <= 0x7fffffffll, "gt_adamw8_create: %lld blocks are more than a group can number", (long long)blocks);
  gt_adamw *o = new gt_adamw();
  o->bits8 = true;
  o->n = n; o->beta1 = beta1; o->beta2 = beta2; o->eps = eps; o->wd = weight_decay; o->clip = clip;
  std::vector<Chunk8> ch;
  ch.reserve((size_t)chunks);
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
  const std::vector<double> zero(SSQ8_MAX_GROUPS + 1, 0.0);
  const float one[2] = {1.0f, 0.0f};
  hipError_t err;
  if ((err = hipMalloc((void **)&o->chunks8, std::max<size_t>(1, ch.size()) * sizeof(Chunk8))) != hipSuccess ||
      (err = hipMalloc((void **)&o->sums8, zero.size() * 8)) != hipSuccess || (err = hipMalloc((void **)&o->scale, 8)) != hipSuccess ||
      (!ch.empty() && (err = hipMemcpy(o->chunks8, ch.data(), ch.size() * sizeof(Chunk8), hipMemcpyHostToDevice)) != hipSuccess) ||
      (err = hipMemcpy(o->sums8, zero.data(), zero.size() * 8, hipMemcpyHostToDevice)) != hipSuccess ||
      (err = hipMemcpy(o->scale, one, 8, hipMemcpyHostToDevice)) != hipSuccess) {
    (void)hipGetLastError();
    adamw_release(o);
    GT_FAIL(ctx, "gt_adamw8_create: setting up the chunk tables failed: %s", hipGetErrorString(err));
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
  if (o->clip > 0) {
    const int nb = (int)std::min<int64_t>({o->nchunks, (int64_t)ctx->num_cu * 8, SSQ8_MAX_GROUPS});
    hipLaunchKernelGGL(adamw8_norm_k, dim3((unsigned)nb), dim3(256), 0, ctx->stream, o->chunks8, o->nchunks, o->sums8, o->clip, o->scale);
    GT_LAUNCHED(ctx);
  }
  // every constant is formed in f64 and rounded to f32 once
  Adam8H h{(float)o->beta1, (float)o->beta2, (float)(1.0 - o->beta1), (float)(1.0 - o->beta2), (float)o->eps, (float)o->wd,
           (float)lr, (float)(1.0 / bc1), (float)(1.0 / bc2), mix2((unsigned)seed ^ mix2((unsigned)(seed >> 32) + 0x9E3779B9u))};
  hipLaunchKernelGGL(adamw8_update_k, dim3((unsigned)o->nchunks), dim3(256), 0, ctx->stream, o->chunks8, o->scale, h);
  GT_LAUNCHED(ctx);
  return 0;
}

static int state8_of(gt_ctx *ctx, const char *who, gt_adamw *o, int i, const Tensor8 **t) {
  GT_REQUIRE(ctx, o && ctx->adamws.count(o), "%s: not an optimizer of this context", who);
  GT_REQUIRE(ctx, o->bits8, "%s: this group's states are held in 32 bits", who);
  GT_REQUIRE(ctx, i >= 0 && i < o->n, "%s: tensor %d of %d", who, i, o->n);
  *t = &o->tensors8[i];
  return 0;
}

int gt_adamw8_read(gt_ctx *ctx, gt_adamw *o, int i, gt_buf m, gt_buf v) {
  GT_ENTER(ctx);
  const Tensor8 *t;
  if (state8_of(ctx, "gt_adamw8_read", o, i, &t)) return 1;
  GT_REQUIRE(ctx, (m | v) % 4 == 0, "gt_adamw8_read: a buffer is not aligned to its elements");
  if (t->size == 0 || (!m && !v)) return 0;
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
  const unsigned nb = (unsigned)std::min<int64_t>(cdiv(t->size, 4 * BLK8), (int64_t)ctx->num_cu * 16);
  hipLaunchKernelGGL(state8_write_k, dim3(nb), dim3(256), 0, ctx->stream, t->size, t->m, t->r, t->e, P<const float>(m), P<const float>(v));
  GT_LAUNCHED(ctx);
  return 0;
}
}
