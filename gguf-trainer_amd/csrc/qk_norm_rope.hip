// Per-head RMS normalisation of q and k and the NeoX rotation of the result in one pass each way: the two rmsNormHeads and
// two rope dispatches of a qwen3 / gemma3 layer (src/arch/qwen3.ts:153-195, src/arch/gemma3.ts:173-223; srcRmsNormFwd /
// BwdX / BwdW and srcRope, src/backend/wgsl.ts:217-303, 346-384).
//
//   forward   r = 1 / sqrt(mean(x^2) + eps);  y = x r w;  out_j = y_j c_j - y_{j+h} s_j,  out_{j+h} = y_j s_j + y_{j+h} c_j
//   backward  gy = R^T g (or g, where the rotation has been undone already);  S = sum(gy w x);
//             dx = r w gy - x r^3 S / hd;  dw = sum over rows and heads of gy x r                        (h = hd / 2)
//
// Bound by memory: 8 bytes per element forward, 12 backward, about 20 operations. A head is handled by LPH lanes of one
// wavefront, each holding four elements of the lower half and the four of the upper half they are rotated with, so a pair
// never leaves its lane and the row sums are the only exchange. r is formed again in the backward (its row is in registers
// anyway) instead of being stored.
//
// The angle of pair j at position p is p * base^(-2j/hd). One thread per (row, pair) of the workgroup's rows forms it in
// 64 bits, as a fraction of a turn with the whole turns taken off, and leaves cos and sin in LDS for every head of the row:
// positions may be anything (a decoding batch's rows each have their own) and no table grows with them.
#include <algorithm>
#include "common.h"

typedef float v4f __attribute__((ext_vector_type(4)));

#define QK_MAX_HD 1024                           // the generic kernels keep a head's gain sums in LDS, one copy per wavefront
#define QK_VEC_HD 512                            // 64 lanes of eight elements

struct QkSide {
  const float *x, *w, *g, *old;                  // rows before the norm, gain, (backward) gradient, what dx is added to
  float *o;                                      // forward: rotated rows, backward: dx (0: not wanted)
  float *part;                                   // backward: one partial row of gain sums per workgroup (0: not wanted)
  int64_t ldx, ldo;                              // elements between rows: of x and dx; of the rotated side (out, g)
  int H, rot;
};
struct QkArgs {
  QkSide s[2];                                   // q, k
  const int *places;                             // position of each row, or 0: (row mod T) + pos
  double log2_base;
  int64_t rows;
  int T, pos, hd;
  float eps;
};

// base^(-2j/hd) / (2 pi): turns per position of pair j
__device__ __forceinline__ double turns_per_place(double log2_base, int j, int hd) {
  return exp2(-2.0 * j / hd * log2_base) * 0.15915494309189533577;
}
__device__ __forceinline__ float2 cos_sin(double place, double turns) {
  double u = place * turns;
  u -= rint(u);
  double s, c;
  sincospi(2.0 * u, &s, &c);
  return make_float2((float)c, (float)s);
}
__device__ __forceinline__ double place_of(const QkArgs &A, int64_t row) {
  return A.places ? (double)A.places[row] : (double)(row % A.T) + (double)A.pos;
}

template <int LPH> __device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
  return v;
}
__device__ __forceinline__ float sum4(v4f t) { return (t[0] + t[1]) + (t[2] + t[3]); }

// A workgroup takes R rows at a time (R * hd/2 <= 256 angles, one per thread) and its 256 / LPH lane groups go through the
// rows' heads, those of q and then those of k row by row.
template <int LPH>
__global__ __launch_bounds__(256) void qk_norm_rope_fwd_k(QkArgs A, int R) {
  constexpr int G = 256 / LPH;
  __shared__ float2 cs[256];
  const int half = A.hd / 2, lq = A.hd / 8;
  const int grp = threadIdx.x / LPH, li = min((int)threadIdx.x % LPH, lq - 1);
  const bool live = (int)threadIdx.x % LPH < lq;
  const int Hq = A.s[0].H, Ht = Hq + A.s[1].H;
  const float invd = 1.0f / (float)A.hd;
  const int ar = threadIdx.x / half, aj = threadIdx.x % half;
  const double turns = turns_per_place(A.log2_base, aj, A.hd);
  v4f w[2][2];
#pragma unroll
  for (int s = 0; s < 2; s++)
#pragma unroll
    for (int p = 0; p < 2; p++) w[s][p] = reinterpret_cast<const v4f *>(A.s[s].w + p * half)[li];
  for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < A.rows; row0 += (int64_t)gridDim.x * R) {
    const int nr = (int)min((int64_t)R, A.rows - row0);
    __syncthreads();
    if (ar < nr) cs[threadIdx.x] = cos_sin(place_of(A, row0 + ar), turns);
    __syncthreads();
    for (int u = grp; u < nr * Ht; u += G) {
      const int rr = u / Ht, h = u - rr * Ht;
      const bool isk = h >= Hq;
      const QkSide &S = isk ? A.s[1] : A.s[0];
      const int hh = isk ? h - Hq : h;
      const float *x = S.x + (row0 + rr) * S.ldx + (int64_t)hh * A.hd;
      v4f a = reinterpret_cast<const v4f *>(x)[li], b = reinterpret_cast<const v4f *>(x + half)[li];
      const v4f q2 = a * a + b * b;
      const float ss = head_sum<LPH>(live ? sum4(q2) : 0.f);
      const float r = 1.0f / sqrtf(ss * invd + A.eps);
      a = a * r * (isk ? w[1][0] : w[0][0]);
      b = b * r * (isk ? w[1][1] : w[0][1]);
      const v4f *cp = reinterpret_cast<const v4f *>(cs + rr * half + 4 * li);
      const v4f c0 = cp[0], c1 = cp[1];
      const v4f c = {c0[0], c0[2], c1[0], c1[2]}, sn = {c0[1], c0[3], c1[1], c1[3]};
      float *o = S.o + (row0 + rr) * S.ldo + (int64_t)hh * A.hd;
      if (live) {
        reinterpret_cast<v4f *>(o)[li] = a * c - b * sn;
        reinterpret_cast<v4f *>(o + half)[li] = a * sn + b * c;
      }
    }
  }
}

template <int LPH>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_k(QkArgs A, int R) {
  constexpr int G = 256 / LPH;
  __shared__ float2 cs[256];
  __shared__ v4f red[2][256];                    // [half][lane group][lane]: the gain sums of one side
  const int half = A.hd / 2, lq = A.hd / 8;
  const int grp = threadIdx.x / LPH, li = min((int)threadIdx.x % LPH, lq - 1);
  const bool live = (int)threadIdx.x % LPH < lq;
  const int Hq = A.s[0].H, Ht = Hq + A.s[1].H;
  const float invd = 1.0f / (float)A.hd;
  const bool turn = A.s[0].rot | A.s[1].rot;
  const int ar = threadIdx.x / half, aj = threadIdx.x % half;
  const double turns = turn ? turns_per_place(A.log2_base, aj, A.hd) : 0.0;
  v4f w[2][2], dw[2][2];
#pragma unroll
  for (int s = 0; s < 2; s++)
#pragma unroll
    for (int p = 0; p < 2; p++) {
      w[s][p] = reinterpret_cast<const v4f *>(A.s[s].w + p * half)[li];
      dw[s][p] = v4f{0, 0, 0, 0};
    }
  for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < A.rows; row0 += (int64_t)gridDim.x * R) {
    const int nr = (int)min((int64_t)R, A.rows - row0);
    if (turn) {
      __syncthreads();
      if (ar < nr) cs[threadIdx.x] = cos_sin(place_of(A, row0 + ar), turns);
      __syncthreads();
    }
    for (int u = grp; u < nr * Ht; u += G) {
      const int rr = u / Ht, h = u - rr * Ht;
      const bool isk = h >= Hq;
      const QkSide &S = isk ? A.s[1] : A.s[0];
      const int hh = isk ? h - Hq : h;
      const int64_t xo = (row0 + rr) * S.ldx + (int64_t)hh * A.hd, go = (row0 + rr) * S.ldo + (int64_t)hh * A.hd;
      const v4f a = reinterpret_cast<const v4f *>(S.x + xo)[li], b = reinterpret_cast<const v4f *>(S.x + xo + half)[li];
      v4f ga = reinterpret_cast<const v4f *>(S.g + go)[li], gb = reinterpret_cast<const v4f *>(S.g + go + half)[li];
      v4f oa = {0, 0, 0, 0}, ob = {0, 0, 0, 0};
      if (S.old) {
        oa = reinterpret_cast<const v4f *>(S.old + xo)[li];
        ob = reinterpret_cast<const v4f *>(S.old + xo + half)[li];
      }
      if (S.rot) {
        const v4f *cp = reinterpret_cast<const v4f *>(cs + rr * half + 4 * li);
        const v4f c0 = cp[0], c1 = cp[1];
        const v4f c = {c0[0], c0[2], c1[0], c1[2]}, sn = {c0[1], c0[3], c1[1], c1[3]};
        const v4f ta = ga * c + gb * sn;
        gb = gb * c - ga * sn;
        ga = ta;
      }
      const v4f wa = isk ? w[1][0] : w[0][0], wb = isk ? w[1][1] : w[0][1];
      const float ss = head_sum<LPH>(live ? sum4(a * a + b * b) : 0.f);
      const float dot = head_sum<LPH>(live ? sum4(ga * wa * a + gb * wb * b) : 0.f);
      const float r = 1.0f / sqrtf(ss * invd + A.eps);
      const float k2 = r * r * r * dot * invd;
      if (S.o && live) {
        reinterpret_cast<v4f *>(S.o + xo)[li] = wa * ga * r - a * k2 + oa;
        reinterpret_cast<v4f *>(S.o + xo + half)[li] = wb * gb * r - b * k2 + ob;
      }
      const v4f ta = ga * a * r, tb = gb * b * r;
      if (isk) { dw[1][0] += ta; dw[1][1] += tb; }
      else { dw[0][0] += ta; dw[0][1] += tb; }
    }
  }
  // the lane groups' sums in group order, one partial row per workgroup and side
#pragma unroll
  for (int s = 0; s < 2; s++) {
    if (!A.s[s].part) continue;
    __syncthreads();
    red[0][threadIdx.x] = dw[s][0];
    red[1][threadIdx.x] = dw[s][1];
    __syncthreads();
    const int t = threadIdx.x;
    if (t < 2 * lq) {
      const int p = t / lq, l = t - p * lq;
      v4f sum = red[p][l];
      for (int q = 1; q < G; q++) sum += red[p][q * LPH + l];
      reinterpret_cast<v4f *>(A.s[s].part + (size_t)blockIdx.x * A.hd + p * half)[l] = sum;
    }
  }
}

// Any even hd up to QK_MAX_HD, any alignment and stride: a workgroup takes one row at a time, a wavefront one head at a
// time, a lane every 64th pair of it.
__global__ __launch_bounds__(256) void qk_norm_rope_fwd_gen(QkArgs A) {
  __shared__ float2 cs[QK_MAX_HD / 2];
  const int half = A.hd / 2, lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
  const int Hq = A.s[0].H, Ht = Hq + A.s[1].H;
  for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
    __syncthreads();
    for (int j = threadIdx.x; j < half; j += 256) cs[j] = cos_sin(place_of(A, row), turns_per_place(A.log2_base, j, A.hd));
    __syncthreads();
    for (int h = wave; h < Ht; h += 4) {
      const QkSide &S = h >= Hq ? A.s[1] : A.s[0];
      const int hh = h >= Hq ? h - Hq : h;
      const float *x = S.x + row * S.ldx + (int64_t)hh * A.hd;
      float *o = S.o + row * S.ldo + (int64_t)hh * A.hd;
      float ss = 0;
      for (int j = lane; j < half; j += WAVE) ss += x[j] * x[j] + x[j + half] * x[j + half];
      const float r = 1.0f / sqrtf(wave_sum(ss) / (float)A.hd + A.eps);
      for (int j = lane; j < half; j += WAVE) {
        const float a = x[j] * r * S.w[j], b = x[j + half] * r * S.w[j + half];
        o[j] = a * cs[j].x - b * cs[j].y;
        o[j + half] = a * cs[j].y + b * cs[j].x;
      }
    }
  }
}
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_gen(QkArgs A) {
  __shared__ float2 cs[QK_MAX_HD / 2];
  extern __shared__ float acc[];                 // [wavefront][side][hd]: a column belongs to one lane of its wavefront
  const int half = A.hd / 2, lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
  const int Hq = A.s[0].H, Ht = Hq + A.s[1].H;
  for (int i = threadIdx.x; i < 8 * A.hd; i += 256) acc[i] = 0.f;
  for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
    __syncthreads();
    for (int j = threadIdx.x; j < half; j += 256) cs[j] = cos_sin(place_of(A, row), turns_per_place(A.log2_base, j, A.hd));
    __syncthreads();
    for (int h = wave; h < Ht; h += 4) {
      const int side = h >= Hq;
      const QkSide &S = A.s[side];
      const int hh = side ? h - Hq : h;
      const int64_t xo = row * S.ldx + (int64_t)hh * A.hd;
      const float *x = S.x + xo, *g = S.g + row * S.ldo + (int64_t)hh * A.hd;
      float ss = 0, dot = 0;
      for (int j = lane; j < half; j += WAVE) {
        const float c = S.rot ? cs[j].x : 1.f, sn = S.rot ? cs[j].y : 0.f;
        const float ga = g[j] * c + g[j + half] * sn, gb = g[j + half] * c - g[j] * sn;
        ss += x[j] * x[j] + x[j + half] * x[j + half];
        dot += ga * S.w[j] * x[j] + gb * S.w[j + half] * x[j + half];
      }
      ss = wave_sum(ss);
      dot = wave_sum(dot);
      const float r = 1.0f / sqrtf(ss / (float)A.hd + A.eps), k2 = r * r * r * dot / (float)A.hd;
      float *dw = acc + (size_t)(wave * 2 + side) * A.hd;
      for (int j = lane; j < half; j += WAVE) {
        const float c = S.rot ? cs[j].x : 1.f, sn = S.rot ? cs[j].y : 0.f;
        const float ga = g[j] * c + g[j + half] * sn, gb = g[j + half] * c - g[j] * sn;
        const float xa = x[j], xb = x[j + half];
        dw[j] += ga * xa * r;
        dw[j + half] += gb * xb * r;
        if (S.o) {
          const float oa = S.old ? S.old[xo + j] : 0.f, ob = S.old ? S.old[xo + j + half] : 0.f;
          S.o[xo + j] = S.w[j] * ga * r - xa * k2 + oa;
          S.o[xo + j + half] = S.w[j + half] * gb * r - xb * k2 + ob;
        }
      }
    }
  }
  __syncthreads();
  for (int s = 0; s < 2; s++)
    if (A.s[s].part)
      for (int c = threadIdx.x; c < A.hd; c += 256) {
        float sum = acc[(size_t)s * A.hd + c];
        for (int wv = 1; wv < 4; wv++) sum += acc[(size_t)(wv * 2 + s) * A.hd + c];
        A.s[s].part[(size_t)blockIdx.x * A.hd + c] = sum;
      }
}
__global__ __launch_bounds__(256) void qk_gain_clear_k(int n, float *a, float *b) {
  for (int i = threadIdx.x; i < n; i += 256) {
    if (a) a[i] = 0.f;
    if (b) b[i] = 0.f;
  }
}

// 16-byte chunks throughout, and heads that 64 lanes of eight elements hold
static bool qk_vec(int hd, const QkSide &q, const QkSide &k) {
  if (hd % 8 || hd > QK_VEC_HD) return false;
  uintptr_t bits = 0;
  for (const QkSide *s : {&q, &k}) {
    for (const float *p : {s->x, s->w, s->g, s->old, (const float *)s->o, (const float *)s->part}) bits |= reinterpret_cast<uintptr_t>(p);
    if (s->ldx % 4 || s->ldo % 4) return false;
  }
  return bits % 16 == 0;
}
static int qk_rows_at_once(int hd) { return std::max(1, 256 / (hd / 2)); }
// workgroups of a backward call, vector or generic kernel alike: one partial row of gain sums each
static int qk_bwd_groups(gt_ctx *ctx, int64_t rows, int hd) {
  const int R = hd % 8 == 0 && hd <= QK_VEC_HD ? qk_rows_at_once(hd) : 1;
  return (int)std::min<int64_t>(cdiv(rows, R), (int64_t)ctx->num_cu * 4);
}

#define QK_LPH(hd, CALL) do { \
    if ((hd) <= 32) { CALL(4); } else if ((hd) <= 64) { CALL(8); } else if ((hd) <= 128) { CALL(16); } \
    else if ((hd) <= 256) { CALL(32); } else { CALL(64); } } while (0)

static int qk_check(gt_ctx *ctx, const char *who, int rows, int T, int Hq, int Hkv, int hd, double base, gt_buf places, gt_buf q, int64_t ldq,
                    gt_buf wq, gt_buf k, int64_t ldk, gt_buf wk, int64_t ldqo, int64_t ldko) {
  GT_REQUIRE(ctx, rows >= 0 && T >= 1 && Hq >= 1 && Hkv >= 1 && q && wq && k && wk, "%s: bad arguments (rows %d, T %d, heads %d and %d)", who, rows,
             T, Hq, Hkv);
  GT_REQUIRE(ctx, hd >= 2 && hd % 2 == 0 && hd <= QK_MAX_HD, "%s: head size %d is not an even number up to %d", who, hd, QK_MAX_HD);
  GT_REQUIRE(ctx, base > 0, "%s: the rotation's base must be positive", who);
  GT_REQUIRE(ctx, places || rows % T == 0, "%s: rows %d is not a whole number of sequences of %d", who, rows, T);
  const int64_t nq = (int64_t)Hq * hd, nk = (int64_t)Hkv * hd;
  GT_REQUIRE(ctx, ldq >= nq && ldk >= nk && ldqo >= nq && ldko >= nk, "%s: a row stride is less than its row (%lld and %lld elements)", who,
             (long long)nq, (long long)nk);
  GT_REQUIRE(ctx, (q | wq | k | wk | places) % 4 == 0, "%s: a buffer is not aligned to its elements", who);
  return 0;
}

static int qk_bwd(gt_ctx *ctx, const char *who, int rows, int T, int Hq, int Hkv, int hd, float eps, double base, int pos, gt_buf places, gt_buf q,
                  int64_t ldq, gt_buf wq, gt_buf gq, int64_t ldgq, int rot_q, gt_buf dq, int acc_q, gt_buf part_q, gt_buf k, int64_t ldk, gt_buf wk,
                  gt_buf gk, int64_t ldgk, int rot_k, gt_buf dk, int acc_k, gt_buf part_k) {
  GT_REQUIRE(ctx, gq && gk && (gq | gk | dq | dk) % 4 == 0, "%s: a gradient is missing or not aligned to its elements", who);
  QkArgs A;
  memset(&A, 0, sizeof A);
  A.s[0] = {P<float>(q), P<float>(wq), P<float>(gq), acc_q ? P<float>(dq) : nullptr, P<float>(dq), P<float>(part_q), ldq, ldgq, Hq, rot_q != 0};
  A.s[1] = {P<float>(k), P<float>(wk), P<float>(gk), acc_k ? P<float>(dk) : nullptr, P<float>(dk), P<float>(part_k), ldk, ldgk, Hkv, rot_k != 0};
  A.places = P<const int>(places);
  A.log2_base = log2(base);
  A.rows = rows; A.T = T; A.pos = pos; A.hd = hd; A.eps = eps;
  const int nb = qk_bwd_groups(ctx, rows, hd);
  if (qk_vec(hd, A.s[0], A.s[1])) {
    const int R = qk_rows_at_once(hd);
#define CALL(L) hipLaunchKernelGGL((qk_norm_rope_bwd_k<L>), dim3((unsigned)nb), dim3(256), 0, ctx->stream, A, R)
    QK_LPH(hd, CALL);
#undef CALL
  } else {
    hipLaunchKernelGGL(qk_norm_rope_bwd_gen, dim3((unsigned)nb), dim3(256), (size_t)8 * hd * sizeof(float), ctx->stream, A);
  }
  GT_LAUNCHED(ctx);
  return 0;
}

extern "C" {

int gt_qk_norm_rope_fwd(gt_ctx *ctx, int rows, int T, int Hq, int Hkv, int hd, float eps, double base, int pos, gt_buf places, gt_buf q, int64_t ldq,
                        gt_buf wq, gt_buf qo, int64_t ldqo, gt_buf k, int64_t ldk, gt_buf wk, gt_buf ko, int64_t ldko) {
  GT_ENTER(ctx);
  if (qk_check(ctx, "gt_qk_norm_rope_fwd", rows, T, Hq, Hkv, hd, base, places, q, ldq, wq, k, ldk, wk, ldqo, ldko)) return 1;
  GT_REQUIRE(ctx, qo && ko && (qo | ko) % 4 == 0, "gt_qk_norm_rope_fwd: an output is missing or not aligned to its elements");
  if (rows == 0) return 0;
  ProfScope ps(ctx, "qknorm.rope", 8.0 * rows * (Hq + Hkv) * hd);
  QkArgs A;
  memset(&A, 0, sizeof A);
  A.s[0] = {P<float>(q), P<float>(wq), nullptr, nullptr, P<float>(qo), nullptr, ldq, ldqo, Hq, 1};
  A.s[1] = {P<float>(k), P<float>(wk), nullptr, nullptr, P<float>(ko), nullptr, ldk, ldko, Hkv, 1};
  A.places = P<const int>(places);
  A.log2_base = log2(base);
  A.rows = rows; A.T = T; A.pos = pos; A.hd = hd; A.eps = eps;
  if (qk_vec(hd, A.s[0], A.s[1])) {
    const int R = qk_rows_at_once(hd);
    const unsigned nb = (unsigned)std::min<int64_t>(cdiv(rows, R), (int64_t)ctx->num_cu * 8);
#define CALL(L) hipLaunchKernelGGL((qk_norm_rope_fwd_k<L>), dim3(nb), dim3(256), 0, ctx->stream, A, R)
    QK_LPH(hd, CALL);
#undef CALL
  } else {
    const unsigned nb = (unsigned)std::min<int64_t>(rows, (int64_t)ctx->num_cu * 8);
    hipLaunchKernelGGL(qk_norm_rope_fwd_gen, dim3(nb), dim3(256), 0, ctx->stream, A);
  }
  GT_LAUNCHED(ctx);
  return 0;
}

int gt_qk_norm_rope_bwd(gt_ctx *ctx, int rows, int T, int Hq, int Hkv, int hd, float eps, double base, int pos, gt_buf places, gt_buf q, int64_t ldq,
                        gt_buf wq, gt_buf gq, int64_t ldgq, int rot_q, gt_buf dq, int acc_q, gt_buf dwq, int acc_wq, gt_buf k, int64_t ldk, gt_buf wk,
                        gt_buf gk, int64_t ldgk, int rot_k, gt_buf dk, int acc_k, gt_buf dwk, int acc_wk) {
  GT_ENTER(ctx);
  if (qk_check(ctx, "gt_qk_norm_rope_bwd", rows, T, Hq, Hkv, hd, base, places, q, ldq, wq, k, ldk, wk, ldgq, ldgk)) return 1;
  GT_REQUIRE(ctx, (dwq | dwk) % 4 == 0 && !(dwq && dwq == dwk), "gt_qk_norm_rope_bwd: the gain gradients are misaligned or one and the same");
  if (rows == 0) {
    float *a = dwq && !acc_wq ? P<float>(dwq) : nullptr, *b = dwk && !acc_wk ? P<float>(dwk) : nullptr;
    if (a || b) {
      hipLaunchKernelGGL(qk_gain_clear_k, dim3(1), dim3(256), 0, ctx->stream, hd, a, b);
      GT_LAUNCHED(ctx);
    }
    return 0;
  }
  if (!dq && !dk && !dwq && !dwk) return 0;
  const int nb = qk_bwd_groups(ctx, rows, hd);
  const size_t one = ((size_t)nb * hd + 3) / 4 * 4;
  float *parts = nullptr;
  if (dwq || dwk) {
    void *ws;
    if (gt_ws_reserve(ctx, 2 * one * sizeof(float), &ws)) return 1;
    parts = static_cast<float *>(ws);
  }
  const gt_buf pq = dwq ? reinterpret_cast<gt_buf>(parts) : 0, pk = dwk ? reinterpret_cast<gt_buf>(parts + one) : 0;
  {
    ProfScope ps(ctx, "qknorm.rope.bwd", 12.0 * rows * (Hq + Hkv) * hd);
    if (qk_bwd(ctx, "gt_qk_norm_rope_bwd", rows, T, Hq, Hkv, hd, eps, base, pos, places, q, ldq, wq, gq, ldgq, rot_q, dq, acc_q, pq, k, ldk, wk, gk,
               ldgk, rot_k, dk, acc_k, pk)) return 1;
  }
  gt_buf sp[2], sd[2];
  int sn[2], sw[2], sa[2], n = 0;
  if (dwq) { sp[n] = pq; sn[n] = nb; sw[n] = hd; sd[n] = dwq; sa[n++] = acc_wq; }
  if (dwk) { sp[n] = pk; sn[n] = nb; sw[n] = hd; sd[n] = dwk; sa[n++] = acc_wk; }
  return gt_colsum_group(ctx, n, sp, sn, sw, sd, sa);
}

int gt_qk_norm_rope_parts_rows(gt_ctx *ctx, int rows, int hd, int *nparts) {
  if (!ctx || !nparts) return 1;
  *nparts = rows >= 1 && hd >= 2 && hd % 2 == 0 && hd <= QK_MAX_HD ? qk_bwd_groups(ctx, rows, hd) : 0;
  return 0;
}

int gt_qk_norm_rope_bwd_parts(gt_ctx *ctx, int rows, int T, int Hq, int Hkv, int hd, float eps, double base, int pos, gt_buf places, gt_buf q,
                              int64_t ldq, gt_buf wq, gt_buf gq, int64_t ldgq, int rot_q, gt_buf dq, int acc_q, gt_buf parts_q, gt_buf k, int64_t ldk,
                              gt_buf wk, gt_buf gk, int64_t ldgk, int rot_k, gt_buf dk, int acc_k, gt_buf parts_k) {
  GT_ENTER(ctx);
  if (qk_check(ctx, "gt_qk_norm_rope_bwd_parts", rows, T, Hq, Hkv, hd, base, places, q, ldq, wq, k, ldk, wk, ldgq, ldgk)) return 1;
  GT_REQUIRE(ctx, rows >= 1 && (parts_q || parts_k) && (parts_q | parts_k) % 16 == 0,
             "gt_qk_norm_rope_bwd_parts: bad arguments (rows %d; 16-byte aligned partial rows for q, k or both)", rows);
  ProfScope ps(ctx, "qknorm.rope.bwd", 12.0 * rows * (Hq + Hkv) * hd);
  return qk_bwd(ctx, "gt_qk_norm_rope_bwd_parts", rows, T, Hq, Hkv, hd, eps, base, pos, places, q, ldq, wq, gq, ldgq, rot_q, dq, acc_q, parts_q, k,
                ldk, wk, gk, ldgk, rot_k, dk, acc_k, parts_k);
}
}
