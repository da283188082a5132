// Per-head RMS normalisation of q and k and the NeoX rotation of the result in one pass each way: the two rmsNormHeads and
// two rope dispatches of a qwen3 / gemma3 layer (src/arch/qwen3.ts:153-195, src/arch/gemma3.ts:173-223; srcRmsNormFwd /
// BwdX / BwdW and srcRope, src/backend/wgsl.ts:217-303, 346-384).
//
//   forward   r = 1 / sqrt(mean(x^2) + eps);  y = x r w;  out_j = y_j c_j - y_{j+h} s_j,  out_{j+h} = y_j s_j + y_{j+h} c_j
//   backward  gy = R^T g (or g, where the rotation has been undone already);  S = sum(gy w x);
//             dx = r w gy - x r^3 S / hd;  dw = sum over rows and heads of gy x r                        (h = hd / 2)
//
// Bound by memory: 8 bytes per element forward, 12 backward, about 20 operations. 16384 rows of 16 + 8 heads of 128 take 63.4 us
// forward (6.35 TB/s) and 98 us backward (6.2 TB/s; the gain sums are another launch of 4 us); a large copy reaches 5.0.
// A head is handled by LPH lanes of one wavefront, each holding four elements of the lower half and the four of the upper half
// they are rotated with, so a pair never leaves its lane and the row sums are the only exchange. r is formed again in the
// backward (its row is in registers anyway) instead of being stored. Every row is read once and far from its next use: all
// accesses are streaming ones.
//
// The angle of pair j at position p is p * base^(-2j/hd). One thread per pair of the workgroup's rows forms it in 64 bits, as a
// fraction of a turn with the whole turns taken off, and leaves cos and sin in LDS for every head of the row: positions may
// be anything (a decoding batch's rows each have their own) and no table grows with them.
#include <algorithm>
#include <initializer_list>
#include "common.h"

typedef float v4f __attribute__((ext_vector_type(4)));

#define QK_MAX_HD 1024                           // the generic kernels keep a head's gain sums in LDS, one copy per wavefront
#define QK_MAX_HEADS 32768                       // of one side: a head's row is found by a 32-bit multiplication
#define QK_VEC_HD 512                            // 64 lanes of eight elements
// Measured on 16384 rows of 16 + 8 heads of 128 and of 10 + 2 heads of 64 (and 32768 rows of the former, backward):
//   forward: 4 to 6 passes (one row of the first) 65.6 and 19.5 us, 12 passes 68.5 and 20.3, 24 passes 71.2 and 20.1
//   backward, workgroups to a CU: 2: 102.7 (197) us, 3: 104.9 (206), 4: 109 (213), 8: 113 (218), 1: 122 (263). More of them read in
//   less of an order; loading a head ahead of its turn made it 111 (210) for the same reason. 12 passes: 33.3 us for heads of 64, 8: 36.3, 16: 35.6
#define QK_FWD_PASSES 6
#define QK_BWD_PASSES 12
#define QK_BWD_PER_CU 2
#define QK_SLICE_GROUPS (1 << 22)                // workgroups to a launch: a grid's threads are counted in 32 bits
#define QK_ANGLES 1024                           // pairs of a workgroup's rows whose cosines and sines LDS holds

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
  int64_t rows, first;                           // all rows, and the first of this launch
  int T, pos, hd;
  float eps;
};

// base^(-2j/hd) / (2 pi): turns per position of pair j
__device__ __forceinline__ double turns_per_place(double log2_base, int j, int hd) {
  return exp2(-2.0 * j / hd * log2_base) * 0.15915494309189533577;
}
// cos and sin of place * turns whole turns. The turns and then the quarters are taken off in 64 bits; what is left is at most an
// eighth of a turn either way, where Taylor's series to the ninth and tenth power is within 2e-9 of sin and cos, and within 7.3e-8 as it is
// evaluated in 32 bits.
__device__ __forceinline__ float2 cos_sin(double place, double turns) {
  double u = place * turns;
  u -= rint(u);
  const double q = rint(4.0 * u);
  const float t = (float)(u - 0.25 * q);
  const float a = __builtin_fmaf(t, 6.28318548f, t * -1.74845553e-7f);       // 2 pi in two parts
  const float z = a * a;
  const float s = __builtin_fmaf(a * z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 2.75573192e-6f, -1.98412698e-4f), 8.33333333e-3f), -1.66666667e-1f), a);
  const float c = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -2.75573192e-7f, 2.48015873e-5f), -1.38888889e-3f),
                                                                     4.16666667e-2f), -0.5f), 1.0f);
  const int k = (int)q;                          // -2 .. 2 quarters
  const float x = k & 1 ? s : c, y = k & 1 ? c : s;
  return make_float2(((k + 1) & 2) ? -x : x, (k & 2) ? -y : y);
}
__device__ __forceinline__ double place_of(const QkArgs &A, int64_t row) {
  return A.places ? (double)A.places[row] : (double)(row % A.T) + (double)A.pos;
}

// Sum over the LPH lanes of a head, in every one of them: within 16 lanes by exchanges of the vector unit, beyond through LDS.
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int LPH> __device__ __forceinline__ float head_sum(float v) {
  v = dpp_add<0xB1>(v);                          // neighbours
  v = dpp_add<0x4E>(v);                          // pairs
  if (LPH >= 8) v = dpp_add<0x141>(v);           // halves of eight
  if (LPH >= 16) v = dpp_add<0x140>(v);          // halves of sixteen
  if (LPH >= 32) v += __shfl_xor(v, 16, WAVE);
  if (LPH >= 64) v += __shfl_xor(v, 32, WAVE);
  return v;
}
__device__ __forceinline__ float sum4(v4f t) { return (t[0] + t[1]) + (t[2] + t[3]); }
// 1 / sqrt(t): the hardware's, which takes no denormals, and one Newton step; zero for infinity, where the step would make 0 * infinity
__device__ __forceinline__ float inv_root(float t) {
  const bool tiny = t < 1.17549435e-38f;
  t = tiny ? t * 1.84467441e19f : t;             // 2^64
  float y = __builtin_amdgcn_rsqf(t);
  if (t < __builtin_inff()) y = __builtin_fmaf(0.5f * y, __builtin_fmaf(-t * y, y, 1.0f), y);
  return tiny ? y * 4294967296.0f : y;
}

// What a workgroup keeps of its rows and the gains: [row][pair] cosines and sines, [side][hd].
struct alignas(16) QkShared { float c[QK_ANGLES], s[QK_ANGLES], w[2][QK_VEC_HD]; };

// A workgroup takes R rows at a time (R * hd/2 <= QK_ANGLES). Its wavefronts go through the rows' heads of q and then of k, 64 / LPH heads at a time, so that all of a wavefront is on one side and what differs between the sides is scalar.
struct QkPlan { int R, half, lq; unsigned mq, mk; };
__device__ __forceinline__ void shared_gains(const QkArgs &A, QkShared &L) {
  for (int i = threadIdx.x; i < 2 * A.hd; i += 256) L.w[i >= A.hd][i >= A.hd ? i - A.hd : i] = i >= A.hd ? A.s[1].w[i - A.hd] : A.s[0].w[i];
}

// A thread forms the angles of one pair, in every 256 / half-th row.
__device__ __forceinline__ void shared_angles(const QkArgs &A, QkShared &L, int64_t row0, int nr, int half, double turns) {
  const int step = 256 / half, r0 = threadIdx.x / half, j = threadIdx.x - r0 * half;
  if (r0 >= step) return;
  for (int r = r0; r < nr; r += step) {
    const float2 cs = cos_sin(place_of(A, row0 + r), turns);
    L.c[r * half + j] = cs.x;
    L.s[r * half + j] = cs.y;
  }
}

template <int LPH>
__global__ __launch_bounds__(256) void qk_norm_rope_fwd_k(QkArgs A, QkPlan P) {
  constexpr int UPW = WAVE / LPH;                // heads that a wavefront takes at once
  __shared__ QkShared L;
  const int half = P.half, lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int sub = lane / LPH, li = min(lane % LPH, P.lq - 1);
  const bool mine = lane % LPH < P.lq;
  const float invd = 1.0f / (float)A.hd;
  const int64_t row0 = A.first + (int64_t)blockIdx.x * P.R;
  const int nr = (int)min((int64_t)P.R, A.rows - row0);
  const int nq = nr * A.s[0].H, nk = nr * A.s[1].H, nqw = (nq + UPW - 1) / UPW, nw = nqw + (nk + UPW - 1) / UPW;
  shared_gains(A, L);
  shared_angles(A, L, row0, nr, half, turns_per_place(A.log2_base, threadIdx.x % half, A.hd));
  __syncthreads();
  for (int i = wave; i < nw; i += 4) {
    const int side = i >= nqw;
    const QkSide &S = A.s[side];
    const int u = (side ? i - nqw : i) * UPW + sub, n = side ? nk : nq;
    const bool live = mine && u < n;
    const int uc = min(u, n - 1);
    const int rr = (int)__umulhi(2u * uc, side ? P.mk : P.mq), h = uc - rr * S.H;
    const float *x = S.x + (row0 + rr) * S.ldx + (int64_t)h * A.hd;
    v4f a = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(x) + li), b = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(x + half) + li);
    const float ss = head_sum<LPH>(mine ? sum4(a * a + b * b) : 0.f);
    const float r = inv_root(ss * invd + A.eps);
    a = a * r * reinterpret_cast<const v4f *>(L.w[side])[li];
    b = b * r * reinterpret_cast<const v4f *>(L.w[side] + half)[li];
    const v4f c = reinterpret_cast<const v4f *>(L.c + rr * half)[li], sn = reinterpret_cast<const v4f *>(L.s + rr * half)[li];
    float *o = S.o + (row0 + rr) * S.ldo + (int64_t)h * A.hd;
    if (live) {
      __builtin_nontemporal_store(a * c - b * sn, reinterpret_cast<v4f *>(o) + li);
      __builtin_nontemporal_store(a * sn + b * c, reinterpret_cast<v4f *>(o + half) + li);
    }
  }
}

template <int LPH>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_k(QkArgs A, QkPlan P) {
  constexpr int UPW = WAVE / LPH;
  __shared__ QkShared L;
  __shared__ v4f red[2][4][QK_VEC_HD / 4];       // [side][wavefront][column]: the gain sums
  const int half = P.half, lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int sub = lane / LPH, li = min(lane % LPH, P.lq - 1);
  const bool mine = lane % LPH < P.lq;
  const float invd = 1.0f / (float)A.hd;
  const bool turn = A.s[0].rot | A.s[1].rot;
  const double turns = turn ? turns_per_place(A.log2_base, threadIdx.x % half, A.hd) : 0.0;
  v4f dw[2][2];
#pragma unroll
  for (int s = 0; s < 2; s++) dw[s][0] = dw[s][1] = v4f{0, 0, 0, 0};
  shared_gains(A, L);
  __syncthreads();
  for (int64_t row0 = (int64_t)blockIdx.x * P.R; row0 < A.rows; row0 += (int64_t)gridDim.x * P.R) {
    const int nr = (int)min((int64_t)P.R, A.rows - row0);
    const int nq = nr * A.s[0].H, nk = nr * A.s[1].H, nqw = (nq + UPW - 1) / UPW, nw = nqw + (nk + UPW - 1) / UPW;
    if (turn) {
      __syncthreads();
      shared_angles(A, L, row0, nr, half, turns);
      __syncthreads();
    }
    for (int i = wave; i < nw; i += 4) {
      const int side = i >= nqw;
      const QkSide &S = A.s[side];
      const int u = (side ? i - nqw : i) * UPW + sub, n = side ? nk : nq;
      const bool live = mine && u < n;
      const int uc = min(u, n - 1);
      const int rr = (int)__umulhi(2u * uc, side ? P.mk : P.mq), h = uc - rr * S.H;
      const int64_t xo = (row0 + rr) * S.ldx + (int64_t)h * A.hd, go = (row0 + rr) * S.ldo + (int64_t)h * A.hd;
      const v4f a = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(S.x + xo) + li);
      const v4f b = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(S.x + xo + half) + li);
      v4f ga = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(S.g + go) + li);
      v4f gb = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(S.g + go + half) + li);
      v4f oa = {0, 0, 0, 0}, ob = {0, 0, 0, 0};
      if (S.old) {
        oa = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(S.old + xo) + li);
        ob = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(S.old + xo + half) + li);
      }
      if (S.rot) {
        const v4f c = reinterpret_cast<const v4f *>(L.c + rr * half)[li], sn = reinterpret_cast<const v4f *>(L.s + rr * half)[li];
        const v4f ta = ga * c + gb * sn;
        gb = gb * c - ga * sn;
        ga = ta;
      }
      const v4f wa = reinterpret_cast<const v4f *>(L.w[side])[li], wb = reinterpret_cast<const v4f *>(L.w[side] + half)[li];
      const float ss = head_sum<LPH>(mine ? sum4(a * a + b * b) : 0.f);
      const float dot = head_sum<LPH>(mine ? sum4(ga * wa * a + gb * wb * b) : 0.f);
      const float r = inv_root(ss * invd + A.eps);
      // x r^3 S / hd as (x r) (r S / hd r), about as large as the result: the cube by itself would leave FP32 at rows below 1e-13
      const float k1 = r * dot * invd * r;
      if (S.o && live) {
        __builtin_nontemporal_store(wa * ga * r - a * r * k1 + oa, reinterpret_cast<v4f *>(S.o + xo) + li);
        __builtin_nontemporal_store(wb * gb * r - b * r * k1 + ob, reinterpret_cast<v4f *>(S.o + xo + half) + li);
      }
      const float rl = u < n ? r : 0.f;          // a head past the last one adds nothing
      const v4f ta = u < n ? ga * a * rl : v4f{0, 0, 0, 0}, tb = u < n ? gb * b * rl : v4f{0, 0, 0, 0};
      if (side) { dw[1][0] += ta; dw[1][1] += tb; }
      else { dw[0][0] += ta; dw[0][1] += tb; }
    }
  }
  // the sums of a wavefront's heads by exchanges, then the four wavefronts' in order: one partial row per workgroup and side
#pragma unroll
  for (int s = 0; s < 2; s++)
#pragma unroll
    for (int p = 0; p < 2; p++) {
#pragma unroll
      for (int o = LPH; o < WAVE; o *= 2)
#pragma unroll
        for (int j = 0; j < 4; j++) dw[s][p][j] += __shfl_xor(dw[s][p][j], o, WAVE);
      if (sub == 0 && mine) red[s][wave][p * P.lq + li] = dw[s][p];
    }
  __syncthreads();
  for (int t = threadIdx.x; t < 4 * P.lq; t += 256) {
    const int s = t >= 2 * P.lq, c = t - s * 2 * P.lq;
    if (A.s[s].part)
      reinterpret_cast<v4f *>(A.s[s].part + (size_t)blockIdx.x * A.hd)[c] = ((red[s][0][c] + red[s][1][c]) + red[s][2][c]) + red[s][3][c];
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
      const float r = 1.0f / sqrtf(ss / (float)A.hd + A.eps), k1 = r * dot / (float)A.hd * r;
      float *dw = acc + (size_t)(wave * 2 + side) * A.hd;
      for (int j = lane; j < half; j += WAVE) {
        const float c = S.rot ? cs[j].x : 1.f, sn = S.rot ? cs[j].y : 0.f;
        const float ga = g[j] * c + g[j + half] * sn, gb = g[j + half] * c - g[j] * sn;
        const float xa = x[j], xb = x[j + half];
        dw[j] += ga * xa * r;
        dw[j + half] += gb * xb * r;
        if (S.o) {
          const float oa = S.old ? S.old[xo + j] : 0.f, ob = S.old ? S.old[xo + j + half] : 0.f;
          S.o[xo + j] = S.w[j] * ga * r - xa * r * k1 + oa;
          S.o[xo + j + half] = S.w[j + half] * gb * r - xb * r * k1 + ob;
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
#define QK_LPH_OF(hd) ((hd) <= 32 ? 4 : (hd) <= 64 ? 8 : (hd) <= 128 ? 16 : (hd) <= 256 ? 32 : 64)
// Rows to a workgroup such that its wavefronts have `passes` heads (or groups of heads) to go through in all, as far as LDS holds
// their angles.
static int qk_rows_at_once(int heads, int hd, int passes) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(QK_ANGLES / (hd / 2), cdiv((int64_t)passes * (WAVE / QK_LPH_OF(hd)), heads)));
}
static QkPlan qk_plan(int hd, int R, int Hq, int Hk) {
  // u / H is the high word of 2 u * ceil(2^31 / H) where u * H < 2^31; u is below H + QK_BWD_PASSES * 16 here, H at most 2^15
  return {R, hd / 2, hd / 8, (unsigned)((0x80000000ull + Hq - 1) / Hq), (unsigned)((0x80000000ull + Hk - 1) / Hk)};
}
// A backward call's workgroups, one partial row of gain sums each, of the vector and of the generic kernel alike; and the rows that
// each takes at a time, fewer where that lets every workgroup have the same number of turns.
static int qk_bwd_rows(gt_ctx *ctx, int64_t rows, int heads, int hd) {
  if (hd % 8 || hd > QK_VEC_HD) return 1;
  const int64_t groups = (int64_t)ctx->num_cu * QK_BWD_PER_CU, turns = cdiv(rows, groups * qk_rows_at_once(heads, hd, QK_BWD_PASSES));
  return (int)cdiv(rows, groups * turns);
}
static int qk_bwd_groups(gt_ctx *ctx, int64_t rows, int heads, int hd) {
  return (int)std::min<int64_t>(cdiv(rows, qk_bwd_rows(ctx, rows, heads, hd)), (int64_t)ctx->num_cu * QK_BWD_PER_CU);
}

#define QK_LPH(hd, CALL) do { \
    switch (QK_LPH_OF(hd)) { case 4: CALL(4); break; case 8: CALL(8); break; case 16: CALL(16); break; case 32: CALL(32); break; \
      default: CALL(64); } } while (0)

static int qk_check(gt_ctx *ctx, const char *who, int rows, int T, int Hq, int Hkv, int hd, double base, gt_buf places, gt_buf q, int64_t ldq,
                    gt_buf wq, gt_buf k, int64_t ldk, gt_buf wk, int64_t ldqo, int64_t ldko) {
  GT_REQUIRE(ctx, rows >= 0 && (T >= 1 || places) && Hq >= 1 && Hkv >= 1 && q && wq && k && wk, "%s: bad arguments (rows %d, T %d, heads %d and %d)", who, rows,
             T, Hq, Hkv);
  GT_REQUIRE(ctx, hd >= 2 && hd % 2 == 0 && hd <= QK_MAX_HD, "%s: head size %d is not an even number up to %d", who, hd, QK_MAX_HD);
  GT_REQUIRE(ctx, base > 0 && base <= 1.7976931348623157e308, "%s: the rotation's base must be positive and finite", who);
  GT_REQUIRE(ctx, places || rows % T == 0, "%s: rows %d is not a whole number of sequences of %d", who, rows, T);
  GT_REQUIRE(ctx, Hq <= QK_MAX_HEADS && Hkv <= QK_MAX_HEADS, "%s: %d and %d heads are more than %d", who, Hq, Hkv, QK_MAX_HEADS);
  const int64_t nq = (int64_t)Hq * hd, nk = (int64_t)Hkv * hd;
  GT_REQUIRE(ctx, ldq >= nq && ldk >= nk && ldqo >= nq && ldko >= nk, "%s: a row stride is less than its row (%lld and %lld elements)", who,
             (long long)nq, (long long)nk);
  GT_REQUIRE(ctx, (q | wq | k | wk | places) % 4 == 0, "%s: a buffer is not aligned to its elements", who);
  return 0;
}

// Buffers of a call that it writes, and which of the others each may not share memory with: every workgroup writes while others still read.
// A buffer is `rows` runs of n bytes, ld bytes apart (a plain one: one run).
struct QkSpan { const char *name; uint64_t at; int64_t rows, ld, n; };
static QkSpan qk_plain(const char *name, gt_buf at, int64_t elems) { return {name, at, 1, 0, elems * 4}; }
static QkSpan qk_rows(const char *name, gt_buf at, int rows, int64_t ld, int64_t elems) { return {name, at, rows, ld * 4, elems * 4}; }
static bool qk_same(const QkSpan &a, const QkSpan &b) { return a.at == b.at && a.n == b.n && (a.ld == b.ld || (a.rows == 1 && b.rows == 1)); }
// Whether a run of a meets a run of b. Where the strides are the same (or one has a single run) that is a multiple k of the stride,
// 1 - b.rows <= k <= a.rows - 1, with b.at - a.at - a.n < k ld < b.at - a.at + b.n. Rows that interleave at different strides count as meeting.
static bool qk_meet(const QkSpan &a, const QkSpan &b) {
  if (!a.at || !b.at || a.rows < 1 || b.rows < 1 || a.n < 1 || b.n < 1) return false;
  typedef __int128 wide;
  const wide ea = (wide)a.at + (wide)(a.rows - 1) * a.ld + a.n, eb = (wide)b.at + (wide)(b.rows - 1) * b.ld + b.n;
  if (ea <= (wide)b.at || eb <= (wide)a.at) return false;
  if (a.rows > 1 && b.rows > 1 && a.ld != b.ld) return true;
  const wide ld = a.rows > 1 ? a.ld : b.rows > 1 ? b.ld : 1, far = (wide)b.at - (wide)a.at;
  const wide low = far - a.n;                    // the least k with k ld above it
  wide k = low >= 0 ? low / ld + 1 : -((-low + ld - 1) / ld) + 1;
  k = std::max<wide>(k, 1 - (wide)b.rows);
  return k <= (wide)a.rows - 1 && k * ld < far + b.n;
}
// out against everything in `others`; `self` may be out itself (in place)
static int qk_apart(gt_ctx *ctx, const char *who, const QkSpan &out, std::initializer_list<QkSpan> self, std::initializer_list<QkSpan> others) {
  for (const QkSpan &o : self)
    GT_REQUIRE(ctx, qk_same(out, o) || !qk_meet(out, o), "%s: %s and %s overlap (in place they have to be the same rows)", who, out.name, o.name);
  for (const QkSpan &o : others) GT_REQUIRE(ctx, !qk_meet(out, o), "%s: %s and %s overlap", who, out.name, o.name);
  return 0;
}

static int qk_bwd(gt_ctx *ctx, const char *who, int rows, int T, int Hq, int Hkv, int hd, float eps, double base, int pos, gt_buf places, gt_buf q,
                  int64_t ldq, gt_buf wq, gt_buf gq, int64_t ldgq, int rot_q, gt_buf dq, int acc_q, gt_buf part_q, gt_buf k, int64_t ldk, gt_buf wk,
                  gt_buf gk, int64_t ldgk, int rot_k, gt_buf dk, int acc_k, gt_buf part_k, gt_buf dwq, gt_buf dwk) {
  GT_REQUIRE(ctx, gq && gk && (gq | gk | dq | dk) % 4 == 0, "%s: a gradient is missing or not aligned to its elements", who);
  GT_REQUIRE(ctx, !(dq && dq == dk), "%s: dq and dk are the same buffer", who);
  GT_REQUIRE(ctx, !(dq == gq && ldq != ldgq) && !(dk == gk && ldk != ldgk), "%s: in place the strides have to be the same", who);
  const int nb = qk_bwd_groups(ctx, rows, Hq + Hkv, hd);
  const int64_t nq = (int64_t)Hq * hd, nk = (int64_t)Hkv * hd, np = (int64_t)nb * hd;
  const QkSpan sq = qk_rows("q", q, rows, ldq, nq), sk = qk_rows("k", k, rows, ldk, nk), sgq = qk_rows("gq", gq, rows, ldgq, nq),
               sgk = qk_rows("gk", gk, rows, ldgk, nk), sdq = qk_rows("dq", dq, rows, ldq, nq), sdk = qk_rows("dk", dk, rows, ldk, nk),
               swq = qk_plain("wq", wq, hd), swk = qk_plain("wk", wk, hd), sp = qk_plain("places", places, rows),
               spq = qk_plain("parts_q", part_q, np), spk = qk_plain("parts_k", part_k, np);
  if (qk_apart(ctx, who, sdq, {sq, sgq}, {sk, sgk, swq, swk, sp, sdk}) || qk_apart(ctx, who, sdk, {sk, sgk}, {sq, sgq, swq, swk, sp}) ||
      qk_apart(ctx, who, spq, {}, {sq, sk, sgq, sgk, swq, swk, sp, sdq, sdk, spk}) ||
      qk_apart(ctx, who, spk, {}, {sq, sk, sgq, sgk, swq, swk, sp, sdq, sdk})) return 1;
  // the gain gradients are written when everything has been read
  const QkSpan sdwq = qk_plain("dwq", dwq, hd), sdwk = qk_plain("dwk", dwk, hd);
  if (qk_apart(ctx, who, sdwq, {}, {sdq, sdk, sdwk}) || qk_apart(ctx, who, sdwk, {}, {sdq, sdk})) return 1;
  QkArgs A;
  memset(&A, 0, sizeof A);
  A.s[0] = {P<float>(q), P<float>(wq), P<float>(gq), acc_q ? P<float>(dq) : nullptr, P<float>(dq), P<float>(part_q), ldq, ldgq, Hq, rot_q != 0};
  A.s[1] = {P<float>(k), P<float>(wk), P<float>(gk), acc_k ? P<float>(dk) : nullptr, P<float>(dk), P<float>(part_k), ldk, ldgk, Hkv, rot_k != 0};
  A.places = P<const int>(places);
  A.log2_base = log2(base);
  A.rows = rows; A.T = T; A.pos = pos; A.hd = hd; A.eps = eps;
  if (qk_vec(hd, A.s[0], A.s[1])) {
    const QkPlan plan = qk_plan(hd, qk_bwd_rows(ctx, rows, Hq + Hkv, hd), Hq, Hkv);
#define CALL(L) hipLaunchKernelGGL((qk_norm_rope_bwd_k<L>), dim3((unsigned)nb), dim3(256), 0, ctx->stream, A, plan)
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
  GT_REQUIRE(ctx, qo != ko, "gt_qk_norm_rope_fwd: the two outputs are the same buffer");
  GT_REQUIRE(ctx, !(qo == q && ldqo != ldq) && !(ko == k && ldko != ldk), "gt_qk_norm_rope_fwd: in place the strides have to be the same");
  if (rows == 0) return 0;
  const int64_t nq = (int64_t)Hq * hd, nk = (int64_t)Hkv * hd;
  const QkSpan sq = qk_rows("q", q, rows, ldq, nq), sk = qk_rows("k", k, rows, ldk, nk), sqo = qk_rows("qo", qo, rows, ldqo, nq),
               sko = qk_rows("ko", ko, rows, ldko, nk), swq = qk_plain("wq", wq, hd), swk = qk_plain("wk", wk, hd), sp = qk_plain("places", places, rows);
  if (qk_apart(ctx, "gt_qk_norm_rope_fwd", sqo, {sq}, {sk, swq, swk, sp, sko}) || qk_apart(ctx, "gt_qk_norm_rope_fwd", sko, {sk}, {sq, swq, swk, sp})) return 1;
  ProfScope ps(ctx, "qknorm.rope", 8.0 * rows * (Hq + Hkv) * hd);
  QkArgs A;
  memset(&A, 0, sizeof A);
  A.s[0] = {P<float>(q), P<float>(wq), nullptr, nullptr, P<float>(qo), nullptr, ldq, ldqo, Hq, 1};
  A.s[1] = {P<float>(k), P<float>(wk), nullptr, nullptr, P<float>(ko), nullptr, ldk, ldko, Hkv, 1};
  A.places = P<const int>(places);
  A.log2_base = log2(base);
  A.rows = rows; A.T = T; A.pos = pos; A.hd = hd; A.eps = eps;
  if (qk_vec(hd, A.s[0], A.s[1])) {
    const QkPlan plan = qk_plan(hd, (int)std::min<int64_t>(qk_rows_at_once(Hq + Hkv, hd, QK_FWD_PASSES), std::max(1, rows / ctx->num_cu)), Hq, Hkv);
    const int64_t most = (int64_t)QK_SLICE_GROUPS * plan.R;
    for (A.first = 0; A.first < rows; A.first += most) {
      const unsigned nb = (unsigned)cdiv(std::min<int64_t>(most, rows - A.first), plan.R);
#define CALL(L) hipLaunchKernelGGL((qk_norm_rope_fwd_k<L>), dim3(nb), dim3(256), 0, ctx->stream, A, plan)
      QK_LPH(hd, CALL);
#undef CALL
    }
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
  const int nb = qk_bwd_groups(ctx, rows, Hq + Hkv, hd);
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
               ldgk, rot_k, dk, acc_k, pk, dwq, dwk)) return 1;
  }
  gt_buf sp[2], sd[2];
  int sn[2], sw[2], sa[2], n = 0;
  if (dwq) { sp[n] = pq; sn[n] = nb; sw[n] = hd; sd[n] = dwq; sa[n++] = acc_wq; }
  if (dwk) { sp[n] = pk; sn[n] = nb; sw[n] = hd; sd[n] = dwk; sa[n++] = acc_wk; }
  return gt_colsum_group(ctx, n, sp, sn, sw, sd, sa);
}

int gt_qk_norm_rope_parts_rows(gt_ctx *ctx, int rows, int Hq, int Hkv, int hd, int *nparts) {
  if (!ctx || !nparts) return 1;
  *nparts = rows >= 1 && Hq >= 1 && Hkv >= 1 && hd >= 2 && hd % 2 == 0 && hd <= QK_MAX_HD ? qk_bwd_groups(ctx, rows, Hq + Hkv, hd) : 0;
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
                ldk, wk, gk, ldgk, rot_k, dk, acc_k, parts_k, 0, 0);
}
}
