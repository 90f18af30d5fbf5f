// Losses of a linear vocabulary head, z = hidden . weight^T + bias, whose logits are never kept (csrc/vocab_gemm.inc has the tiles).
//
//   cross entropy            l_r = lse(z_r) - z_r[y_r]
//   top-logit distillation   q = softmax(t / T) over the K entries a teacher gives for row r,
//                            l_r = T^2 sum_k q_k (log q_k - z_r[i_k] / T + lse(z_r / T))
//   both with target q (one entry of weight 1 for the label) and u = z / T:
//       d l / d z_r[v] = T (exp(u_rv - lse(u_r)) - q_r[v]),     d hidden = dz . weight,  d weight = dz^T . hidden,  d bias = sum_r dz_r
//
// A call, in launches:
//   targets      (distillation) the teacher's softmax per row; entries of one token are merged; rows with no entry do not count
//   compact      row numbers of the rows that count, in order; how many
//   gather       those rows of `hidden`, next to one another, padded with zero rows and columns: a row that does not count takes no
//                part in any product, so whatever its hidden state holds (NaN, infinities) reaches nothing
//   lse          logits tile by tile, every lane keeping a running maximum and sum of its own columns; a workgroup walks a slice of
//                the vocabulary for one block of rows, slices are joined by `finish`
//   finish       row losses in the caller's order, lse
//   reduce       their sum or mean in a fixed order
// and for the gradients, one piece of the vocabulary after the other (as many columns as the workspace holds):
//   dlogits      the same products again, then g (p - q) rounded to bf16: the operand type of the two products that follow.  The
//                rounding is 2^-9 of each entry, independent from entry to entry, and the targets are subtracted before it.
//                Column sums for d bias are taken from the unrounded values.
//   dhidden      split over the vocabulary into fp32 slabs that later pieces add to; `dh_join` adds the slabs in order
//   dweight      the piece's rows of d weight, complete
// Nothing is accumulated with atomics: equal calls give equal bits.
#define CACO_WAVE_SYNC_FENCE
#include "common.h"
#include "kernels.h"
#include "vocab_gemm.inc"

namespace caco {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int MAX_WG = 512;          // most workgroups of a persistent launch (two per CU)
constexpr int DH_UNITS = 512;        // (row block, column block, slab) units that fill the chip in `dhidden`

typedef VgTile<8, 4, 2, 4> Big;      // 256 x 256, one workgroup per CU
typedef VgTile<4, 2, 1, 4> Small;    // 64 x 128, two per CU: 64 tokens or fewer, where a call reads the weights and does little else

// what the kernels share; device pointers into the caller's tensors or the workspace
struct LossArgs {
  const bf16_t* hidden; int64_t ld_h;
  const bf16_t* weight; int64_t ld_w;
  const float* bias;
  const int64_t* labels; int64_t ignore_index;
  const float* teacher; int64_t ld_t;
  const void* teacher_idx; int64_t ld_i; int idx64;
  int topk, kp;                      // entries per row; kp = next power of two, the pitch of the target lists
  float inv_t, temperature;
  int64_t rows; int vocab, dim, hp;  // hp = dim rounded up to the K-tile
  int reduction;
  const float* row_weight;
  const float* grad_scale;
  float *row_loss, *lse, *loss;
  bf16_t* dh; int64_t ld_dh;
  bf16_t* dw; int64_t ld_dw;
  float* db;
  // workspace
  int* count;                        // rows that count
  int *rowmap, *inv;                 // compact -> caller's row; caller's row -> compact or -1
  int *tgt_idx0; float *tgt_q0;      // targets in the caller's order [rows, kp] (distillation)
  int *tgt_idx; float *tgt_q;        // targets of the compact rows [npad, kp]
  bf16_t* hc;                        // [npad, hp]
  float2* part;                      // (max, sum) of log2-logits, [slice][row block rows]
  float* zt;                         // cross entropy: the label's log2-logit; distillation: sum_k q_k (log q_k - z_k / T)
  float *lse2, *g;                   // compact: lse in log2 units, gradient scale of the row
  bf16_t* dl;                        // [npad, piece]
  float* slab;                       // [slabs][row blocks * BM, hs]
  float* dbp;                        // [row halves, piece]
  int piece, v0;                     // columns of the piece, its first column
  int hs;                            // columns of a slab row
};

// ------------------------------------------------------------------------------------------------------------------------------------
// rows
// ------------------------------------------------------------------------------------------------------------------------------------
// One wave per row: q = softmax(t / T) over the entries whose index lies in the vocabulary; an index that occurs again adds its weight
// to its first place.  A row without entries gets none (all indices -1).
__global__ __launch_bounds__(256) void targets_kernel(LossArgs a) {
  __shared__ int s_idx[4][128];
  __shared__ float s_q[4][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= a.rows) return;      // a wave keeps to its own part of the LDS: no barrier follows
  int idx[2];
  float t[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k = h * 64 + lane;
    idx[h] = -1;
    t[h] = -INFINITY;
    if (k < a.topk) {
      const int64_t i = a.idx64 ? reinterpret_cast<const int64_t*>(a.teacher_idx)[row * a.ld_i + k]
                                : (int64_t)reinterpret_cast<const int*>(a.teacher_idx)[row * a.ld_i + k];
      const float v = a.teacher[row * a.ld_t + k];
      if (i >= 0 && i < a.vocab && v != -INFINITY) {      // a logit of -inf is no entry
        idx[h] = (int)i;
        t[h] = v * a.inv_t;
      }
    }
  }
  // fmaxf drops a NaN; it comes back through the exponentials below
  const float m = wave_max(fmaxf(t[0], t[1]));
  const bool some = __ballot(idx[0] >= 0 || idx[1] >= 0) != 0;
  float e[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) e[h] = idx[h] < 0 ? 0.f : __builtin_amdgcn_exp2f((t[h] - m) * LOG2E);
  const float sum = wave_sum(e[0] + e[1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    s_idx[wave][h * 64 + lane] = idx[h];
    s_q[wave][h * 64 + lane] = idx[h] < 0 ? 0.f : e[h] / sum;
  }
  CACO_WAVE_LDS_SYNC();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k = h * 64 + lane;
    float q = 0.f;
    int out = idx[h];
    if (out >= 0)
      for (int o = 0; o < a.topk; ++o)
        if (s_idx[wave][o] == out) {
          if (o < k) { out = -1; break; }
          q += s_q[wave][o];
        }
    if (k < a.kp) {
      a.tgt_idx0[row * a.kp + k] = out;
      a.tgt_q0[row * a.kp + k] = out < 0 ? 0.f : q;
    }
  }
  if (lane == 0) a.inv[row] = some;                        // for `compact`
}

// does row r count?
__device__ __forceinline__ bool row_counts(const LossArgs& a, int64_t r) {
  if (a.labels) {
    const int64_t y = a.labels[r];
    return y != a.ignore_index && y >= 0 && y < a.vocab;
  }
  return a.inv[r] != 0;
}

// One workgroup: every thread counts a run of consecutive rows, a scan over the threads gives each run its first place.
__global__ __launch_bounds__(1024) void compact_kernel(LossArgs a) {
  __shared__ int s_wave[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t per = (a.rows + 1023) / 1024;
  const int64_t r0 = min(a.rows, tid * per), r1 = min(a.rows, r0 + per);
  int n = 0;
  for (int64_t r = r0; r < r1; ++r) n += row_counts(a, r);
  int incl = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl(incl, max(lane - o, 0), 64);
    if (lane >= o) incl += v;
  }
  if (lane == 63) s_wave[wave] = incl;
  __syncthreads();
  int at = incl - n;
  for (int w = 0; w < wave; ++w) at += s_wave[w];
  for (int64_t r = r0; r < r1; ++r) {
    const bool c = row_counts(a, r);      // this thread's own rows: read before they are overwritten
    a.inv[r] = c ? at : -1;
    if (c) a.rowmap[at++] = (int)r;
  }
  if (tid == 1023) *a.count = at;
}

// compact row <- its hidden state, targets, gradient scale.  One wave per row; rows up to the next multiple of 256 are zero rows.
__global__ __launch_bounds__(256) void gather_kernel(LossArgs a, int backward, int from_lse) {
  const int lane = threadIdx.x & 63;
  const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int n = *a.count;
  if (c >= ((int64_t)n + 255) / 256 * 256) return;
  const bool real = c < n;
  const int64_t row = real ? a.rowmap[c] : 0;
  const bf16x8* src = reinterpret_cast<const bf16x8*>(a.hidden + row * a.ld_h);
  bf16x8* dst = reinterpret_cast<bf16x8*>(a.hc + c * a.hp);
  for (int i = lane; i < a.hp / 8; i += 64) dst[i] = real && i < a.dim / 8 ? src[i] : bf16x8{};
  for (int k = lane; k < a.kp; k += 64) {
    int idx = -1;
    float q = 0.f;
    if (real) {
      idx = a.labels ? (int)a.labels[row] : a.tgt_idx0[row * a.kp + k];
      q = a.labels ? 1.f : a.tgt_q0[row * a.kp + k];
    }
    a.tgt_idx[c * a.kp + k] = idx;
    a.tgt_q[c * a.kp + k] = q;
  }
  if (backward && lane == 0) {
    float g = real ? a.temperature : 0.f;
    if (real && a.row_weight) g *= a.row_weight[row];
    if (real && a.grad_scale) g *= *a.grad_scale;
    if (real && a.reduction == CACO_REDUCE_MEAN) g /= (float)n;
    a.g[c] = g;
    if (from_lse) a.lse2[c] = real ? a.lse[row] * LOG2E : 0.f;
  }
}

// (distillation) sum_k q_k (log q_k - z_k / T) of a compact row: 16 lanes per entry, the entries' rows of weight gathered.
// Also in log2 units, so that `finish` treats both losses alike.
__global__ __launch_bounds__(256) void target_logits_kernel(LossArgs a) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, grp = lane >> 4;
  const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (c >= *a.count) return;
  const bf16_t* h = a.hc + c * a.hp;
  float sum = 0.f;
  for (int k0 = 0; k0 < a.kp; k0 += 4) {
    const int k = k0 + grp;
    const int idx = k < a.kp ? a.tgt_idx[c * a.kp + k] : -1;
    const float q = k < a.kp ? a.tgt_q[c * a.kp + k] : 0.f;
    float z = 0.f;
    if (idx >= 0) {
      const bf16_t* w = a.weight + (int64_t)idx * a.ld_w;
      for (int i = l16 * 8; i < a.dim; i += 128) {
        const bf16x8 x = *reinterpret_cast<const bf16x8*>(h + i), y = *reinterpret_cast<const bf16x8*>(w + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) z = __builtin_fmaf((float)x[e], (float)y[e], z);
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
    if (q != 0.f && l16 == 0) {      // 0 log 0 = 0: an entry of weight 0 (or none) adds nothing, whatever its logit is
      if (a.bias) z += a.bias[idx];
      sum += q * (log2f(q) - z * a.inv_t * LOG2E);
    }
  }
  sum = wave_sum(sum);
  if (lane == 0) a.zt[c] = -sum;
}

// ------------------------------------------------------------------------------------------------------------------------------------
// logits -> running maximum and sum
// ------------------------------------------------------------------------------------------------------------------------------------
// Units (row block, slice of the vocabulary's tiles).  Consecutive units go to one XCD, slices of a row block next to one another:
// an XCD's L2 holds the few row blocks its workgroups share while their slices of the weights stream through it.
struct LseUnits {
  int rb, tiles, slices, units;
  __device__ __forceinline__ LseUnits(int n, int vocab, int bm, int bn, int wgs) {
    rb = (n + bm - 1) / bm;
    tiles = (vocab + bn - 1) / bn;
    slices = rb > 0 ? max(1, min(tiles, wgs / rb)) : 1;
    units = rb * slices;
  }
};

template <typename C>
__device__ __forceinline__ void lse_body(const LossArgs& a, char* smem) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int n = *a.count;
  const LseUnits U(n, a.vocab, C::BM, C::BN, gridDim.x);
  const int wg = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const float cs = a.inv_t * LOG2E;
  const bool label = a.labels != nullptr;
  for (int u = wg; u < U.units; u += gridDim.x) {
    const int rb = u / U.slices, sl = u % U.slices;
    const int t0 = (int)((int64_t)sl * U.tiles / U.slices), t1 = (int)((int64_t)(sl + 1) * U.tiles / U.slices);
    const int64_t m0 = (int64_t)rb * C::BM;
    float mx[C::MI], sm[C::MI];
    int y[C::MI];
#pragma unroll
    for (int i = 0; i < C::MI; ++i) {
      mx[i] = -3.0e38f;            // finite: exp2(-inf - mx) = 0 for logits of -inf
      sm[i] = 0.f;
      y[i] = label ? a.tgt_idx[m0 + (wm * C::MI + i) * 16 + l16] : -1;
    }
    vg_run<C, false, false>(
        t1 - t0, smem,
        [&](int i, VgOperand& X, VgOperand& W, int& k0, int& k1) {
          const int n0 = (t0 + i) * C::BN;
          X = VgOperand{a.hc + m0 * a.hp, a.hp, C::BM, a.hp};
          W = VgOperand{a.weight + (int64_t)n0 * a.ld_w, a.ld_w, a.vocab - n0, a.dim};
          k0 = 0;
          k1 = a.hp / VG_K;
        },
        [&](int i, f32x4 (&acc)[C::MI][C::NI]) {
          const int n0 = (t0 + i) * C::BN + wn * 16 * C::NI + lq * 4;      // this lane's columns: n0 + j * 16 + e
          float b2[C::NI][4];
#pragma unroll
          for (int j = 0; j < C::NI; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int v = n0 + j * 16 + e;
              b2[j][e] = v < a.vocab ? (a.bias ? a.bias[v] * cs : 0.f) : -INFINITY;
            }
#pragma unroll
          for (int q = 0; q < C::MI; ++q) {
            float z[C::NI][4];
            float m = mx[q];
#pragma unroll
            for (int j = 0; j < C::NI; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                z[j][e] = b2[j][e] == -INFINITY ? -INFINITY : __builtin_fmaf(acc[q][j][e], cs, b2[j][e]);
                m = fmaxf(m, z[j][e]);
              }
            float s = sm[q] * __builtin_amdgcn_exp2f(mx[q] - m);
#pragma unroll
            for (int j = 0; j < C::NI; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f(z[j][e] - m);
            mx[q] = m;
            sm[q] = s;
            const int d = y[q] - n0;                       // the label's place among this lane's columns
            if ((unsigned)d < 16u * C::NI && (d & 12) == 0) {
              float zy = 0.f;
#pragma unroll
              for (int j = 0; j < C::NI; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (d == j * 16 + e) zy = z[j][e];
              a.zt[m0 + (wm * C::MI + q) * 16 + l16] = zy;
            }
          }
        });
    // the four lanes of a row, then the waves that share it
    float2* red = reinterpret_cast<float2*>(vg_slab<C>(smem, 0));      // [WN][BM]
    static_assert(C::WN * C::BM * 8 <= C::WAVES * C::SLAB, "the joint of the waves fits the slabs");
#pragma unroll
    for (int q = 0; q < C::MI; ++q) {
      float m = mx[q], s = sm[q];
#pragma unroll
      for (int o = 16; o <= 32; o <<= 1) {
        const float om = __shfl_xor(m, o, 64), os = __shfl_xor(s, o, 64);
        const float nm = fmaxf(m, om);
        s = s * __builtin_amdgcn_exp2f(m - nm) + os * __builtin_amdgcn_exp2f(om - nm);
        m = nm;
      }
      if (lq == 0) red[wn * C::BM + (wm * C::MI + q) * 16 + l16] = make_float2(m, s);
    }
    __syncthreads();
    for (int r = threadIdx.x; r < C::BM; r += C::THREADS) {
      float m = red[r].x, s = red[r].y;
#pragma unroll
      for (int w = 1; w < C::WN; ++w) {
        const float2 o = red[w * C::BM + r];
        const float nm = fmaxf(m, o.x);
        s = s * __builtin_amdgcn_exp2f(m - nm) + o.y * __builtin_amdgcn_exp2f(o.x - nm);
        m = nm;
      }
      a.part[(int64_t)sl * U.rb * C::BM + m0 + r] = make_float2(m, s);
    }
    __syncthreads();               // the next unit's run fills the stages, its joint the slabs
  }
}
template <typename C>
__global__ __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) void lse_kernel(LossArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  lse_body<C>(a, smem);
}

// One wave per row of the caller: joins the slices, row loss and lse; rows that do not count get zeros.
__global__ __launch_bounds__(256) void finish_kernel(LossArgs a, int bm, int bn, int wgs) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const int c = a.inv[row];
  if (c < 0) {
    if (lane == 0) {
      if (a.row_loss) a.row_loss[row] = 0.f;
      if (a.lse) a.lse[row] = 0.f;
    }
    return;
  }
  const LseUnits U(*a.count, a.vocab, bm, bn, wgs);
  float m = -3.0e38f, s = 0.f;
  for (int sl = lane; sl < U.slices; sl += 64) {
    const float2 o = a.part[(int64_t)sl * U.rb * bm + c];
    const float nm = fmaxf(m, o.x);
    s = s * __builtin_amdgcn_exp2f(m - nm) + o.y * __builtin_amdgcn_exp2f(o.x - nm);
    m = nm;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float om = __shfl_xor(m, o, 64), os = __shfl_xor(s, o, 64);
    const float nm = fmaxf(m, om);
    s = s * __builtin_amdgcn_exp2f(m - nm) + os * __builtin_amdgcn_exp2f(om - nm);
    m = nm;
  }
  if (lane == 0) {
    const float l2 = m + log2f(s);
    if (a.lse2) a.lse2[c] = l2;
    if (a.lse) a.lse[row] = l2 * LN2;
    if (a.row_loss) a.row_loss[row] = (l2 - a.zt[c]) * LN2 * a.temperature * a.temperature;
  }
}

// One workgroup, fixed order: sum or mean of the (weighted) row losses.
__global__ __launch_bounds__(1024) void reduce_kernel(LossArgs a) {
  __shared__ double s_wave[16];
  const int tid = threadIdx.x;
  double s = 0.;
  for (int64_t r = tid; r < a.rows; r += 1024)
    if (a.inv[r] >= 0) s += a.row_weight ? (double)a.row_loss[r] * a.row_weight[r] : (double)a.row_loss[r];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((tid & 63) == 0) s_wave[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    double t = 0.;
    for (int w = 0; w < 16; ++w) t += s_wave[w];
    *a.loss = (float)(a.reduction == CACO_REDUCE_MEAN ? t / (double)*a.count : t);      // no row counts: 0 / 0, as torch has it
  }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// gradients
// ------------------------------------------------------------------------------------------------------------------------------------
// Tile order of a piece: an XCD takes a run of consecutive tiles; blocks of 8 row blocks, inside them the vocabulary's tiles, row blocks
// fastest: 8 panels of hidden states stay in the XCD's L2 and a panel of weights is used 8 times while it is there.
struct Order2 {
  int a, b, units, q, r;
  __device__ __forceinline__ Order2(int a_, int b_) : a(a_), b(b_), units(a_ * b_), q(units >> 3), r(units & 7) {}
  __device__ __forceinline__ int count(int xcd) const { return q + (xcd < r ? 1 : 0); }
  __device__ __forceinline__ int first(int xcd) const { return xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q; }
  __device__ __forceinline__ void at(int t, int& ia, int& ib) const {
    const int per = 8 * b, grp = t / per, a0 = grp * 8, wdt = min(8, a - a0), rem = t - grp * per;
    ia = a0 + rem % wdt;
    ib = rem / wdt;
  }
};

template <typename C>
__device__ __forceinline__ void dlogits_body(const LossArgs& a, char* smem) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int n = *a.count;
  const Order2 O((n + C::BM - 1) / C::BM, a.piece / C::BN);
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3, slots = gridDim.x >> 3;
  const int cnt = O.count(xcd), base = O.first(xcd);
  if (slot >= cnt) return;
  const float cs = a.inv_t * LOG2E;
  const int lkp = 31 - __builtin_clz((unsigned)a.kp);
  float* slab = vg_slab<C>(smem, wave);
  vg_run<C, false, false>(
      (cnt - slot + slots - 1) / slots, smem,
      [&](int i, VgOperand& X, VgOperand& W, int& k0, int& k1) {
        int tm, tn;
        O.at(base + slot + i * slots, tm, tn);
        const int n0 = a.v0 + tn * C::BN;
        X = VgOperand{a.hc + (int64_t)tm * C::BM * a.hp, a.hp, C::BM, a.hp};
        W = VgOperand{a.weight + (int64_t)min(n0, a.vocab - 1) * a.ld_w, a.ld_w, max(1, a.vocab - n0), a.dim};
        k0 = 0;
        k1 = a.hp / VG_K;
      },
      [&](int i, f32x4 (&acc)[C::MI][C::NI]) {
        int tm, tn;
        O.at(base + slot + i * slots, tm, tn);
        const int64_t m0 = (int64_t)tm * C::BM + wm * 16 * C::MI;
        const int c0 = tn * C::BN + wn * 16 * C::NI;                  // the wave's first column in the piece
        const int v0 = a.v0 + c0;
        float b2[C::NI][4];
#pragma unroll
        for (int j = 0; j < C::NI; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int v = v0 + j * 16 + lq * 4 + e;
            b2[j][e] = v < a.vocab && a.bias ? a.bias[v] * cs : 0.f;
          }
        constexpr int LPR = C::SLAB_COLS / 8, RPP = 64 / LPR;         // lanes per row on the way out, rows per pass
        float col[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) col[e] = 0.f;
#pragma unroll
        for (int q = 0; q < C::MI; ++q) {
          const int64_t r0 = m0 + q * 16;
          const float lse2 = r0 + l16 < n ? a.lse2[r0 + l16] : 0.f, g = r0 + l16 < n ? a.g[r0 + l16] : 0.f;
#pragma unroll
          for (int j = 0; j < C::NI; ++j) {
            f32x4 p;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = g * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[q][j][e], cs, b2[j][e]) - lse2);
              p[e] = g != 0.f && v0 + j * 16 + lq * 4 + e < a.vocab ? x : 0.f;      // a row of weight 0 has no gradient, whatever its logits are
            }
            *reinterpret_cast<f32x4*>(slab + vg_slab_at<C>(l16, j * 4 + lq)) = p;
          }
          CACO_WAVE_LDS_SYNC();
          // the targets of these 16 rows that fall into the wave's columns (indices of one row are distinct)
          for (int t = lane; t < 16 << lkp; t += 64) {
            const int64_t r = r0 + (t >> lkp);
            const int c = a.tgt_idx[(r0 << lkp) + t] - v0;
            if ((unsigned)c < (unsigned)C::SLAB_COLS && r < n) {
              const float gr = a.g[r];
              if (gr != 0.f) slab[vg_slab_at<C>(t >> lkp, c >> 2) + (c & 3)] -= gr * a.tgt_q[(r0 << lkp) + t];
            }
          }
          CACO_WAVE_LDS_SYNC();
#pragma unroll
          for (int ps = 0; ps < 16 / RPP; ++ps) {
            const int row = ps * RPP + lane / LPR, ch = (lane % LPR) * 2;
            const f32x4 u = *reinterpret_cast<const f32x4*>(slab + vg_slab_at<C>(row, ch)), v = *reinterpret_cast<const f32x4*>(slab + vg_slab_at<C>(row, ch + 1));
            bf16x8 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[e] = (bf16_t)u[e];
              o[e + 4] = (bf16_t)v[e];
              col[e] += u[e];
              col[e + 4] += v[e];
            }
            *reinterpret_cast<bf16x8*>(a.dl + (r0 + row) * a.piece + c0 + ch * 4) = o;
          }
          CACO_WAVE_LDS_SYNC();
        }
        if (a.db) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int o = LPR; o < 64; o <<= 1) col[e] += __shfl_xor(col[e], o, 64);
          if (lane < LPR) {
            float* d = a.dbp + ((int64_t)tm * C::WM + wm) * a.piece + c0 + lane * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = col[e];
          }
        }
      });
}
template <typename C>
__global__ __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) void dlogits_kernel(LossArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  dlogits_body<C>(a, smem);
}

__global__ __launch_bounds__(256) void dbias_kernel(LossArgs a, int bm, int wm) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.piece || a.v0 + c >= a.vocab) return;
  const int parts = (*a.count + bm - 1) / bm * wm;
  float s = 0.f;
  for (int p = 0; p < parts; ++p) s += a.dbp[(int64_t)p * a.piece + c];
  a.db[a.v0 + c] = s;
}

// d hidden of the piece: (row block, column block, slab) units, the piece's K-tiles split evenly over the slabs
struct DhUnits {
  int rb, cb, slabs, units;
  __device__ __forceinline__ DhUnits(int n, int dim, int piece, int bm, int bn) {
    rb = (n + bm - 1) / bm;
    cb = (dim + bn - 1) / bn;
    slabs = rb > 0 ? max(1, min(piece / VG_K, DH_UNITS / (rb * cb))) : 1;
    units = rb * cb * slabs;
  }
};
template <typename C>
__device__ __forceinline__ void dhidden_body(const LossArgs& a, int first_piece, int full_piece, char* smem) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int n = *a.count;
  const DhUnits U(n, a.dim, full_piece, C::BM, C::BN);
  const int wg = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (wg >= U.units) return;
  const int nk = a.piece / VG_K;
  vg_run<C, false, true>(
      (U.units - wg + gridDim.x - 1) / gridDim.x, smem,
      [&](int i, VgOperand& X, VgOperand& W, int& k0, int& k1) {
        const int u = wg + i * gridDim.x, cb = u % U.cb, rest = u / U.cb, rb = rest % U.rb, s = rest / U.rb;
        k0 = (int)((int64_t)s * nk / U.slabs);
        k1 = (int)((int64_t)(s + 1) * nk / U.slabs);
        X = VgOperand{a.dl + (int64_t)rb * C::BM * a.piece, a.piece, C::BM, a.piece};
        W = VgOperand{a.weight + (int64_t)a.v0 * a.ld_w + cb * C::BN, a.ld_w, a.dim - cb * C::BN, a.vocab - a.v0};
      },
      [&](int i, f32x4 (&acc)[C::MI][C::NI]) {
        const int u = wg + i * gridDim.x, cb = u % U.cb, rest = u / U.cb, rb = rest % U.rb, s = rest / U.rb;
        const int64_t m0 = (int64_t)rb * C::BM + wm * 16 * C::MI + l16;
        const int c0 = cb * C::BN + wn * 16 * C::NI + lq * 4;
#pragma unroll
        for (int q = 0; q < C::MI; ++q) {
          if (m0 + q * 16 >= n) continue;
          float* d = a.slab + ((int64_t)s * U.rb * C::BM + m0 + q * 16) * a.hs + c0;
#pragma unroll
          for (int j = 0; j < C::NI; ++j) {
            if (c0 + j * 16 >= a.dim) continue;
            f32x4 v = acc[q][j];
            f32x4* p = reinterpret_cast<f32x4*>(d + j * 16);
            if (!first_piece) v += *p;
            *p = v;
          }
        }
      });
}
template <typename C>
__global__ __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) void dhidden_kernel(LossArgs a, int first_piece, int full_piece) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  dhidden_body<C>(a, first_piece, full_piece, smem);
}

// rows of d hidden in the caller's order: the slabs added in order and rounded once; zeros for rows that do not count
__global__ __launch_bounds__(256) void dh_join_kernel(LossArgs a, int full_piece, int bm, int bn) {
  const int64_t row = blockIdx.x;
  const int c = a.inv[row];
  const DhUnits U(*a.count, a.dim, full_piece, bm, bn);
  for (int x = threadIdx.x * 8; x < a.dim; x += 2048) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c >= 0)
      for (int s = 0; s < U.slabs; ++s) {
        const float* p = a.slab + ((int64_t)s * U.rb * bm + c) * a.hs + x;
        const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] += lo[e]; v[e + 4] += hi[e]; }
      }
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (bf16_t)v[e];
    *reinterpret_cast<bf16x8*>(a.dh + row * a.ld_dh + x) = o;
  }
}

// the piece's rows of d weight: sums over the tokens, both operands with the token slowest
__device__ __forceinline__ void dweight_body(const LossArgs& a, char* smem) {
  typedef Big C;
  const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int n = *a.count, nk = (n + VG_K - 1) / VG_K;
  const int cbs = (a.dim + C::BN - 1) / C::BN;
  const Order2 O(cbs, min(a.piece, (a.vocab - a.v0 + 255) / 256 * 256) / C::BM);
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3, slots = gridDim.x >> 3;
  const int cnt = O.count(xcd), base = O.first(xcd);
  if (slot >= cnt) return;
  float* slab = vg_slab<C>(smem, wave);
  vg_run<C, true, true>(
      (cnt - slot + slots - 1) / slots, smem,
      [&](int i, VgOperand& X, VgOperand& W, int& k0, int& k1) {
        int tn, tm;
        O.at(base + slot + i * slots, tn, tm);
        X = VgOperand{a.dl + tm * C::BM, a.piece, C::BM, (int64_t)nk * VG_K};
        W = VgOperand{a.hc + tn * C::BN, a.hp, a.hp - tn * C::BN, (int64_t)nk * VG_K};
        k0 = 0;
        k1 = nk;
      },
      [&](int i, f32x4 (&acc)[C::MI][C::NI]) {
        int tn, tm;
        O.at(base + slot + i * slots, tn, tm);
        const int v0 = a.v0 + tm * C::BM + wm * 16 * C::MI;
        const int c0 = tn * C::BN + wn * 16 * C::NI;
        constexpr int LPR = C::SLAB_COLS / 8, RPP = 64 / LPR;
#pragma unroll
        for (int q = 0; q < C::MI; ++q) {
#pragma unroll
          for (int j = 0; j < C::NI; ++j) *reinterpret_cast<f32x4*>(slab + vg_slab_at<C>(l16, j * 4 + lq)) = acc[q][j];
          CACO_WAVE_LDS_SYNC();
#pragma unroll
          for (int ps = 0; ps < 16 / RPP; ++ps) {
            const int row = ps * RPP + lane / LPR, ch = (lane % LPR) * 2;
            const f32x4 u = *reinterpret_cast<const f32x4*>(slab + vg_slab_at<C>(row, ch)), v = *reinterpret_cast<const f32x4*>(slab + vg_slab_at<C>(row, ch + 1));
            bf16x8 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) { o[e] = (bf16_t)u[e]; o[e + 4] = (bf16_t)v[e]; }
            const int vv = v0 + q * 16 + row, cc = c0 + ch * 4;
            if (vv < a.vocab && cc < a.dim) *reinterpret_cast<bf16x8*>(a.dw + (int64_t)vv * a.ld_dw + cc) = o;
          }
          CACO_WAVE_LDS_SYNC();
        }
      });
}
__global__ __launch_bounds__(Big::THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) void dweight_kernel(LossArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  dweight_body(a, smem);
}

// ------------------------------------------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------------------------------------------
int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// Where everything lies in the workspace.  Sizes are for all `rows`; how many of them count is known on the device only.
struct Plan {
  int64_t npad, bytes = 0;
  int hp, hs, kp;
  int64_t piece;
  bool small;
  int64_t o_count, o_rowmap, o_inv, o_ti0, o_tq0, o_ti, o_tq, o_hc, o_part, o_zt, o_lse2, o_g, o_dl, o_slab, o_dbp;
  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += up(n, 256);
    return at;
  }
  // piece_cols 0: losses alone
  Plan(int64_t rows, int vocab, int dim, int topk, int64_t piece_cols) {
    npad = up(rows > 0 ? rows : 1, 256);
    hp = (int)up(dim, VG_K);
    hs = (int)up(dim, 4);
    kp = 1;
    while (kp < topk) kp *= 2;
    small = rows <= Small::BM;
    const int bm = small ? Small::BM : Big::BM, bn = small ? Small::BN : Big::BN;
    o_count = take(4);
    o_rowmap = take(npad * 4);
    o_inv = take(npad * 4);
    o_ti0 = topk ? take(npad * kp * 4) : 0;
    o_tq0 = topk ? take(npad * kp * 4) : 0;
    o_ti = take(npad * kp * 4);
    o_tq = take(npad * kp * 4);
    o_hc = take(npad * hp * 2);
    o_part = take((npad + (int64_t)MAX_WG * bm) * 8);          // slices * row blocks <= max(row blocks, workgroups)
    o_zt = take(npad * 4);
    o_lse2 = take(npad * 4);
    o_g = take(npad * 4);
    piece = piece_cols;
    o_dl = o_slab = o_dbp = 0;
    if (piece) {
      o_dl = take(npad * piece * 2);
      const int64_t tiles = up(npad, bm) / bm * ((dim + bn - 1) / bn);
      // slabs * row blocks * BM rows of hs columns; slabs * row blocks * column blocks <= max(DH_UNITS, tiles)
      o_slab = take((tiles > DH_UNITS ? tiles : DH_UNITS) / ((dim + bn - 1) / bn) * bm * hs * 4);
      o_dbp = take(npad / bm * (small ? Small::WM : Big::WM) * piece * 4);
    }
  }
};

// columns of a piece: the vocabulary in as few equal pieces as d logits of `budget` bytes allow, in whole tiles
int64_t piece_for(int64_t rows, int vocab, int64_t budget) {
  const int64_t npad = up(rows > 0 ? rows : 1, 256), all = up(vocab, 256);
  int64_t most = budget / (npad * 2) / 256 * 256;
  if (most < 256) most = 256;
  const int64_t pieces = (all + most - 1) / most;
  return up((all + pieces - 1) / pieces, 256);
}

template <typename K, typename... A>
int launch(const char* what, K kern, dim3 grid, int threads, int lds, hipStream_t st, A... args) {
  int num_cu = 0;
  if (lds) CACO_TRY_RC(prepare_launch(reinterpret_cast<const void*>(kern), lds, &num_cu));
  hipLaunchKernelGGL(kern, grid, dim3(threads), lds, st, args...);
  return check_hip(hipGetLastError(), what);
}

template <typename C>
int run_loss(LossArgs& a, const Plan& P, int what, int wgs, hipStream_t st) {
  const dim3 rows4((unsigned)((a.rows + 3) / 4));
  const dim3 pad4((unsigned)(P.npad / 4));
  if (a.topk && a.rows) CACO_TRY_RC(launch("loss targets", targets_kernel, rows4, 256, 0, st, a));
  CACO_TRY_RC(launch("loss compact", compact_kernel, dim3(1), 1024, 0, st, a));
  CACO_TRY_RC(launch("loss gather", gather_kernel, pad4, 256, 0, st, a, (what & CACO_LOSS_BACKWARD) != 0, (what & CACO_LOSS_FORWARD) == 0));
  if (what & CACO_LOSS_FORWARD) {
    if (a.topk) CACO_TRY_RC(launch("loss target logits", target_logits_kernel, pad4, 256, 0, st, a));
    CACO_TRY_RC(launch("loss lse", lse_kernel<C>, dim3(wgs), C::THREADS, C::SMEM, st, a));
    if (a.rows) CACO_TRY_RC(launch("loss finish", finish_kernel, rows4, 256, 0, st, a, (int)C::BM, (int)C::BN, wgs));
    if (a.loss) CACO_TRY_RC(launch("loss reduce", reduce_kernel, dim3(1), 1024, 0, st, a));
  }
  if (!(what & CACO_LOSS_BACKWARD)) return CACO_OK;
  const int full = a.piece;
  int num_cu = 0;
  CACO_TRY_RC(prepare_launch(reinterpret_cast<const void*>(&dweight_kernel), Big::SMEM, &num_cu));
  for (int v0 = 0; v0 < a.vocab; v0 += full) {
    a.v0 = v0;
    CACO_TRY_RC(launch("loss dlogits", dlogits_kernel<C>, dim3(wgs), C::THREADS, C::SMEM, st, a));
    if (a.db) CACO_TRY_RC(launch("loss dbias", dbias_kernel, dim3((a.piece + 255) / 256), 256, 0, st, a, (int)C::BM, (int)C::WM));
    if (a.dh) CACO_TRY_RC(launch("loss dhidden", dhidden_kernel<C>, dim3(wgs), C::THREADS, C::SMEM, st, a, v0 == 0, full));
    if (a.dw) CACO_TRY_RC(launch("loss dweight", dweight_kernel, dim3(num_cu / 8 * 8), Big::THREADS, Big::SMEM, st, a));
  }
  if (a.dh && a.rows) CACO_TRY_RC(launch("loss dhidden join", dh_join_kernel, dim3((unsigned)a.rows), 256, 0, st, a, full, (int)C::BM, (int)C::BN));
  return CACO_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_sizes(int64_t rows, int32_t vocab, int32_t dim, int32_t topk) {
  CACO_REQUIRE(rows >= 0 && rows <= (int64_t)1 << 24, "linear loss: rows must be 0 .. 2^24, got %lld", (long long)rows);
  CACO_REQUIRE(vocab >= 1 && vocab <= 1 << 24, "linear loss: vocab must be 1 .. 2^24, got %d", vocab);
  CACO_REQUIRE(dim >= 8 && dim <= 1 << 16 && dim % 8 == 0, "linear loss: dim must be a multiple of 8 in 8 .. 65536, got %d", dim);
  CACO_REQUIRE(topk >= 0 && topk <= 128, "linear loss: topk must be 1 .. 128, got %d", topk);
  return CACO_OK;
}

}  // namespace

int64_t linear_loss_workspace(int64_t rows, int32_t vocab, int32_t dim, int32_t topk, int64_t piece_bytes, int32_t what) {
  if (check_sizes(rows, vocab, dim, topk) != CACO_OK) return CACO_ERR_INVALID;
  return Plan(rows, vocab, dim, topk, what & CACO_LOSS_BACKWARD ? piece_for(rows, vocab, piece_bytes) : 0).bytes;
}

int linear_loss(const LinearLoss& c, hipStream_t st) {
  CACO_TRY_RC(check_sizes(c.rows, c.vocab, c.dim, c.topk));
  CACO_REQUIRE(c.what >= 1 && c.what <= 3, "linear loss: `what` must be CACO_LOSS_FORWARD, CACO_LOSS_BACKWARD or both");
  CACO_REQUIRE(c.reduction >= CACO_REDUCE_NONE && c.reduction <= CACO_REDUCE_SUM, "linear loss: unknown reduction %d", c.reduction);
  CACO_REQUIRE(c.weight && c.ws && (c.rows == 0 || (c.hidden && (c.topk ? c.teacher && c.teacher_idx : c.labels != nullptr))), "linear loss: null argument");
  CACO_REQUIRE(c.topk == 0 || (c.temperature > 0.f && c.temperature < INFINITY), "linear loss: temperature must be positive and finite");
  const bool fwd = c.what & CACO_LOSS_FORWARD, bwd = c.what & CACO_LOSS_BACKWARD;
  CACO_REQUIRE(!fwd || c.rows == 0 || c.row_loss, "linear loss: the forward pass needs row_loss");
  CACO_REQUIRE(!c.loss || (fwd && c.reduction != CACO_REDUCE_NONE), "linear loss: a reduced loss needs the forward pass and a reduction");
  CACO_REQUIRE(fwd || c.rows == 0 || c.lse, "linear loss: the backward pass alone needs the forward pass's lse");
  CACO_REQUIRE(!bwd || c.d_hidden || c.d_weight || c.d_bias, "linear loss: the backward pass has no output");
  CACO_REQUIRE(c.ld_h >= c.dim && c.ld_h % 8 == 0 && c.ld_w >= c.dim && c.ld_w % 8 == 0 && c.ld_w < 1 << 22 && aligned16(c.hidden) && aligned16(c.weight),
               "linear loss: rows of hidden and weight must start at multiples of 16 bytes (strides >= dim, multiples of 8)");
  CACO_REQUIRE(!bwd || ((!c.d_hidden || (c.ld_dh >= c.dim && c.ld_dh % 8 == 0 && aligned16(c.d_hidden))) &&
                        (!c.d_weight || (c.ld_dw >= c.dim && c.ld_dw % 8 == 0 && aligned16(c.d_weight)))),
               "linear loss: rows of d_hidden and d_weight must start at multiples of 16 bytes (strides >= dim, multiples of 8)");
  CACO_REQUIRE(c.topk == 0 || (c.ld_t >= c.topk && c.ld_i >= c.topk), "linear loss: teacher strides must be >= topk");
  CACO_REQUIRE(aligned16(c.ws), "linear loss: the workspace must be 16-byte aligned");
  // as large a piece as the workspace holds
  int64_t piece = 0;
  if (bwd) {
    const int64_t all = up(c.vocab, 256);
    int64_t lo = 1, hi = all / 256;                      // in tiles; the plan's size grows with the piece
    CACO_REQUIRE(Plan(c.rows, c.vocab, c.dim, c.topk, 256).bytes <= c.ws_bytes, "linear loss: the workspace is too small (caco_linear_loss_workspace)");
    while (lo < hi) {
      const int64_t mid = (lo + hi + 1) / 2;
      if (Plan(c.rows, c.vocab, c.dim, c.topk, mid * 256).bytes <= c.ws_bytes) lo = mid; else hi = mid - 1;
    }
    const int64_t pieces = (all + lo * 256 - 1) / (lo * 256);
    piece = up((all + pieces - 1) / pieces, 256);
  }
  const Plan P(c.rows, c.vocab, c.dim, c.topk, piece);
  CACO_REQUIRE(P.bytes <= c.ws_bytes, "linear loss: the workspace is too small (caco_linear_loss_workspace)");
  LossArgs a{};
  a.hidden = c.hidden; a.ld_h = c.ld_h; a.weight = c.weight; a.ld_w = c.ld_w; a.bias = c.bias;
  a.labels = c.topk ? nullptr : c.labels; a.ignore_index = c.ignore_index;
  if (!c.topk && !c.labels) a.labels = reinterpret_cast<const int64_t*>(c.ws);      // no rows: never read, but it marks the loss
  a.teacher = c.teacher; a.ld_t = c.ld_t; a.teacher_idx = c.teacher_idx; a.ld_i = c.ld_i; a.idx64 = c.idx64;
  a.topk = c.topk; a.kp = P.kp;
  a.temperature = c.topk ? c.temperature : 1.f;
  a.inv_t = 1.f / a.temperature;
  a.rows = c.rows; a.vocab = c.vocab; a.dim = c.dim; a.hp = P.hp; a.hs = P.hs;
  a.reduction = c.reduction; a.row_weight = c.row_weight; a.grad_scale = c.grad_scale;
  a.row_loss = c.row_loss; a.lse = c.lse; a.loss = c.loss;
  a.dh = bwd ? c.d_hidden : nullptr; a.ld_dh = c.ld_dh; a.dw = bwd ? c.d_weight : nullptr; a.ld_dw = c.ld_dw; a.db = bwd ? c.d_bias : nullptr;
  char* w = reinterpret_cast<char*>(c.ws);
  a.count = (int*)(w + P.o_count); a.rowmap = (int*)(w + P.o_rowmap); a.inv = (int*)(w + P.o_inv);
  a.tgt_idx0 = (int*)(w + P.o_ti0); a.tgt_q0 = (float*)(w + P.o_tq0); a.tgt_idx = (int*)(w + P.o_ti); a.tgt_q = (float*)(w + P.o_tq);
  a.hc = (bf16_t*)(w + P.o_hc); a.part = (float2*)(w + P.o_part); a.zt = (float*)(w + P.o_zt); a.lse2 = (float*)(w + P.o_lse2); a.g = (float*)(w + P.o_g);
  a.dl = (bf16_t*)(w + P.o_dl); a.slab = (float*)(w + P.o_slab); a.dbp = (float*)(w + P.o_dbp);
  a.piece = (int)piece;
  int num_cu = 0;
  CACO_TRY_RC(prepare_launch(reinterpret_cast<const void*>(&lse_kernel<Big>), Big::SMEM, &num_cu));
  const int cus = num_cu / 8 * 8 < 8 ? 8 : num_cu / 8 * 8;
  const int wgs = P.small ? 2 * cus : cus;
  CACO_REQUIRE(wgs <= MAX_WG, "linear loss: %d compute units", num_cu);
  return P.small ? run_loss<Small>(a, P, c.what, wgs, st) : run_loss<Big>(a, P, c.what, wgs, st);
}

}  // namespace caco
