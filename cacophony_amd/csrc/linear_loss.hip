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
//   compact      row numbers of the rows that count, in order; how many (64 rows or fewer: part of `gather`)
//   gather       those rows of `hidden`, next to one another, padded with zero rows and columns: a row that does not count takes no
//                part in any product, so whatever its hidden state holds (NaN, infinities) reaches nothing
//   lse          logits tile by tile; a workgroup stays with a block of rows for many tiles of the vocabulary, every lane keeps a sum of
//                exp2 over its own columns against a reference that only moves when a sum would leave the range (see lse_body)
//   finish       row losses in the caller's order, lse: a wave joins the workgroups that shared the row; their sum or mean in a fixed order
// and for the gradients, one piece of the vocabulary after the other (as many columns as the workspace holds):
//   dlogits      the same products again, then g (p - q), g the row's weight, rounded to bf16: the operand type of the two products that
//                follow.  The rounding is at most 2^-8 of each entry (2^-9 on average), and the targets are subtracted before it.  What all rows
//                have in common (T, the incoming gradient, 1 / count) waits for the fp32 results: inside the entries it would round
//                1 - p of every confident row alike, an error that does not average out over the rows.
//                Column sums for d bias are taken from the unrounded values.
//   targets2     (distillation) the entries of the teacher's tokens, from the logits that the loss was taken from
//   grads        d weight's tiles (sums over the tokens, complete) and d hidden (sums over the vocabulary, cut into one run per
//                workgroup that makes up for the uneven number of d weight's tiles; partial sums are kept in fp32)
//   join weight  (few of d weight's tiles and many tokens) adds d weight's runs of tokens in order
//   close        adds d hidden's partial sums and d bias's column sums in order
// Nothing is accumulated in an order that can change: equal calls give equal bits.
#define CACO_WAVE_SYNC_FENCE
#include "common.h"
#include "kernels.h"
#include "vocab_gemm.inc"

namespace caco {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int MAX_WG = 512;          // most workgroups of a persistent launch (two per CU)
constexpr int MAX_CU = 256;
// From this many rows on d hidden reads transposed weights.  Transposing costs 4 bytes of traffic per weight, whatever the rows, and saves its share of every
// K-tile.  Calls with gradients, us as the weights lie / transposed, rows x (vocabulary x dim):
//            50265 x 768    32007 x 520    10000 x 2048    20000 x 4096
//   1187      444 / 471      298 / 298      250 / 269       775 / 805
//   1800      681 / 719      400 / 389      388 / 392      1081 / 1101
//   2304      745 / 764      480 / 471      444 / 454      1299 / 1285
//   4096     1270 / 1227     732 / 703      657 / 659      2115 / 2044
//   8192     2389 / 2271    1375 / 1300    1188 / 1149     4216 / 4004
// The two meet between 1200 and 4100 rows, another number for every head; at 2048 the choice is within 3 % of the better one for all of these.
constexpr int WT_ROWS = 2048;

typedef VgTile<8, 4, 2, 4> Big;      // 256 x 256, one workgroup per CU
typedef VgTile<4, 2, 1, 4> Small;    // 64 x 128, two per CU: for calls that read the weights and do little else
// Up to this many rows take Small.  With gradients, 768 x 50265: 65 / 128 rows 135 / 143 us, with Big 143 / 150 (520 x 32007: 106 / 110, 121 / 125); from 129
// rows on Big is as fast or faster (149 rows: 154 us, with Small 173).  Losses alone, 768 x 50265: one token's logits 18 us (4.3 TB/s), with Big 30; whole
// calls for 65 / 128 / 129 / 256 rows 37 / 37 / 46 / 44 us, with Big 39 / 38 / 38 / 39.  (A head as large as 4096 x 131072 changes over earlier: 32 / 65 / 128
// rows 187 / 250 / 251, with Big 231 / 228 / 233.)
constexpr int SMALL_ROWS = 128;
// ... and so do calls that would have at most this many of Big's tiles, which would leave half the CUs idle.  Calls with gradients, us, rows x
// vocabulary x dim: 24 tiles (700 x 2000 x 2048) 94, with Big 147; 48 (300 x 6000 x 512) 63, 84; 118 (300 x 15000 x 512) 102, 107; 160 (1000 x 10000 x 512)
// 119, 114; 236 (300 x 30000 x 1000) 208, 197.  Losses alone on 20000 x 2048: 79 tiles (128 / 256 rows) 36 / 48, with Big 56 / 56; 158 (300 rows) 64, 58.
constexpr int SMALL_TILES = 128;

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
  int64_t rows, npad; int vocab, dim, hp;      // npad, hp: rows rounded up to 256, dim to the K-tile
  int reduction;
  const float* row_weight;
  const float* grad_scale;
  float *row_loss, *lse, *lse_rest, *loss;      // lse_rest: what the rounding of lse to fp32 leaves, or null
  bf16_t* dh; int64_t ld_dh;
  bf16_t* dw; int64_t ld_dw;
  float* db;
  // workspace
  int* count;                        // rows that count
  unsigned* arrived; double* sums;   // workgroups of `finish` that are through, their sums
  int *rowmap, *inv;                 // compact -> caller's row; caller's row -> compact or -1
  int* some;                         // distillation: caller's row has an entry
  int *tgt_idx0; float *tgt_q0;      // targets in the caller's order [rows, kp] (distillation)
  int *tgt_idx; float *tgt_q;        // targets of the compact rows [npad, kp]
  bf16_t* hc;                        // [npad, hp]
  bf16_t* hct;                       // [hp, npad]: its transpose, for d weight
  float2* part;                      // (max, sum) of log2-logits, [group of row blocks][workgroup][rows of a block]
  float* zt;                         // cross entropy: the label's logit
  float* tgt_z;                      // distillation: the entries' logits [npad, kp]
  // compact: lse in log2 units is lse2 + a rest of at most 0.6 (see split_lse); the row's weight in the gradients g, and g 2^-rest
  float *lse2, *g, *gr;
  // distillation, d bias: sums of g q per word as integers [16 ranges of exponents, vpad], and whether one is not finite (see targets2_kernel)
  unsigned long long* db64; unsigned* dbn;
  // d logits of the piece in blocks of 256 rows x 256 columns, [row block][column block][256][256], once with the columns next to one another
  // (d hidden sums over them) and once with the rows (d weight): both products then read fragments of 16 bytes.  (One copy and
  // transposing reads in one of the products: 2.2 us per K-tile of it instead of 1.6; those reads and the loads into LDS get in each
  // other's way, either alone is as fast.)
  bf16_t *dl, *dlt;
  bf16_t* wt;                        // the piece's weights transposed [dim, piece], zeros past the vocabulary; or null
  float* wslab; int lw;              // d weight in 2^lw runs of tokens: partial sums [piece's tile][run][256][256]
  float* slab;                       // d hidden's partial sums [output tile + workgroup][256][256]
  float* dbp; int64_t vpad;          // column sums of d logits [row halves, vpad = vocabulary rounded up to 256]
  int piece, v0;                     // columns of the piece, its first column
};

// ------------------------------------------------------------------------------------------------------------------------------------
// rows
// ------------------------------------------------------------------------------------------------------------------------------------
// One wave per row: q = softmax(t / T) over the entries whose index lies in the vocabulary; an index that occurs again adds its weight
// to its first place.  A row without entries gets none (all indices -1).
__global__ __launch_bounds__(256) void targets_kernel(LossArgs a) {
  __shared__ __attribute__((aligned(16))) int s_idx[4][128];
  __shared__ __attribute__((aligned(16))) float s_q[4][128];
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
    bool again = false;
    // every entry against every other, four at a time and without a branch, so that the reads do not wait for one another
    for (int o = 0; o < a.topk; o += 4) {
      typedef int i32x4 __attribute__((ext_vector_type(4)));
      const i32x4 si = *reinterpret_cast<const i32x4*>(&s_idx[wave][o]);
      const f32x4 sq = *reinterpret_cast<const f32x4*>(&s_q[wave][o]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        again |= si[e] == out && o + e < k;
        q += si[e] == out ? sq[e] : 0.f;
      }
    }
    if (again) out = -1;
    if (k < a.kp) {
      a.tgt_idx0[row * a.kp + k] = out;
      a.tgt_q0[row * a.kp + k] = out < 0 ? 0.f : q;
    }
  }
  if (lane == 0) a.some[row] = some;
}

// the 256 x 256 block of d logits that holds (row, col)
__device__ __forceinline__ int64_t dl_block(const LossArgs& a, int64_t row, int col) { return ((row >> 8) * (a.piece >> 8) + (col >> 8)) * 65536; }

// does row r count?
__device__ __forceinline__ bool row_counts(const LossArgs& a, int64_t r) {
  if (a.labels) {
    const int64_t y = a.labels[r];
    return y != a.ignore_index && y >= 0 && y < a.vocab;
  }
  return a.some[r] != 0;
}

// up to this many rows are counted by every workgroup of `gather` for itself, which saves `compact` and its launch (3.5 us of 35)
constexpr int FEW_ROWS = 64;

// One workgroup: every wave counts a run of consecutive rows, 64 at a time; a scan over the waves gives each run its first place.
__global__ __launch_bounds__(1024) void compact_kernel(LossArgs a) {
  __shared__ int s_n[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t per = (a.rows + 1023) / 1024 * 64;
  const int64_t r0 = min(a.rows, wave * per), r1 = min(a.rows, r0 + per);
  int n = 0;
  for (int64_t r = r0; r < r1; r += 64) n += __builtin_popcountll(__ballot(r + lane < r1 && row_counts(a, min(r + lane, r1 - 1))));
  if (lane == 0) s_n[wave] = n;
  __syncthreads();
  int at = 0;
  for (int w = 0; w < wave; ++w) at += s_n[w];
  for (int64_t r = r0; r < r1; r += 64) {
    const int64_t row = r + lane;
    const bool c = row < r1 && row_counts(a, min(row, r1 - 1));
    const unsigned long long mask = __ballot(c);
    const int place = at + __builtin_popcountll(mask & ((1ull << lane) - 1));
    if (row < r1) a.inv[row] = c ? place : -1;
    if (c) a.rowmap[place] = (int)row;
    at += __builtin_popcountll(mask);
  }
  if (threadIdx.x == 1023) {
    *a.count = at;
    *a.arrived = 0;
  }
}

// what the gradients of all n rows have in common: T from the logits' scale and the loss's T^2, the incoming gradient, the mean
__device__ __forceinline__ float common_scale(const LossArgs& a, int n) {
  if (n == 0) return 0.f;
  float g = a.temperature;
  if (a.grad_scale) g *= *a.grad_scale;
  if (a.reduction == CACO_REDUCE_MEAN) g /= (float)n;
  return g;
}

// compact row <- its hidden state (64 rows x 64 of dim to a workgroup, by rows and, for d weight, by columns), targets, weight.
// Rows up to the next multiple of 256 are zero rows.
// FEW: `compact` has not run.  Every wave counts the call's rows, one lane each, and the first workgroup writes down what `compact` does.
template <bool FEW>
__global__ __launch_bounds__(256) void gather_kernel(LossArgs a, int backward, int from_lse) {
  __shared__ bf16_t s_t[64][72];
  __shared__ int s_row[FEW ? FEW_ROWS : 1];
  const int t = threadIdx.x;
  const int64_t c0 = (int64_t)blockIdx.x * 64;
  int n;
  if (FEW) {
    const int r = t & 63;
    const bool c = r < a.rows && row_counts(a, r);
    const unsigned long long mask = __ballot(c);
    n = __builtin_popcountll(mask);
    const int place = __builtin_popcountll(mask & ((1ull << r) - 1));
    if (t < 64 && c) s_row[place] = r;
    if (t < 64 && blockIdx.x == 0 && blockIdx.y == 0) {
      if (r < a.rows) a.inv[r] = c ? place : -1;
      if (c) a.rowmap[place] = r;
      if (r == 0) {
        *a.count = n;
        *a.arrived = 0;
      }
    }
    __syncthreads();
  } else {
    n = *a.count;
  }
  const int* rowmap = FEW ? s_row : a.rowmap;
  const int h0 = blockIdx.y * 64;
  if (backward && a.db && a.topk) {
    const int64_t all = (int64_t)gridDim.x * gridDim.y * 256, at = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + t;
    typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
    for (int64_t v = at; v < 8 * a.vpad; v += all) reinterpret_cast<u64x2*>(a.db64)[v] = u64x2{0, 0};
    for (int64_t v = at; v < a.vpad; v += all) a.dbn[v] = 0;
  }
  if (c0 >= ((int64_t)n + 255) / 256 * 256) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = i * 32 + t / 8, k = t % 8 * 8;
    const int64_t c = c0 + r;
    bf16x8 v = {};
    if (c < n && h0 + k < a.dim) v = *reinterpret_cast<const bf16x8*>(a.hidden + rowmap[c] * a.ld_h + h0 + k);
    *reinterpret_cast<bf16x8*>(a.hc + c * a.hp + h0 + k) = v;
    *reinterpret_cast<bf16x8*>(&s_t[r][k]) = v;
  }
  if (backward && a.dw) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int h = i * 32 + t / 8, r = t % 8 * 8;
      bf16x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = s_t[r + e][h];
      *reinterpret_cast<bf16x8*>(a.hct + (h0 + h) * a.npad + c0 + r) = v;
    }
  }
  const int lkp = 31 - __builtin_clz((unsigned)a.kp);
  for (int k = blockIdx.y * 256 + t; k < 64 << lkp; k += 256 * gridDim.y) {
    const int64_t c = c0 + (k >> lkp);
    int idx = -1;
    float q = 0.f;
    if (c < n) {
      const int64_t row = rowmap[c];
      const int64_t at = (row << lkp) + (k & (a.kp - 1));
      idx = a.topk ? a.tgt_idx0[at] : (int)a.labels[row];
      q = a.topk ? a.tgt_q0[at] : 1.f;
    }
    a.tgt_idx[c0 * a.kp + k] = idx;
    a.tgt_q[c0 * a.kp + k] = q;
  }
  if (backward && blockIdx.y == 0 && t < 64) {
    const bool real = c0 + t < n;
    const int64_t row = real ? rowmap[c0 + t] : 0;
    const float g = real && common_scale(a, n) != 0.f ? a.row_weight ? a.row_weight[row] : 1.f : 0.f;
    a.g[c0 + t] = g;
    if (from_lse) {
      const double l = real ? ((double)a.lse[row] + (a.lse_rest ? (double)a.lse_rest[row] : 0.)) * 1.4426950408889634074 : 0.;
      const float l2 = (float)l;
      a.lse2[c0 + t] = l2;
      a.gr[c0 + t] = g * __builtin_amdgcn_exp2f(-(float)(l - (double)l2));
    }
  }
}

// The piece's weights by columns: dst [cols, ld_d] <- src [rows, cols] (ld_s), 64 x 64 at a time through the LDS; rows past the end become zeros,
// columns past the end (8 of them exist or none) are not written.
__global__ __launch_bounds__(256) void transpose_kernel(const bf16_t* src, int64_t ld_s, int64_t rows, int cols, bf16_t* dst, int64_t ld_d) {
  __shared__ bf16_t s_t[64][72];
  const int64_t c0 = (int64_t)blockIdx.x * 64;
  const int h0 = blockIdx.y * 64, t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = i * 32 + t / 8, k = t % 8 * 8;
    const bool there = c0 + r < rows && h0 + k < cols;
    *reinterpret_cast<bf16x8*>(&s_t[r][k]) = there ? *reinterpret_cast<const bf16x8*>(src + (c0 + r) * ld_s + h0 + k) : bf16x8{};
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int h = i * 32 + t / 8, r = t % 8 * 8;
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = s_t[r + e][h];
    if (h0 + h < cols) *reinterpret_cast<bf16x8*>(dst + (int64_t)(h0 + h) * ld_d + c0 + r) = v;
  }
}

// (distillation) The entries' logits: a wave takes 16 entries of a compact row at a time, their rows of weight gathered.  The same instruction
// as in the tiles, over k in the same order and from the same first sum, so that an entry has the bits its word's logit has in `lse` and `dlogits`:
// what is left when it is taken from the row's reference has no rounding at the logits' size.  15 of the 16 columns of a product are
// spent for that; what the kernel takes is the gathers' latency (eight loads of 8 rows x 128 bytes on their way) and, where the vocabulary is small
// enough to stay in the L2s, their bandwidth: whole lines through the LDS there, since loads in the products' own layout, half a line of every
// row, fetch the lines twice (2048 x 400 x 768, 128 entries: 58 us, with whole lines 27).
constexpr int target_waves(int kp) { return kp > 32 ? 4 : kp > 16 ? 2 : 1; }      // waves of a row
__global__ __launch_bounds__(256) void target_logits_kernel(LossArgs a) {
  __shared__ bf16x8 s_w[4][4][128], s_h[4][32];      // a wave's 16 rows x 256 k in four K-tiles, chunk c of row r at c ^ (r & 7); its row's hidden states
  const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4, wave = threadIdx.x >> 6;
  const int waves = target_waves(a.kp), part = wave & (waves - 1);
  const int64_t c = (int64_t)blockIdx.x * (4 / waves) + wave / waves;
  if (c >= *a.count) return;
  const bf16_t* h = a.hc + c * a.hp;
  for (int e0 = part * 16; e0 < a.kp; e0 += 16 * waves) {
    const int64_t first = c * a.kp + e0;
    const int idx = e0 + l16 < a.kp ? a.tgt_idx[first + l16] : -1;      // of the row of weight that this lane brings
    const float b = a.bias && idx >= 0 ? a.bias[idx] : 0.f;
    f32x4 acc;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = __shfl(b, lq * 4 + e, 64);
    const int r8 = lane >> 3, c8 = lane & 7;      // loading: rows r8 and r8 + 8, 16-byte chunk c8 of a line
    const bf16_t* wr[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) wr[i] = a.weight + (int64_t)max(__shfl(idx, i * 8 + r8, 64), 0) * a.ld_w;      // an absent entry reads word 0, its logit is not used
    for (int k0 = 0; k0 < a.dim; k0 += 256) {
      bf16x8 y[4][2], x = {};
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) y[t][i] = *reinterpret_cast<const bf16x8*>(wr[i] + min(k0 + t * 64 + c8 * 8, a.dim - 8));
      if (lane < 32 && k0 + lane * 8 < a.dim) x = *reinterpret_cast<const bf16x8*>(h + k0 + lane * 8);
      if (lane < 32) s_h[wave][lane] = x;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (k0 + t * 64 + c8 * 8 >= a.dim) y[t][i] = bf16x8{};
          s_w[wave][t][(i * 8 + r8) * 8 + (c8 ^ r8)] = y[t][i];
        }
      CACO_WAVE_LDS_SYNC();
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(s_w[wave][t][l16 * 8 + ((u * 4 + lq) ^ (l16 & 7))], s_h[wave][t * 8 + u * 4 + lq], acc, 0, 0, 0);
      CACO_WAVE_LDS_SYNC();
    }
    // every column holds the row's logits, those of entries lq * 4 .. + 3 in this lane: lanes l16 = 0 .. 3 take one each
    const int entry = lq * 4 + l16;
    if (l16 >= 4 || e0 + entry >= a.kp) continue;
    const float z = l16 == 0 ? acc[0] : l16 == 1 ? acc[1] : l16 == 2 ? acc[2] : acc[3];
    a.tgt_z[first + entry] = z;
  }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// logits -> running sums of exponentials
// ------------------------------------------------------------------------------------------------------------------------------------
// The order of the (row block, vocabulary tile) pairs.  Row blocks in groups of 8, then 4, 2, 1; inside a group the vocabulary's tiles, row blocks
// fastest.  An XCD takes a run of consecutive pairs, its workgroups one after the other: 8 panels of hidden states stay in its L2 and a
// panel of weights is used 8 times while it is there.  The width of a group divides the number of an XCD's workgroups, so a workgroup
// keeps its row block for a whole group.
struct Order {
  int rb, tiles, units;
  int slots, cnt, base;              // of this XCD: workgroups, pairs, first pair
  __device__ __forceinline__ Order(int n, int vocab, int bm, int bn, int wgs, int xcd) {
    rb = (n + bm - 1) / bm;
    tiles = (vocab + bn - 1) / bn;
    units = rb * tiles;
    slots = wgs >> 3;
    cnt = (units >> 3) + (xcd < (units & 7) ? 1 : 0);
    base = xcd * (units >> 3) + min(xcd, units & 7);
  }
};
struct Walk {
  int t, end;                        // pair, the run's end
  int rb, vt;                        // what it is
  int group, lw, gend;               // number of the group, log2 of its width, the pair behind it
  __device__ __forceinline__ void set(const Order& o) {
    const int full = o.rb >> 3;
    int g0 = 0, gs = 0;
    lw = 3;
    if (t < full * 8 * o.tiles) {
      group = t / (8 * o.tiles);
      g0 = group * 8;
      gs = g0 * o.tiles;
    } else {
      group = full - 1;
      g0 = full * 8;
      for (int l = 2; l >= 0; --l)
        if ((o.rb >> l) & 1) {
          ++group;
          gs = g0 * o.tiles;
          lw = l;
          if (t < gs + (o.tiles << l)) break;
          g0 += 1 << l;
        }
    }
    gend = gs + (o.tiles << lw);
    rb = g0 + ((t - gs) & ((1 << lw) - 1));
    vt = (t - gs) >> lw;
  }
  __device__ __forceinline__ Walk(const Order& o, int slot) : t(o.base + slot), end(o.base + o.cnt) { if (t < end) set(o); }
  __device__ __forceinline__ int left(const Order& o) const { return t < end ? (end - t + o.slots - 1) / o.slots : 0; }
  __device__ __forceinline__ bool last_of_group(const Order& o) const { return t + o.slots >= min(gend, end); }
  __device__ __forceinline__ void next(const Order& o) {
    t += o.slots;
    if (t < gend) vt += o.slots >> lw;
    else if (t < end) set(o);
  }
};
// groups of at most `rb` row blocks
__host__ __device__ inline int64_t most_groups(int64_t rb) { return rb / 8 + 3; }

// The words of an output tile: bias of its columns, labels (and for d logits lse, g and g 2^-rest) of its rows.
template <typename C>
struct Words {
  static constexpr int BIAS = 0, Y = C::BN * 4, LSE = Y + C::BM * 4, G = LSE + C::BM * 4, GR = G + C::BM * 4;
  static __device__ __forceinline__ void bring(const LossArgs& a, int n0, int64_t m0, bool grad, char* lds) {
    const int lane = vg_lane();
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int pc = wave; pc < (C::BN + (grad ? 4 : 1) * C::BM) / 64; pc += C::WAVES) {
      if (pc < C::BN / 64) {
        if (a.bias) vg_words(a.bias + min(n0 + pc * 64, a.vocab), a.vocab - n0 - pc * 64, lds + BIAS + pc * 256, lane);
        continue;
      }
      const int r = pc - C::BN / 64, which = r / (C::BM / 64), m = r % (C::BM / 64) * 64;
      if (which == 0 && !a.topk) vg_words(a.tgt_idx + m0 + m, 64, lds + Y + m * 4, lane);
      if (which == 1) vg_words(a.lse2 + m0 + m, 64, lds + LSE + m * 4, lane);
      if (which == 2) vg_words(a.g + m0 + m, 64, lds + G + m * 4, lane);
      if (which == 3) vg_words(a.gr + m0 + m, 64, lds + GR + m * 4, lane);
    }
  }
  // sums begin with the bias; a column past the vocabulary with -inf, its logit and nothing else comes of it
  static __device__ __forceinline__ void start(const LossArgs& a, int n0, int wn, const char* lds, f32x4 (&acc)[C::MI][C::NI]) {
    const int lq = vg_lane() >> 4;
    const bool edge = n0 + C::BN > a.vocab;
#pragma unroll
    for (int j = 0; j < C::NI; ++j) {
      const int c = wn * 16 * C::NI + j * 16 + lq * 4;
      f32x4 b = {0.f, 0.f, 0.f, 0.f};
      if (a.bias) b = *reinterpret_cast<const f32x4*>(lds + BIAS + c * 4);
      if (edge)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n0 + c + e >= a.vocab) b[e] = -INFINITY;
#pragma unroll
      for (int i = 0; i < C::MI; ++i) acc[i][j] = b;
    }
  }
};

// Per element one multiply-add, one v_exp_f32 and one addition.  The reference of a lane's row is the maximum over the row's first tile of
// this wave (four lanes share it) and stays there while a tile adds less than 2^8; when one does not (or is NaN) the whole wave goes
// over the tile again with its maxima.  Logits far below the reference add what they should: nothing.  No exponent passes 8, so its
// rounding stays below 2^-22 whatever the logits' size; and a reference that moves has grown by 4 at least, which few tiles see.
template <typename C>
__device__ __forceinline__ void lse_body(const LossArgs& a, char* smem) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const Order O(*a.count, a.vocab, C::BM, C::BN, gridDim.x, blockIdx.x & 7);
  const int wg = (blockIdx.x & 7) * O.slots + (blockIdx.x >> 3);
  Walk L(O, blockIdx.x >> 3), M = L;      // the operands, the results
  const int tiles = M.left(O);
  if (tiles == 0) return;
  const float cs = a.inv_t * LOG2E;
  const bool label = !a.topk;
  float nref[C::MI], sm[C::MI];      // minus the reference, the sum
#pragma unroll
  for (int q = 0; q < C::MI; ++q) { nref[q] = 3.0e38f; sm[q] = 0.f; }
  vg_run<C, false, true, true, true>(
      tiles, smem,
      [&](int, int& k0, int& k1) { k0 = 0; k1 = a.hp / VG_K; },
      [&](int) { return VgOperand{a.hc + (int64_t)L.rb * C::BM * a.hp, a.hp, C::BM, a.hp, 0}; },      // of the tile whose weights were asked for before
      [&](int i) {
        if (i > 0) L.next(O);
        const int n0 = L.vt * C::BN;
        return VgOperand{a.weight + (int64_t)n0 * a.ld_w, a.ld_w, a.vocab - n0, a.dim, 0};
      },
      [&](int i, char* w) {
        Walk A = M;
        if (i >= 0) A.next(O);
        Words<C>::bring(a, A.vt * C::BN, (int64_t)M.rb * C::BM, false, w);
      },
      [&](int, f32x4 (&acc)[C::MI][C::NI], char* w) { Words<C>::start(a, M.vt * C::BN, wn, w, acc); },
      [&](int, f32x4 (&acc)[C::MI][C::NI], char* slot) {
        const int lane = vg_lane(), l16 = lane & 15, lq = lane >> 4;
        const char* w = slot + C::O_WORDS;
        const int rb = M.rb, tn = M.vt;
        const int n0 = tn * C::BN + wn * 16 * C::NI + lq * 4;      // this lane's columns: n0 + j * 16 + e
#pragma unroll
        for (int q = 0; q < C::MI; ++q) {
          float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < C::NI; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[q][j][e], cs, nref[q]));
          s[0] = (s[0] + s[1]) + (s[2] + s[3]);
          if (__ballot(!(s[0] < 0x1p8f))) {
            float m = -nref[q];
#pragma unroll
            for (int j = 0; j < C::NI; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) m = fmaxf(m, acc[q][j][e] * cs);
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            sm[q] *= __builtin_amdgcn_exp2f(-nref[q] - m);
            s[0] = 0.f;
#pragma unroll
            for (int j = 0; j < C::NI; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[0] += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[q][j][e], cs, -m));
            nref[q] = -m;
          }
          sm[q] += s[0];
        }
        if (label) {
#pragma unroll
          for (int q = 0; q < C::MI; ++q) {
            const int row = (wm * C::MI + q) * 16 + l16;
            const int d = *reinterpret_cast<const int*>(w + Words<C>::Y + row * 4) - n0;      // the label's place among this lane's columns
            if ((unsigned)d < 16u * C::NI && (d & 12) == 0) {
              float zy = 0.f;
#pragma unroll
              for (int j = 0; j < C::NI; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (d == j * 16 + e) zy = acc[q][j][e];
              a.zt[(int64_t)rb * C::BM + row] = zy;
            }
          }
        }
        const bool more = !M.last_of_group(O);
        const int part = M.group * gridDim.x + wg;
        M.next(O);
        if (more) return;
        // the last tile of this row block here: the four lanes of a row, then the waves that share it
        float2* red = reinterpret_cast<float2*>(slot + C::O_RED);      // [WN][BM]
#pragma unroll
        for (int q = 0; q < C::MI; ++q) {
          float m = -nref[q], s = sm[q];
#pragma unroll
          for (int o = 16; o <= 32; o <<= 1) {
            const float om = __shfl_xor(m, o, 64), os = __shfl_xor(s, o, 64);
            const float nm = fmaxf(m, om);
            s = s * __builtin_amdgcn_exp2f(m - nm) + os * __builtin_amdgcn_exp2f(om - nm);
            m = nm;
          }
          if (lq == 0) red[wn * C::BM + (wm * C::MI + q) * 16 + l16] = make_float2(m, s);
          nref[q] = 3.0e38f;
          sm[q] = 0.f;
        }
        __syncthreads();
        for (int r = threadIdx.x; r < C::BM; r += C::THREADS) {
          float m = red[r].x, s = red[r].y;
#pragma unroll
          for (int v = 1; v < C::WN; ++v) {
            const float2 o = red[v * C::BM + r];
            const float nm = fmaxf(m, o.x);
            s = s * __builtin_amdgcn_exp2f(m - nm) + o.y * __builtin_amdgcn_exp2f(o.x - nm);
            m = nm;
          }
          a.part[(int64_t)part * C::BM + r] = make_float2(m, s);
        }
      });
}
template <typename C>
__global__ __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) void lse_kernel(LossArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  lse_body<C>(a, smem);
}

// log2 of the sum s 2^m as `whole` + `rest`.  With s = f 2^k, 0.75 <= f < 1.5, it is m + k + log2 f: `whole` is m + k rounded, `rest` log2 f and
// what that rounding lost, so the two together are good to a rounding of f.  One number would be good to a rounding of m, and all that
// is left of a confident row, log2 s of its loss and 1 - p of its gradient, would go under where the logits have a large part in common.
__device__ __forceinline__ void split_lse(float m, float s, float& k, float& lf, float& whole, float& rest) {
  const unsigned u = __float_as_uint(s);
  const int e = u - 0x00800000u < 0x7f000000u ? (int)((u + 0x00400000u) >> 23) - 127 : 0;      // positive, normal, finite; others stay as they are
  k = (float)e;
  lf = log1pf(ldexpf(s, -e) - 1.f) * LOG2E;
  whole = m + k;
  const float b = whole - m;
  rest = (m - (whole - b)) + (k - b) + lf;
}

// One wave: joins the parts of one of the caller's rows, row loss (returned, too) and lse; rows that do not count get zeros.
template <typename C>
__device__ __forceinline__ float finish_row(const LossArgs& a, int wgs, int64_t row) {
  const int lane = threadIdx.x & 63;
  const int c = a.inv[row];
  if (c < 0) {
    if (lane == 0) {
      a.row_loss[row] = 0.f;
      if (a.lse) a.lse[row] = 0.f;
      if (a.lse_rest) a.lse_rest[row] = 0.f;
    }
    return 0.f;
  }
  // the row block's group: its number, first row block, width; its pairs [gs, ge)
  const Order O(*a.count, a.vocab, C::BM, C::BN, wgs, 0);
  const int rb = c / C::BM, full = O.rb >> 3, lslots = 31 - __builtin_clz((unsigned)O.slots);
  int group = rb >> 3, g0 = group * 8, lw = 3;
  if (group >= full) {
    group = full - 1;
    g0 = full * 8;
    for (int l = 2; l >= 0; --l)
      if ((O.rb >> l) & 1) {
        ++group;
        lw = l;
        if (rb < g0 + (1 << l)) break;
        g0 += 1 << l;
      }
  }
  const int gs = g0 * O.tiles, ge = gs + (O.tiles << lw);
  float m = -3.0e38f, s = 0.f;
  for (int w0 = lane; w0 < wgs; w0 += 256) {      // the workgroups that had this row block: they have a pair of its group
    float2 o[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {                  // four loads on their way together
      const int w = w0 + u * 64;
      const int xcd = w >> lslots, q = O.units >> 3, r = O.units & 7;
      const int base = xcd * q + min(xcd, r), lo = max(gs, base), hi = min(ge, base + q + (xcd < r ? 1 : 0));
      const int t = lo + ((base + (w & (O.slots - 1)) - lo) & (O.slots - 1));
      const bool had = w < wgs && t < hi && ((t - gs) & ((1 << lw) - 1)) == rb - g0;
      o[u] = make_float2(-3.0e38f, 0.f);
      if (had) o[u] = a.part[(int64_t)(group * wgs + w) * C::BM + c % C::BM];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float nm = fmaxf(m, o[u].x);
      s = s * __builtin_amdgcn_exp2f(m - nm) + o[u].y * __builtin_amdgcn_exp2f(o[u].x - nm);
      m = nm;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float om = __shfl_xor(m, o, 64), os = __shfl_xor(s, o, 64);
    const float nm = fmaxf(m, om);
    s = s * __builtin_amdgcn_exp2f(m - nm) + os * __builtin_amdgcn_exp2f(om - nm);
    m = nm;
  }
  float k, lf, whole, rest;
  split_lse(m, s, k, lf, whole, rest);
  // -log2 of a word's probability: its logit is taken from the reference first, so nothing is rounded at the logits' size
  const float cs = a.inv_t * LOG2E;
  const auto minus_log2_p = [&](float z) { return (__builtin_fmaf(-z, cs, m) + k) + lf; };
  float d;
  if (!a.topk) {
    d = minus_log2_p(a.zt[c]);
  } else {
    d = 0.f;
    for (int i = lane; i < a.kp; i += 64) {
      const float q = a.tgt_q[(int64_t)c * a.kp + i];
      if (q != 0.f) d += q * (log2f(q) + minus_log2_p(a.tgt_z[(int64_t)c * a.kp + i]));      // 0 log 0 = 0, whatever the logit is
    }
    d = wave_sum(d);
  }
  const float loss = d * LN2 * a.temperature * a.temperature;
  if (lane == 0) {
    if (a.gr) {
      a.lse2[c] = whole;
      a.gr[c] = a.g[c] * __builtin_amdgcn_exp2f(-rest);
    }
    if (a.lse) {
      const double l = ((double)whole + (double)rest) * 0.69314718055994530942;
      a.lse[row] = (float)l;
      if (a.lse_rest) a.lse_rest[row] = fabsf((float)l) < INFINITY ? (float)(l - (double)(float)l) : 0.f;
    }
    a.row_loss[row] = loss;
  }
  return loss;
}

__device__ __forceinline__ float reduced(const LossArgs& a, double sum) {
  return (float)(a.reduction == CACO_REDUCE_MEAN ? sum / (double)*a.count : sum);      // no row counts: 0 / 0, as torch has it
}
// 16 rows to a workgroup.  The sum or mean of the (weighted) row losses: every workgroup leaves its own in `sums`, the last one to arrive
// adds them in a fixed order.  What passes from one workgroup to another goes past the XCDs' L2s (agent scope), and a workgroup
// counts itself only after its sum has arrived.
template <typename C>
__global__ __launch_bounds__(1024) void finish_kernel(LossArgs a, int wgs) {
  __shared__ double s_sum[16];
  __shared__ int s_last;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double sum = 0.;
  const int64_t row = (int64_t)blockIdx.x * 16 + wave;
  if (row < a.rows) {
    const float l = finish_row<C>(a, wgs, row);
    if (a.loss && a.inv[row] >= 0) sum = a.row_weight ? (double)l * a.row_weight[row] : (double)l;
  }
  if (!a.loss) return;
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  if (gridDim.x == 1) {
    if (threadIdx.x == 0) {
      for (int w = 1; w < 16; ++w) sum += s_sum[w];
      *a.loss = reduced(a, sum);
    }
    return;
  }
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) sum += s_sum[w];
    vg_agent_store(a.sums + blockIdx.x, sum);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    s_last = atomicAdd(a.arrived, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  sum = 0.;
  for (unsigned b = threadIdx.x; b < gridDim.x; b += 1024) sum += vg_agent_load(a.sums + b);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) sum += s_sum[w];
    *a.loss = reduced(a, sum);
  }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// gradients
// ------------------------------------------------------------------------------------------------------------------------------------
template <typename C>
__device__ __forceinline__ void dlogits_body(const LossArgs& a, char* smem) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const Order O(*a.count, a.piece, C::BM, C::BN, gridDim.x, blockIdx.x & 7);
  Walk L(O, blockIdx.x >> 3), M = L;      // the operands, the results
  const int tiles = M.left(O);
  if (tiles == 0) return;
  const float cs = a.inv_t * LOG2E;
  const bool label = !a.topk;
  vg_run<C, false, true, true, true>(
      tiles, smem,
      [&](int, int& k0, int& k1) { k0 = 0; k1 = a.hp / VG_K; },
      [&](int) { return VgOperand{a.hc + (int64_t)L.rb * C::BM * a.hp, a.hp, C::BM, a.hp, 0}; },      // of the tile whose weights were asked for before
      [&](int i) {
        if (i > 0) L.next(O);
        const int n0 = a.v0 + L.vt * C::BN;
        return VgOperand{a.weight + (int64_t)min(n0, a.vocab - 1) * a.ld_w, a.ld_w, max(1, a.vocab - n0), a.dim, 0};
      },
      [&](int i, char* w) {
        Walk A = M;
        if (i >= 0) A.next(O);
        Words<C>::bring(a, a.v0 + A.vt * C::BN, (int64_t)M.rb * C::BM, true, w);
      },
      [&](int, f32x4 (&acc)[C::MI][C::NI], char* w) { Words<C>::start(a, a.v0 + M.vt * C::BN, wn, w, acc); },
      [&](int, f32x4 (&acc)[C::MI][C::NI], char* slot) {
        const int lane = vg_lane(), l16 = lane & 15, lq = lane >> 4;
        const char* w = slot + C::O_WORDS;
        char* slab = slot + wave * C::SLAB;
        const int tm = M.rb, tn = M.vt;
        M.next(O);
        const int64_t m0 = (int64_t)tm * C::BM + wm * 16 * C::MI;
        const int c0 = tn * C::BN + wn * 16 * C::NI;                  // the wave's first column in the piece
        const int v0 = a.v0 + c0, n0 = v0 + lq * 4;                   // its word; this lane's columns: n0 + j * 16 + e
        f32x4 col[C::NI];
#pragma unroll
        for (int j = 0; j < C::NI; ++j) col[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        typedef VgTurn<C> Turn;
        const int64_t block = dl_block(a, m0, c0);      // the wave's rows and columns lie in one block
        const int br = (int)(m0 & 255), bc = c0 & 255;
#pragma unroll
        for (int q2 = 0; q2 < C::MI / 2; ++q2) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {                  // 32 rows x half the columns at a time
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int q = q2 * 2 + u, row = (wm * C::MI + q) * 16 + l16;
              const float nl = -*reinterpret_cast<const float*>(w + Words<C>::LSE + row * 4), g = *reinterpret_cast<const float*>(w + Words<C>::G + row * 4);
              const float gr = *reinterpret_cast<const float*>(w + Words<C>::GR + row * 4);
              f32x4 p[Turn::NJ];
#pragma unroll
              for (int j = 0; j < Turn::NJ; ++j) p[j] = f32x4{0.f, 0.f, 0.f, 0.f};
              if (g != 0.f) {      // a row of weight 0 has no gradient, whatever its logits are
#pragma unroll
                for (int j = 0; j < Turn::NJ; ++j)
#pragma unroll
                  for (int e = 0; e < 4; ++e) p[j][e] = gr * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[q][h * Turn::NJ + j][e], cs, nl));
                if (label) {
                  const int d = *reinterpret_cast<const int*>(w + Words<C>::Y + row * 4) - n0 - h * Turn::NJ * 16;
                  if ((unsigned)d < 16u * Turn::NJ && (d & 12) == 0) {
#pragma unroll
                    for (int j = 0; j < Turn::NJ; ++j)
#pragma unroll
                      for (int e = 0; e < 4; ++e)
                        if (d == j * 16 + e) p[j][e] -= g;
                  }
                }
              }
#pragma unroll
              for (int j = 0; j < Turn::NJ; ++j) {
                col[h * Turn::NJ + j] += p[j];
                vg_here(col[h * Turn::NJ + j]);
                Turn::put(slab, u * 16 + l16, lq, j, p[j]);
              }
            }
            CACO_WAVE_LDS_SYNC();
            const int r0 = br + q2 * 32, k0 = bc + h * Turn::NJ * 16;
            Turn::rows(slab, lane, [&](int r, int ch, bf16x8 v) { vg_stream(a.dl + block + (r0 + r) * 256 + k0 + ch * 8, v); });
            if (a.dw) Turn::columns(slab, l16, lq, [&](int k, int oct, bf16x8 v) { vg_stream(a.dlt + block + (k0 + k) * 256 + r0 + oct * 8, v); });
            CACO_WAVE_LDS_SYNC();
            __builtin_amdgcn_sched_barrier(0);      // one part's registers at a time
          }
        }
        if (a.db && v0 < a.vpad) {
#pragma unroll
          for (int j = 0; j < C::NI; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int o = 1; o < 16; o <<= 1) col[j][e] += __shfl_xor(col[j][e], o, 64);
          if (l16 == 0)
#pragma unroll
            for (int j = 0; j < C::NI; ++j) *reinterpret_cast<f32x4*>(a.dbp + ((int64_t)tm * C::WM + wm) * a.vpad + v0 + j * 16 + lq * 4) = col[j];
        }
      });
}
template <typename C>
__global__ __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) void dlogits_kernel(LossArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  dlogits_body<C>(a, smem);
}

// (distillation) d logits at the teacher's tokens of the piece: one thread per entry.  The tokens of a row are distinct, so an entry is
// written by one thread.  Their share of d bias, g q, is added up exactly, as integers, whose sum does not depend on the order: 16 sums for a word, one for every
// 16 exponents, so that a share is its 24 bits shifted by 15 at most, and the sum of 2^22 rows stays below 2^61.  (One sum in units that the word's largest share
// sets takes a pass of its own to find that one: 36 us where 2048 x 128 entries meet on 400 words.)  A share that is not finite marks the word.
__global__ __launch_bounds__(256) void targets2_kernel(LossArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t c = t / a.kp;
  if (c >= *a.count) return;
  const int idx = a.tgt_idx[t], v = idx - a.v0;
  const float g = a.g[c], q = a.tgt_q[t];
  if (idx < 0 || v < 0 || v >= a.piece || g == 0.f || q == 0.f) return;
  const bf16_t d = (bf16_t)(a.gr[c] * __builtin_amdgcn_exp2f(__builtin_fmaf(a.tgt_z[t], a.inv_t * LOG2E, -a.lse2[c])) - g * q);
  const int64_t block = dl_block(a, c, v);
  a.dl[block + (c & 255) * 256 + (v & 255)] = d;
  if (a.dw) a.dlt[block + (v & 255) * 256 + (c & 255)] = d;
  if (!a.db) return;
  const unsigned u = __float_as_uint(g * q);
  const int E = u >> 23 & 255;
  if (E == 255) {
    atomicMax(a.dbn + idx, 1u);
    return;
  }
  const long long m = (long long)((u & 0x7fffff) | (E ? 0x800000 : 0)) << (max(E, 1) - (E & ~15));      // in units of 2^((E & ~15) - 150)
  atomicAdd(a.db64 + (int64_t)(E >> 4) * a.vpad + idx, (unsigned long long)(u >> 31 ? -m : m));
}

// How a piece's gradient work is shared out, XCD by XCD.
//   d weight   an XCD takes a run of whole tiles, its workgroups one after the other, column blocks fastest: they share a panel of d logits.
//   d hidden   `ks` slices of the vocabulary times 8 / ks runs of the output tiles: the fewest slices that leave an XCD a tile for each of its
//              workgroups, so that these walk the same part of the vocabulary together, with few panels between them: at 22 row blocks and
//              3 column blocks the launch takes 1.8 GB through the L2s, which hold 72 % of what it reads, and 653 us; with one
//              slice 4.0 GB, 41 % and 768 us.  Tiles beyond a multiple of the
//              workgroups make one list of K-tiles, cut so that workgroups with one d weight tile less get more of it.
// A slice of a whole tile is kept at [tile][slice], a part of the list at [XCD][tile of the list + workgroup] (the sum grows from part to
// part, so the places are distinct).
struct Share {
  int rb, cb, tiles, nk, ks;       // d hidden: row blocks, column blocks, output tiles, K-tiles of one, slices
  int nka, nkw, slots;             // d weight: K-tiles of a tile, at most of one of its runs; workgroups of an XCD
  int wcnt, wbase;                 // this XCD's d weight runs, the first
  int slice, k0, nkx;              // its slice, the slice's first K-tile and length
  int t0, whole, rest;             // its output tiles: the first, whole ones per workgroup, tiles in the list
  int more, few, many;             // workgroups with a d weight tile more; K-tiles of the list for these and for the others
  // wgs, ks and with them everything divided by below but `slots - more` are powers of two
  __device__ __forceinline__ Share(const LossArgs& a, int n, int wgs, int xcd) {
    slots = wgs >> 3;
    const int lslots = 31 - __builtin_clz((unsigned)slots);
    rb = a.dh ? (n + 255) / 256 : 0;
    cb = (a.dim + 255) / 256;
    tiles = rb * cb;
    nk = a.piece / VG_K;
    nka = (n + VG_K - 1) / VG_K;
    nkw = (nka + (1 << a.lw) - 1) >> a.lw;
    const int wt = a.dw ? (a.piece / 256 * cb) << a.lw : 0;
    wcnt = (wt >> 3) + (xcd < (wt & 7) ? 1 : 0);
    wbase = xcd * (wt >> 3) + min(xcd, wt & 7);
    int lks = 0;
    while (lks < 3 && (tiles << lks) < 8 * slots) ++lks;
    ks = 1 << lks;
    const int lgroups = 3 - lks, grp = xcd >> lks;
    slice = xcd & (ks - 1);
    k0 = (int)(((int64_t)slice * nk) >> lks);
    nkx = (int)(((int64_t)(slice + 1) * nk) >> lks) - k0;
    t0 = (int)(((int64_t)grp * tiles) >> lgroups);
    const int nt = (int)(((int64_t)(grp + 1) * tiles) >> lgroups) - t0;
    whole = nt >> lslots;
    rest = nt & (slots - 1);
    const int f = wcnt >> lslots;
    more = wcnt & (slots - 1);
    const int list = rest * nkx;   // < slots * 2^18
    few = max(0, (int)(((list + (int64_t)wcnt * nkw + slots - 1) >> lslots) - (int64_t)(f + 1) * nkw));
    many = (unsigned)(list - (int)min((int64_t)list, (int64_t)few * more) + slots - more - 1) / (unsigned)(slots - more);
  }
  // first K-tile of workgroup s in the list
  __device__ __forceinline__ int first(int s) const {
    const int m = min(s, more);
    return s >= slots ? rest * nkx : (int)min((int64_t)rest * nkx, (int64_t)m * few + (int64_t)(s - m) * many);
  }
  __device__ __forceinline__ int64_t slab_whole(int tile) const { return (int64_t)tile * ks + slice; }
  __device__ __forceinline__ int64_t slab_list(int xcd, int i, int s) const { return (int64_t)tiles * ks + xcd * (min(tiles, slots) + slots) + i + s; }
  // slabs that can be needed with `most` output tiles at most
  static int64_t slabs(int64_t most, int slots) {
    return (most > 16 * slots ? most : (most * 8 < 16 * slots ? most * 8 : 16 * slots)) + 8 * ((most < slots ? most : slots) + slots);
  }
};

template <bool WT>
__device__ __forceinline__ void grads_body(const LossArgs& a, char* smem) {
  typedef Big C;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int n = *a.count;
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
  const float scale = common_scale(a, n);
  const Share S(a, n, gridDim.x, xcd);
  // d weight: both operands with the token fastest
  if (slot < S.wcnt)
    vg_run<C, false, false, false, false>(
        (S.wcnt - slot + S.slots - 1) / S.slots, smem,
        [&](int i, int& k0, int& k1) {
          const int run = (S.wbase + slot + i * S.slots) & ((1 << a.lw) - 1);
          k0 = (run * S.nka) >> a.lw;
          k1 = ((run + 1) * S.nka) >> a.lw;
        },
        [&](int i) {
          const int tm = ((S.wbase + slot + i * S.slots) >> a.lw) / S.cb;
          return VgOperand{a.dlt + (int64_t)tm * 65536, 256, C::BM, S.nka * VG_K, (int64_t)a.piece * 256};
        },
        [&](int i) {
          const int c = ((S.wbase + slot + i * S.slots) >> a.lw) % S.cb * C::BN;
          return VgOperand{a.hct + c * a.npad, a.npad, a.hp - c, S.nka * VG_K, 0};
        },
        VgNoWords{}, VgZero{},
        [&](int i, f32x4 (&acc)[C::MI][C::NI], char* free_slot) {
          const int lane = vg_lane(), l16 = lane & 15, lq = lane >> 4;
          char* slab = free_slot + wave * C::SLAB;
          const int u = S.wbase + slot + i * S.slots, t = u >> a.lw, tn = t % S.cb, tm = t / S.cb;
          if (a.lw) {
            float* d = a.wslab + (int64_t)u * C::BM * C::BN + (wm * 16 * C::MI + l16) * C::BN + wn * 16 * C::NI + lq * 4;
#pragma unroll
            for (int q = 0; q < C::MI; ++q)
#pragma unroll
              for (int j = 0; j < C::NI; ++j) *reinterpret_cast<f32x4*>(d + q * 16 * C::BN + j * 16) = acc[q][j];
            return;
          }
          const int v0 = a.v0 + tm * C::BM + wm * 16 * C::MI, c0 = tn * C::BN + wn * 16 * C::NI;
#pragma unroll
          for (int q = 0; q < C::MI; ++q) {
#pragma unroll
            for (int j = 0; j < C::NI; ++j) vg_slab_put<C>(slab, l16, lq, j, acc[q][j] * scale);
            CACO_WAVE_LDS_SYNC();
            vg_slab_rows<C>(slab, lane, [&](int r, int ch, bf16x8 v) {
              const int vv = v0 + q * 16 + r, cc = c0 + ch * 8;
              if (vv < a.vocab && cc < a.dim) vg_stream(a.dw + (int64_t)vv * a.ld_dw + cc, v);
            });
            CACO_WAVE_LDS_SYNC();
          }
        });
  // d hidden: the workgroup's whole tiles, then its part of the list.  The weights as they lie (word slowest), or transposed (WT)
  const int f0 = S.first(slot), f1 = S.first(slot + 1), l0 = f0 < f1 ? f0 / S.nkx : 0;
  const int parts = S.whole + (f0 < f1 ? (f1 - 1) / S.nkx - l0 + 1 : 0);
  if (parts == 0) return;
  const bool first_piece = a.v0 == 0;
  auto out_tile = [&](int i) { return i < S.whole ? S.t0 + slot + i * S.slots : S.t0 + S.whole * S.slots + l0 + i - S.whole; };
  vg_run<C, !WT, false, false, false>(
      parts, smem,
      [&](int i, int& k0, int& k1) {
        const int at = i < S.whole ? 0 : (l0 + i - S.whole) * S.nkx;      // the tile's first K-tile in the list
        k0 = S.k0 + (i < S.whole ? 0 : max(0, f0 - at));
        k1 = S.k0 + (i < S.whole ? S.nkx : min(S.nkx, f1 - at));
      },
      [&](int i) { return VgOperand{a.dl + (int64_t)(out_tile(i) / S.cb) * C::BM * a.piece, 256, C::BM, a.piece, 65536}; },
      [&](int i) {
        const int c = out_tile(i) % S.cb * C::BN;
        if (WT) return VgOperand{a.wt + (int64_t)c * a.piece, a.piece, a.dim - c, a.piece, 0};
        return VgOperand{a.weight + (int64_t)a.v0 * a.ld_w + c, a.ld_w, a.dim - c, a.vocab - a.v0, 0};
      },
      VgNoWords{}, VgZero{},
      [&](int i, f32x4 (&acc)[C::MI][C::NI], char*) {
        const int o = out_tile(i), rb = o / S.cb;
        const int lane = vg_lane(), l16 = lane & 15, lq = lane >> 4;
        const int64_t place = i < S.whole ? S.slab_whole(o) : S.slab_list(xcd, l0 + i - S.whole, slot);
        float* d = a.slab + place * C::BM * C::BN + (wm * 16 * C::MI + l16) * C::BN + wn * 16 * C::NI + lq * 4;
#pragma unroll
        for (int q = 0; q < C::MI; ++q) {
          if (rb * C::BM + (wm * C::MI + q) * 16 >= n) continue;
#pragma unroll
          for (int j = 0; j < C::NI; ++j) {
            f32x4 v = acc[q][j];
            f32x4* p = reinterpret_cast<f32x4*>(d + q * 16 * C::BN + j * 16);
            if (!first_piece) v += *p;
            *p = v;
          }
        }
      });
}
template <bool WT>
__global__ __launch_bounds__(Big::THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) void grads_kernel(LossArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  grads_body<WT>(a, smem);
}

// d weight from its runs of tokens, in order: 8 rows of a tile to a workgroup
__global__ __launch_bounds__(256) void join_weight_kernel(LossArgs a) {
  const int cb = (a.dim + 255) / 256, tile = blockIdx.x >> 5, row = (blockIdx.x & 31) * 8 + threadIdx.x / 32, col = threadIdx.x % 32 * 8;
  const int v = a.v0 + tile / cb * 256 + row, x = tile % cb * 256 + col;
  if (v >= a.vocab || x >= a.dim) return;
  const float* p = a.wslab + ((int64_t)tile << a.lw) * 65536 + row * 256 + col;
  f32x4 s[2] = {};
#pragma unroll 4
  for (int r = 0; r < 1 << a.lw; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) s[h] += *reinterpret_cast<const f32x4*>(p + (int64_t)r * 65536 + h * 4);
  const float scale = common_scale(a, *a.count);
  bf16x8 o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (bf16_t)(s[e / 4][e % 4] * scale);
  *reinterpret_cast<bf16x8*>(a.dw + (int64_t)v * a.ld_dw + x) = o;
}

__device__ __forceinline__ void dbias(const LossArgs& a, int v, int bm, int wm) {
  if (v >= a.vocab) return;
  const int parts = (*a.count + bm - 1) / bm * wm;
  float s = 0.f;
#pragma unroll 8
  for (int p = 0; p < parts; ++p) s += a.dbp[p * a.vpad + v];
  if (a.topk) {
    double t = 0., unit = 0x1p-150;
#pragma unroll
    for (int b = 0; b < 16; ++b, unit *= 0x1p16) t += (double)(long long)a.db64[b * a.vpad + v] * unit;
    s = a.dbn[v] ? NAN : (float)((double)s - t);
  }
  a.db[v] = s * common_scale(a, *a.count);
}

// What is left to add up, in order, once the pieces are through.  The first `joins` workgroups: d hidden's parts, rounded once, 8 compact rows x
// 256 of dim each, and zeros for those of the caller's rows with the same numbers that do not count.  The others: d bias, 256 words each.
// G = 8: one row to a workgroup, every eighth part to 32 threads, these eight sums added in order.  With one block of rows a tile has up to 8 * 32
// parts and there are few rows to share them out by.
template <int G>
__global__ __launch_bounds__(256) void close_kernel(LossArgs a, int wgs, int joins, int bm, int wm) {
  if ((int)blockIdx.x >= joins) {
    dbias(a, ((int)blockIdx.x - joins) * 256 + threadIdx.x, bm, wm);
    return;
  }
  const int cbs = (a.dim + 255) / 256, by = (int)blockIdx.x % cbs;
  __shared__ int s_parts[4], s_list[MAX_CU];
  __shared__ f32x4 s_sum[G == 1 ? 1 : 256][2];
  const int n = *a.count, t = threadIdx.x, grp = G == 1 ? 0 : t / 32;
  const int64_t c0 = (int64_t)((int)blockIdx.x / cbs) * (8 / G), c = G == 1 ? c0 + t / 32 : c0;
  const int x = by * 256 + t % 32 * 8;
  if (grp == 0 && c < a.rows && x < a.dim && a.inv[c] < 0) *reinterpret_cast<bf16x8*>(a.dh + c * a.ld_dh + x) = bf16x8{};
  if (c0 >= n) return;
  // where the parts of this output tile are: a thread per workgroup of `grads`, 32 to an XCD; the list in their order
  static_assert(MAX_CU == 256, "a thread per workgroup");
  int place = -1;
  {
    const Share S(a, n, wgs, t >> 5);
    const int o = (int)(c0 / 256) * S.cb + by, i = o - S.t0 - S.whole * S.slots, s = t & 31;      // i: the tile's place in the list
    if (o >= S.t0 && i < S.rest && s < S.slots) {
      if (i < 0) {
        if (s == 0) place = (int)S.slab_whole(o);
      } else {
        const int f0 = S.first(s), f1 = S.first(s + 1);
        if (f0 < (i + 1) * S.nkx && f1 > i * S.nkx && f1 > f0) place = (int)S.slab_list(t >> 5, i, s);
      }
    }
  }
  const unsigned long long mask = __ballot(place >= 0);
  if ((t & 63) == 0) s_parts[t >> 6] = __builtin_popcountll(mask);
  __syncthreads();
  int parts = 0, at = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < t >> 6) at += s_parts[w];
    parts += s_parts[w];
  }
  if (place >= 0) s_list[at + __builtin_popcountll(mask & ((1ull << (t & 63)) - 1))] = place;
  __syncthreads();
  if (G == 1 && (x >= a.dim || c >= n)) return;
  f32x4 v[2] = {};
  const float* p = a.slab + (c % 256) * 256 + t % 32 * 8;
  int k = grp;
  for (; k + 7 * G < parts; k += 8 * G) {      // their loads must not wait for one another
    f32x4 u[8][2];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) u[j][h] = *reinterpret_cast<const f32x4*>(p + (int64_t)s_list[k + j * G] * 65536 + h * 4);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) v[h] += u[j][h];
  }
  for (; k < parts; k += G)
#pragma unroll
    for (int h = 0; h < 2; ++h) v[h] += *reinterpret_cast<const f32x4*>(p + (int64_t)s_list[k] * 65536 + h * 4);
  if (G != 1) {
#pragma unroll
    for (int h = 0; h < 2; ++h) s_sum[t][h] = v[h];
    __syncthreads();
    if (grp || x >= a.dim) return;
#pragma unroll
    for (int g = 1; g < G; ++g)
#pragma unroll
      for (int h = 0; h < 2; ++h) v[h] += s_sum[g * 32 + t][h];
  }
  const float scale = common_scale(a, n);
  bf16x8 o8;
#pragma unroll
  for (int e = 0; e < 8; ++e) o8[e] = (bf16_t)(v[e / 4][e % 4] * scale);
  *reinterpret_cast<bf16x8*>(a.dh + (int64_t)a.rowmap[c] * a.ld_dh + x) = o8;
}

// ------------------------------------------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------------------------------------------
int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// Where everything lies in the workspace.  Sizes are for all `rows`; how many of them count is known on the device only.
struct Plan {
  int64_t npad, vpad = 0, bytes = 0;
  int hp, kp;
  int64_t piece;
  bool small;
  int lw = 0;
  int64_t o_wslab = 0, o_count, o_sums, o_some, o_rowmap, o_inv, o_ti0, o_tq0, o_ti, o_tq, o_tz, o_hc, o_hct, o_part, o_zt, o_lse2, o_g, o_gr, o_db64, o_dbn, o_dl, o_dlt, o_wt, o_slab, o_dbp;
  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += up(n, 256);
    return at;
  }
  // piece_cols 0: losses alone
  Plan(int64_t rows, int vocab, int dim, int topk, int64_t piece_cols) {
    npad = up(rows > 0 ? rows : 1, 256);
    hp = (int)up(dim, VG_K);
    kp = 1;
    while (kp < topk) kp *= 2;
    small = rows <= SMALL_ROWS || npad / 256 * ((vocab + 255) / 256) <= SMALL_TILES;
    const int bm = small ? Small::BM : Big::BM;
    o_count = take(8);                                         // and `arrived`
    o_sums = take(npad / 16 * 8);
    o_some = topk ? take(npad * 4) : 0;
    o_rowmap = take(npad * 4);
    o_inv = take(npad * 4);
    o_ti0 = topk ? take(npad * kp * 4) : 0;
    o_tq0 = topk ? take(npad * kp * 4) : 0;
    o_tz = topk ? take(npad * kp * 4) : 0;
    o_ti = take(npad * kp * 4);
    o_tq = take(npad * kp * 4);
    o_hc = take(npad * hp * 2);
    o_part = take(most_groups(npad / bm) * (small ? MAX_WG : MAX_CU) * bm * 8);
    o_zt = take(npad * 4);
    piece = piece_cols;
    o_lse2 = o_g = o_gr = o_hct = o_db64 = o_dbn = o_dl = o_dlt = o_slab = o_dbp = 0;
    o_wt = -1;
    if (piece) {
      o_lse2 = take(npad * 4);
      o_g = take(npad * 4);
      o_gr = take(npad * 4);
      vpad = up(vocab, 256);
      if (topk) o_db64 = take(16 * vpad * 8), o_dbn = take(vpad * 4);
      o_hct = take((int64_t)hp * npad * 2);
      o_dl = take(npad * piece * 2);
      o_dlt = take(npad * piece * 2);
      o_wt = rows >= WT_ROWS ? take((int64_t)dim * piece * 2) : -1;
      o_slab = take(Share::slabs(npad / 256 * ((dim + 255) / 256), MAX_CU / 8) * 65536 * 4);
      // A small vocabulary has few tiles of d weight, and many tokens make them long: they are cut into runs of 8 K-tiles or more as long as
      // there are CUs for them, from 1536 tokens on.  Calls with gradients, us, rows x vocabulary x dim: 1000 x 6000 x 512 103, uncut 96; 2000 x 2000 x 1000
      // 125, 143; 8192 x 300 x 2000 196, 294; 8192 x 1000 x 64 119, 233.  (The whole vocabulary's tiles count: the size is then the same for every piece.)
      const int64_t wtiles = (int64_t)(vocab + 255) / 256 * ((dim + 255) / 256);
      while (npad >= 1536 && (wtiles << (lw + 1)) <= MAX_CU && (npad / VG_K >> (lw + 1)) >= 8) ++lw;
      if (lw) o_wslab = take((wtiles << lw) * 65536 * 4);
      o_dbp = take(npad / bm * (small ? Small::WM : Big::WM) * vpad * 4);
    }
  }
};

// columns of a piece: the vocabulary in as few equal pieces as d logits of `budget` bytes allow, in whole tiles
// The 256 rows of a tile are addressed from its first one with 32 bits: 255 strides of bf16 stay below 2^31.  The strides are `dim`,
// the weight's, and in the transposed operands the rows (padded) and the piece.
constexpr int64_t MAX_LD = (int64_t)1 << 22;
static_assert(255 * MAX_LD * 2 + VG_K * 2 < 0x7fffffff, "a tile's last row lies within its descriptor");

int64_t piece_for(int64_t rows, int vocab, int64_t budget) {
  const int64_t npad = up(rows > 0 ? rows : 1, 256), all = up(vocab, 256);
  int64_t most = budget / (npad * 4) / 256 * 256;      // two copies
  if (most < 256) most = 256;
  if (most > MAX_LD) most = MAX_LD;
  const int64_t pieces = (all + most - 1) / most;
  return up((all + pieces - 1) / pieces, 256);
}

// Up to this many rows `close` takes one row to a workgroup.  768 x 50265, us for 37 / 256 / 1000 / 2000 rows: 5.4 / 12.7 / 17.1 / 22.5; with eight rows
// 15.4 / 18.8 / 20.2 / 21.5.
constexpr int ONE_ROW = 1024;

template <typename K, typename... A>
int launch(const char* what, K kern, dim3 grid, int threads, int lds, hipStream_t st, A... args) {
  int num_cu = 0;
  if (lds) CACO_TRY_RC(prepare_launch(reinterpret_cast<const void*>(kern), lds, &num_cu));
  hipLaunchKernelGGL(kern, grid, dim3(threads), lds, st, args...);
  return check_hip(hipGetLastError(), what);
}

template <typename C>
int run_loss(LossArgs& a, const Plan& P, int what, int cus, hipStream_t st) {
  const dim3 rows4((unsigned)((a.rows + 3) / 4));
  const int wgs = P.small ? 2 * cus : cus;
  const bool fwd = what & CACO_LOSS_FORWARD, bwd = what & CACO_LOSS_BACKWARD;
  if (a.topk && a.rows) CACO_TRY_RC(launch("loss targets", targets_kernel, rows4, 256, 0, st, a));
  const bool few = a.rows <= FEW_ROWS;
  if (!few) CACO_TRY_RC(launch("loss compact", compact_kernel, dim3(1), 1024, 0, st, a));
  CACO_TRY_RC(launch("loss gather", few ? gather_kernel<true> : gather_kernel<false>, dim3((unsigned)(P.npad / 64), a.hp / 64), 256, 0, st, a, (int)bwd, (int)!fwd));
  if (a.topk) CACO_TRY_RC(launch("loss target logits", target_logits_kernel, dim3((unsigned)(P.npad / (4 / target_waves(a.kp)))), 256, 0, st, a));
  if (fwd) {
    CACO_TRY_RC(launch("loss lse", lse_kernel<C>, dim3(wgs), C::THREADS, C::SMEM_WFAR, st, a));
    const int64_t fin = (a.rows + 15) / 16;
    if (a.rows || a.loss) CACO_TRY_RC(launch("loss finish", finish_kernel<C>, dim3((unsigned)(fin ? fin : 1)), 1024, 0, st, a, wgs));
  }
  if (!bwd) return CACO_OK;
  for (; a.v0 < a.vocab; a.v0 += a.piece) {
    CACO_TRY_RC(launch("loss dlogits", dlogits_kernel<C>, dim3(wgs), C::THREADS, C::SMEM_WFAR, st, a));
    if (a.topk) CACO_TRY_RC(launch("loss targets2", targets2_kernel, dim3((unsigned)(P.npad * a.kp / 256)), 256, 0, st, a));
    if (a.dh && a.wt)
      CACO_TRY_RC(launch("loss weight transpose", transpose_kernel, dim3(a.piece / 64, (a.dim + 63) / 64), 256, 0, st, a.weight + a.v0 * a.ld_w, a.ld_w,
                         (int64_t)(a.vocab - a.v0), a.dim, a.wt, (int64_t)a.piece));
    if (a.dh || a.dw) CACO_TRY_RC(launch("loss grads", a.wt ? grads_kernel<true> : grads_kernel<false>, dim3(cus), Big::THREADS, Big::SMEM_XFAR, st, a));
    if (a.dw && a.lw) CACO_TRY_RC(launch("loss join weight", join_weight_kernel, dim3((unsigned)(a.piece / 256 * ((a.dim + 255) / 256) * 32)), 256, 0, st, a));
  }
  const bool one = a.rows <= ONE_ROW;
  const int64_t joins = a.dh ? (one ? a.rows : (a.rows + 7) / 8) * ((a.dim + 255) / 256) : 0, words = a.db ? (a.vocab + 255) / 256 : 0;
  if (joins + words)
    CACO_TRY_RC(launch("loss close", one ? close_kernel<8> : close_kernel<1>, dim3((unsigned)(joins + words)), 256, 0, st, a, cus, (int)joins, (int)C::BM, (int)C::WM));
  return CACO_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_sizes(int64_t rows, int32_t vocab, int32_t dim, int32_t topk) {
  CACO_REQUIRE(rows >= 0 && rows <= MAX_LD, "linear loss: rows must be 0 .. 2^22, got %lld", (long long)rows);
  CACO_REQUIRE(vocab >= 1 && vocab <= 1 << 24, "linear loss: vocab must be 1 .. 2^24, got %d", vocab);
  CACO_REQUIRE(dim >= 8 && dim <= 1 << 16 && dim % 8 == 0, "linear loss: dim must be a multiple of 8 in 8 .. 65536, got %d", dim);
  CACO_REQUIRE(up(rows, 256) * up(vocab, 256) <= (int64_t)1 << 46, "linear loss: rows * vocab must not exceed 2^46, got %lld * %d", (long long)rows, vocab);
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
  CACO_REQUIRE((c.what & 3) && !(c.what & ~7), "linear loss: `what` must be CACO_LOSS_FORWARD, CACO_LOSS_BACKWARD or both, with CACO_LOSS_LSE_PAIR or without");
  CACO_REQUIRE(c.reduction >= CACO_REDUCE_NONE && c.reduction <= CACO_REDUCE_SUM, "linear loss: unknown reduction %d", c.reduction);
  CACO_REQUIRE(c.weight && c.ws && (c.rows == 0 || (c.hidden && (c.topk ? c.teacher && c.teacher_idx : c.labels != nullptr))), "linear loss: null argument");
  CACO_REQUIRE(c.topk == 0 || (c.temperature > 0.f && c.temperature < INFINITY), "linear loss: temperature must be positive and finite");
  CACO_REQUIRE(c.topk == 0 || (c.temperature >= 0x1p-20f && c.temperature <= 0x1p20f), "linear loss: temperature must be within 2^-20 .. 2^20, got %g", (double)c.temperature);
  const bool fwd = c.what & CACO_LOSS_FORWARD, bwd = c.what & CACO_LOSS_BACKWARD;
  CACO_REQUIRE(!fwd || c.rows == 0 || c.row_loss, "linear loss: the forward pass needs row_loss");
  CACO_REQUIRE(!c.loss || (fwd && c.reduction != CACO_REDUCE_NONE), "linear loss: a reduced loss needs the forward pass and a reduction");
  CACO_REQUIRE(fwd || c.rows == 0 || c.lse, "linear loss: the backward pass alone needs the forward pass's lse");
  CACO_REQUIRE(!bwd || c.d_hidden || c.d_weight || c.d_bias, "linear loss: the backward pass has no output");
  CACO_REQUIRE(c.ld_h >= c.dim && c.ld_h % 8 == 0 && c.ld_w >= c.dim && c.ld_w % 8 == 0 && c.ld_w < MAX_LD && aligned16(c.hidden) && aligned16(c.weight),
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
    int64_t lo = 1, hi = (all < MAX_LD ? all : MAX_LD) / 256;      // in tiles; the plan's size grows with the piece
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
  a.rows = c.rows; a.npad = P.npad; a.vocab = c.vocab; a.dim = c.dim; a.hp = P.hp;
  a.reduction = c.reduction; a.row_weight = c.row_weight; a.grad_scale = c.grad_scale;
  a.row_loss = c.row_loss; a.lse = c.lse; a.lse_rest = c.lse && (c.what & CACO_LOSS_LSE_PAIR) ? c.lse + c.rows : nullptr; a.loss = c.loss;
  a.dh = bwd ? c.d_hidden : nullptr; a.ld_dh = c.ld_dh; a.dw = bwd ? c.d_weight : nullptr; a.ld_dw = c.ld_dw; a.db = bwd ? c.d_bias : nullptr;
  char* w = reinterpret_cast<char*>(c.ws);
  a.count = (int*)(w + P.o_count); a.some = (int*)(w + P.o_some); a.rowmap = (int*)(w + P.o_rowmap); a.inv = (int*)(w + P.o_inv);
  a.tgt_idx0 = (int*)(w + P.o_ti0); a.tgt_q0 = (float*)(w + P.o_tq0); a.tgt_idx = (int*)(w + P.o_ti); a.tgt_q = (float*)(w + P.o_tq);
  a.hc = (bf16_t*)(w + P.o_hc); a.hct = (bf16_t*)(w + P.o_hct); a.part = (float2*)(w + P.o_part); a.zt = (float*)(w + P.o_zt); a.tgt_z = (float*)(w + P.o_tz); 
  a.lse2 = (float*)(w + P.o_lse2); a.g = (float*)(w + P.o_g); a.gr = bwd ? (float*)(w + P.o_gr) : nullptr;
  a.dl = (bf16_t*)(w + P.o_dl); a.dlt = (bf16_t*)(w + P.o_dlt); a.wt = P.o_wt >= 0 && c.d_hidden ? (bf16_t*)(w + P.o_wt) : nullptr; a.slab = (float*)(w + P.o_slab); a.wslab = (float*)(w + P.o_wslab); a.lw = P.lw; a.dbp = (float*)(w + P.o_dbp); a.vpad = P.vpad;
  a.arrived = (unsigned*)(a.count + 1); a.sums = (double*)(w + P.o_sums); a.db64 = (unsigned long long*)(w + P.o_db64); a.dbn = (unsigned*)(w + P.o_dbn);
  a.piece = (int)piece;
  int num_cu = 0;
  CACO_TRY_RC(prepare_launch(reinterpret_cast<const void*>(&lse_kernel<Big>), Big::SMEM_WFAR, &num_cu));
  // a power of two of workgroups per XCD, 8 at least (Order)
  int cus = 64;
  while (cus * 2 <= num_cu && cus < MAX_CU) cus *= 2;
  return P.small ? run_loss<Small>(a, P, c.what, cus, st) : run_loss<Big>(a, P, c.what, cus, st);
}

}  // namespace caco
