// Eviction from a latent cache by accumulated attention weight: the account of a step's attention, the selection of the
// rows that stay, and the moves that bring them together. On compact pages (compact.h) and on bf16 ones.
#include <type_traits>

#include "compact.h"

namespace hla {
namespace {

// ---- account -----------------------------------------------------------------------------------------------------
// account[r, j] += sum over the tokens t of request r and the 16 heads h of exp(scale q[t, h] K[r, j] - lse[h, t]), for
// j < ctx[t]. The lse is the caller's: of the whole softmax, which may cover more keys than these. Sums are fp32 and in a
// fixed order: every row's sum is made by one wave.
struct AccountParams {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint8_t* cache;     // compact: page_stride in bytes
  const uint16_t* cache16;  // bf16: page_stride and row_stride in elements
  int64_t page_stride, row_stride;
  int block;
  int64_t num_blocks;
  const int32_t* bt;
  int64_t bt_stride;
  int bt_cols;
  const int32_t* qsl;
  const int32_t* ctx;
  const float* lse;  // [16][T]
  int T;
  float scale;
  float* account;
  int64_t a_st;
  int cols;      // columns of the account
  int per_wg;    // keys per workgroup (single tokens)
  float* partial;  // chunks: [shares][R][cols] sums of the shares of each request's tokens, or null (one share)
};

// K of one tile as the A operand of S^T = K Q^T, and the columns of its steps. Compact pages: step 4i + j of lane (x, g)
// holds columns 32 (4i + g) + 8j .. + 8 of row x; bf16 pages: step s holds columns 32s + 8g .. + 8.
template <int W, bool kCompact>
struct KeyTile {
  KTile<W> c;
  // where the tile of row `row` begins, in bytes (compact) or elements (bf16)
  static __device__ __forceinline__ int64_t place(const AccountParams& a, const int32_t* btr, int row) {
    const int64_t page = clamp_page(btr[row / a.block], a.num_blocks);
    return page * a.page_stride + (row % a.block) / kTile * compact_tile_bytes(W);
  }
  template <bool kOnce>
  __device__ __forceinline__ void load(const AccountParams& a, int64_t at, int x, int g) {
    load_k<W, kOnce>(a.cache + at, x, g, c);
  }
  __device__ __forceinline__ u32x4 operand(int s) const {
    return eight_bf16(c.code[s / 4][s % 4], scale_of(c.scale[s / 16], s / 4 % 4));
  }
  static __device__ __forceinline__ int column(int s, int g) { return 32 * (s / 4 * 4 + g) + 8 * (s % 4); }
};

template <int W>
struct KeyTile<W, false> {
  u32x4 v[W / 32];
  static __device__ __forceinline__ int64_t place(const AccountParams& a, const int32_t* btr, int row) {
    const int64_t page = clamp_page(btr[row / a.block], a.num_blocks);
    return page * a.page_stride + (int64_t)(row % a.block / kTile * kTile) * a.row_stride;
  }
  template <bool kOnce>
  __device__ __forceinline__ void load(const AccountParams& a, int64_t at, int x, int g) {
    const uint16_t* p = a.cache16 + at + (int64_t)x * a.row_stride + 8 * g;
#pragma unroll
    for (int s = 0; s < W / 32; ++s) v[s] = ld_row<kOnce>(p + 32 * s);
  }
  __device__ __forceinline__ u32x4 operand(int s) const { return v[s]; }
  static __device__ __forceinline__ int column(int s, int g) { return 32 * s + 8 * g; }
};

// sum over the 16 lanes of a row (every lane gets it)
__device__ __forceinline__ float row_sum16(float v) {
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x128, 0xf, 0xf, false));  // row_ror:8
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x124, 0xf, 0xf, false));
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x122, 0xf, 0xf, false));
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x121, 0xf, 0xf, false));
  return v;
}

// weight of a score under its softmax's lse (+inf: an empty row, which weighs nothing; the callers drop a NaN or infinite
// score's there)
__device__ __forceinline__ float weight(float s, float scale, float lse) {
  return fast_exp2(__builtin_fmaf(s, scale, -lse) * kLog2e);
}
__device__ __forceinline__ float row_lse(const AccountParams& a, int t, int h) {
  const float v = a.lse[(int64_t)h * a.T + t];
  return v == -INFINITY ? INFINITY : v;
}

// the four keys' weights of a tile summed over the heads: lane h < 4 of group g gets that of key 4g + h
__device__ __forceinline__ float head_sums(int h, const float (&w)[4]) {
  float s[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) s[e] = row_sum16(w[e]);
  return h == 0 ? s[0] : h == 1 ? s[1] : h == 2 ? s[2] : s[3];
}

// Single tokens: Q^T lies in LDS, K streams by, two tiles a step and wave (one where they are large). The sums of the
// workgroup's keys gather in LDS and go to the account at the end: an account read in each step stood behind the loads of the
// next one's rows, and waited for them.
constexpr int kMaxStepKeys = 4096;  // per workgroup

template <int W, bool kCompact>
__global__ __launch_bounds__(256) void account_step_kernel(AccountParams a) {
  using K = KeyTile<W, kCompact>;
  constexpr int STEPS = W / 32, NT = kCompact ? (W <= 512 ? 2 : 1) : (W <= 256 ? 2 : 1), SPAN = 4 * NT * kTile;
  // past the caches as in compact_history_kernel (64 rows of 8160: 33.2 -> 28.1 us; bf16 rows, and narrow ones, gain nothing)
  constexpr bool kOnce = kCompact && W >= 512;
  __shared__ u32x4 q_lds[STEPS][64];
  __shared__ float sum_lds[kMaxStepKeys];
  const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63, h = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cap = (int)min((int64_t)a.bt_cols * a.block, (int64_t)a.cols);
  const int t0 = max(a.qsl[r], 0), t1 = min(a.qsl[r + 1], a.T);
  const int begin = blockIdx.x * a.per_wg;
  const int32_t* btr = a.bt + (int64_t)r * a.bt_stride;
  for (int i = tid; i < a.per_wg; i += 256) sum_lds[i] = 0.f;
  for (int t = t0; t < t1; ++t) {
    const int end = min(min(a.ctx[t], cap), begin + a.per_wg);
    if (begin >= end) continue;  // uniform over the workgroup
    int j = begin + wave * NT * kTile;
    // places of the tiles of all the wave's steps, one per lane; the last step loads nothing (see compact_history_kernel)
    static_assert(kMaxStepKeys <= 64 / NT * SPAN, "a wave's lanes hold the places of all its tiles");
    const int64_t at = K::place(a, btr, min(j + lane / NT * SPAN + lane % NT * kTile, (end - 1) / kTile * kTile));
    const uint32_t at_lo = (uint32_t)at, at_hi = (uint32_t)((uint64_t)at >> 32);
    auto tile = [&](int i) {
      const uint32_t lo = __builtin_amdgcn_readlane(at_lo, i), hi = __builtin_amdgcn_readlane(at_hi, i);
      return (int64_t)(((uint64_t)hi << 32) | lo);
    };
    u32x4 q[STEPS / 4];
    const uint16_t* qp = a.q + (int64_t)t * a.q_st + (int64_t)h * a.q_sh;
#pragma unroll
    for (int s = 0; s < STEPS / 4; ++s) q[s] = ld16(qp + K::column(wave * (STEPS / 4) + s, g));
    const float lse = row_lse(a, t, h);
    K k[NT];
#pragma unroll
    for (int x = 0; x < NT; ++x) k[x].template load<kOnce>(a, tile(x), h, g);
    __syncthreads();  // (the reads of the token before)
#pragma unroll
    for (int s = 0; s < STEPS / 4; ++s) q_lds[wave * (STEPS / 4) + s][lane] = q[s];
    __syncthreads();
    int step = 1;
    auto one_step = [&](auto last) {
      floatx4 s[NT];
#pragma unroll
      for (int x = 0; x < NT; ++x) s[x] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const u32x4 qi = q_lds[i][lane];
#pragma unroll
        for (int x = 0; x < NT; ++x) s[x] = mfma16x16x32(k[x].operand(i), qi, s[x]);
      }
      if constexpr (!last.value) {
#pragma unroll
        for (int x = 0; x < NT; ++x) k[x].template load<kOnce>(a, tile(step * NT + x), h, g);
      }
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = lse == INFINITY ? 0.f : weight(s[x][e], a.scale, lse);
        const float sum = head_sums(h, w);
        const int key = j + x * kTile + 4 * g + h;
        if (h < 4 && key < end) sum_lds[key - begin] += sum;  // (the same lane for every token)
      }
    };
    for (; j + SPAN < end; j += SPAN, ++step) one_step(std::false_type{});
    if (j < end) one_step(std::true_type{});
  }
  __syncthreads();
  float* row = a.account + (int64_t)r * a.a_st;
  for (int i = tid; i < a.per_wg && begin + i < cap; i += 256)
    if (sum_lds[i] != 0.f) row[begin + i] += sum_lds[i];  // (rows behind the request stay untouched; NaN passes)
}

// Prompt chunks: a product of all rows with all queries of the request, whose epilogue takes the weights and sums them over the
// tokens in registers. A wave keeps 64 rows of K (32 at W = 1024) as bf16 operands; the queries stream by through LDS in
// operand order, two tokens ahead, so that a KB of LDS feeds four products. Reads from LDS go four steps ahead of their
// products (the next token's first ones ahead of this one's last), and a token's weights are worked out in the shadow of the
// next one's products. 4 x 512 tokens over 8160 rows at width 512: 392 us with 32 rows a wave (LDS at its full rate), 343
// with 64 (every read waited for), 269 with reads ahead, 260 with the next token's, 231 with the weights between the products:
// 1.19 PFLOP/s, what a large library product reaches. One tile in four of K lies in accumulation registers: all of it
// and its neighbours do not fit the 256 others.
// The tokens of a request may be shared out over blockIdx.z.
template <int W, bool kCompact>
__global__ __launch_bounds__(256, W <= 256 ? 2 : 1) void account_chunk_kernel(AccountParams a) {
  using K = KeyTile<W, kCompact>;
  constexpr int NT = W <= 512 ? 4 : 2, STEPS = W / 32, MINE = STEPS / 4;  // steps of Q that a wave stages
  constexpr int GROUP = STEPS >= 16 ? 4 : 2, PARTS = STEPS / GROUP;
  __shared__ u32x4 q_lds[3][STEPS][64];
  __shared__ int n_lds[4];
  const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63, h = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cap = (int)min((int64_t)a.bt_cols * a.block, (int64_t)a.cols);
  int t0 = max(a.qsl[r], 0), t1 = min(a.qsl[r + 1], a.T);
  const int share = (max(t1 - t0, 0) + gridDim.z - 1) / gridDim.z;
  t0 += blockIdx.z * share;
  t1 = min(t1, t0 + share);
  int most = 0;
  for (int t = t0 + tid; t < t1; t += 256) most = max(most, a.ctx[t]);
  most = wave_max(most);
  if (lane == 0) n_lds[wave] = most;
  __syncthreads();
  most = min(max(max(n_lds[0], n_lds[1]), max(n_lds[2], n_lds[3])), cap);
  const int wg0 = blockIdx.x * (4 * NT * kTile), key0 = wg0 + wave * (NT * kTile);
  float* row = a.partial ? a.partial + ((int64_t)blockIdx.z * gridDim.y + r) * a.cols : a.account + (int64_t)r * a.a_st;
  float w[NT][4];
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e) w[x][e] = 0.f;
  if (wg0 < most) {  // uniform over the workgroup
    u32x4 k[NT][STEPS];
    {
      const int32_t* btr = a.bt + (int64_t)r * a.bt_stride;
      K tile[NT];
#pragma unroll
      for (int x = 0; x < NT; ++x)
        tile[x].template load<false>(a, K::place(a, btr, min(key0 + x * kTile, (most - 1) / kTile * kTile)), h, g);
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          k[x][s] = tile[x].operand(s);
          if (W == 512 && x == 3) asm("" : "+a"(k[x][s]));  // (the products read them there)
        }
    }
    floatx4 last[NT];  // scores of the token before
#pragma unroll
    for (int x = 0; x < NT; ++x) last[x] = floatx4{0.f, 0.f, 0.f, 0.f};
    float lse = INFINITY;  // (before the first token: weights of 0)
    int limit = 0;
    auto take = [&](int part) {  // the weights of the token before, one share of them
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((x * 4 + e) * PARTS / (NT * 4) != part) continue;
          const float p = weight(last[x][e], a.scale, lse);
          w[x][e] += x * kTile + e < limit ? p : 0.f;
        }
    };
    auto hold = [&](int part) {  // keeps the share of `take` behind this place
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((x * 4 + e) * PARTS / (NT * 4) == part) {
            float v = last[x][e];
            asm volatile("" : "+v"(v));
            last[x][e] = v;
          }
    };
    auto copy = [&](int t, int slot) {  // this wave's steps of token t's queries
      const uint16_t* qp = a.q + (int64_t)t * a.q_st + (int64_t)h * a.q_sh;
#pragma unroll
      for (int s = 0; s < MINE; ++s) copy16_to_lds_v(qp + K::column(wave * MINE + s, g), q_lds[slot][wave * MINE + s]);
    };
    // Wait for this wave's copies (nothing else is long on its way here), then for everybody's.
    auto arrive = [&]() {
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
      plain_barrier();
    };
    copy(t0, 0);
    arrive();
    copy(min(t0 + 1, t1 - 1), 1);
    u32x4 qa[GROUP], qb[GROUP];
#pragma unroll
    for (int i = 0; i < GROUP; ++i) qa[i] = q_lds[0][i][lane];
    int slot = 0;
    for (int t = t0; t < t1; ++t) {
      const int slot1 = slot == 2 ? 0 : slot + 1;
      const float lse_now = row_lse(a, t, h);
      const int n_now = a.ctx[t];
      floatx4 s[NT];
#pragma unroll
      for (int x = 0; x < NT; ++x) s[x] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        if (part + 1 < PARTS) {
#pragma unroll
          for (int i = 0; i < GROUP; ++i) qb[i] = q_lds[slot][(part + 1) * GROUP + i][lane];
        } else {
          // The next token's queries, ahead of this one's last products: behind the barrier they are whole, and every wave
          // has read the token before this one, whose place the one after the next takes.
          arrive();
          copy(min(t + 2, t1 - 1), slot1 == 2 ? 0 : slot1 + 1);  // (past the end the last one again: no branch here)
#pragma unroll
          for (int i = 0; i < GROUP; ++i) qb[i] = q_lds[slot1][i][lane];  // (behind the last token: unused)
        }
        // The reads, then the products with the last token's weights in their shadow: a product keeps the matrix unit for the
        // time of four vector instructions. The scheduler would put all of the weights ahead of the products otherwise.
        __builtin_amdgcn_sched_barrier(0);
        hold(part);
#pragma unroll
        for (int i = 0; i < GROUP; ++i)
#pragma unroll
          for (int x = 0; x < NT; ++x) s[x] = mfma16x16x32(k[x][part * GROUP + i], qa[i], s[x]);
        take(part);
#pragma unroll
        for (int i = 0; i < GROUP * NT; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // one product,
          __builtin_amdgcn_sched_group_barrier(0x402, 2, 0);  // two vector instructions
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < GROUP; ++i) qa[i] = qb[i];
      }
      lse = lse_now;
      limit = lse_now == INFINITY ? 0 : min(n_now, cap) - key0 - 4 * g;
#pragma unroll
      for (int x = 0; x < NT; ++x) last[x] = s[x];
      slot = slot1;
    }
#pragma unroll
    for (int part = 0; part < PARTS; ++part) take(part);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 15));  // no copy into LDS outlives the workgroup
  }
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    const float sum = head_sums(h, w[x]);
    const int key = key0 + x * kTile + 4 * g + h;
    if (h < 4 && key < (a.partial ? a.cols : most)) {
      if (a.partial) row[key] = sum;
      else row[key] += sum;
    }
  }
}

// account += the shares' sums, in their order (rows that nothing was given keep their bits)
__global__ __launch_bounds__(256) void account_reduce_kernel(const float* partial, int shares, int R, int cols,
                                                             float* account, int64_t a_st) {
  const int j = blockIdx.x * 256 + threadIdx.x, r = blockIdx.y;
  if (j >= cols) return;
  float s = 0.f;
  for (int z = 0; z < shares; ++z) s += partial[((int64_t)z * R + r) * cols + j];
  if (s != 0.f) account[(int64_t)r * a_st + j] += s;
}

// ---- selection -----------------------------------------------------------------------------------------------------
// Of a request's n rows the best `budget` stay: first the rows whose position is at least protect_from, then by account,
// descending, ties to the earlier row (NaN ranks last). One workgroup of 16 waves per request; wave w holds rows
// [w, w + 1) * 64 * items, lane by lane, so that every rank in row order is a sum of ballots. The threshold (the account of
// the last row to stay) is found a byte at a time from counts in LDS. Bound by latency: a chain of loads, four rounds of
// counting with two barriers each, three sums over the workgroup, and the gather of what fills the holes: 7.4 us for 3
// requests of 1,000 rows, 15 for 64 of 8,000 (two bits a round: 25 and 44).
struct SelectParams {
  const float* account;
  int64_t a_st;
  const int32_t* positions;
  int64_t p_st;
  const int32_t* lengths;
  int budget;
  const int32_t* budgets;  // per request, or null
  const int32_t* protect_from;
  int cols;
  int32_t* out_lengths;
  float* out_account;      // [R][cols]
  int32_t* out_positions;  // [R][cols]
  int32_t* source;         // [R][cols / 2]
  int32_t* target;
};

constexpr int kSelWaves = 16, kSelThreads = 64 * kSelWaves;

// Order of accounts as an unsigned number above 0: NaN 1, then -inf to +inf, the zeros alike
__device__ __forceinline__ uint32_t rank_key(float a) {
  if (a != a) return 1u;
  const uint32_t u = __float_as_uint(a + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int below(uint64_t mask, int lane) {
  return __popcll(mask & ((1ull << lane) - 1));
}

// f(i) for the rows i of a lane
template <int kItems, class F>
__device__ __forceinline__ void each_row(int items, F f) {
  if constexpr (kItems > 0) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) f(i);
  } else {
    for (int i = 0; i < items; ++i) f(i);
  }
}

// kItems > 0: the rank keys of kItems rows per lane stay in registers; kLdsKeys: up to kMaxLdsItems in LDS; kReadKeys: any
// number, made anew in every pass
constexpr int kLdsKeys = 0, kReadKeys = -1, kMaxLdsItems = 32;
// copies of the counts, one per lane modulo this: accounts share their leading byte (sign and exponent), and lanes that
// count in one word wait for each other
constexpr int kCopies = 8;

template <int kItems>
__global__ __launch_bounds__(kSelThreads) void select_rows_kernel(SelectParams a) {
  __shared__ int sums[2][kSelWaves][2];
  __shared__ uint32_t keys_lds[kItems == kLdsKeys ? kMaxLdsItems * kSelThreads : 1];
  __shared__ __attribute__((aligned(16))) int counts[256 * kCopies];
  __shared__ __attribute__((aligned(16))) int bins[256];
  __shared__ int fill_lds[kItems > 0 ? kItems * kSelThreads / 2 : 1];  // sources, for the holes
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float* __restrict__ acc = a.account + (int64_t)r * a.a_st;
  const int32_t* __restrict__ pos = a.positions + (int64_t)r * a.p_st;
  const int n = min(max(a.lengths[r], 0), a.cols);
  const int b = min(n, max(a.budgets ? a.budgets[r] : a.budget, 0));
  const int first = a.protect_from[r];
  const int items = kItems > 0 ? kItems : (a.cols + kSelThreads - 1) / kSelThreads;
  const int j0 = wave * items * 64 + lane;
  const bool all = n == b;  // nothing goes

  int turn = 0;  // `sums` alternates between two buffers: one barrier per total
  // sums of x and y (uniform over a wave) over all waves, and over the waves before this one
  auto total = [&](int x, int y, int& before_x, int& before_y) {
    if (lane == 0) {
      sums[turn][wave][0] = x;
      sums[turn][wave][1] = y;
    }
    __syncthreads();
    int sx = 0, sy = 0;
    before_x = before_y = 0;
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) {
      const int ux = sums[turn][w][0], uy = sums[turn][w][1];
      before_x += w < wave ? ux : 0;
      before_y += w < wave ? uy : 0;
      sx += ux;
      sy += uy;
    }
    turn ^= 1;
    return make_int2(sx, sy);
  };
  int skip_x, skip_y;

  uint32_t reg[kItems > 0 ? kItems : 1];
  uint64_t guarded = 0;  // bit i: row i of this lane is protected (not kReadKeys)
  bool among_protected = false;
  int need = 0;
  if (!all) {
    for (int i = tid; i < 256 * kCopies; i += kSelThreads) counts[i] = 0;
    int here = 0;
    if constexpr (kItems > 0) {
      float w[kItems];
      int p[kItems];
#pragma unroll
      for (int i = 0; i < kItems; ++i) {  // (all loads on their way before the first is used)
        const int j = min(j0 + 64 * i, n - 1);
        w[i] = acc[j];
        p[i] = pos[j];
      }
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const bool in = j0 + 64 * i < n, prot = in && p[i] >= first;
        reg[i] = in ? rank_key(w[i]) : 0u;
        guarded |= (uint64_t)prot << i;
        here += __popcll(__ballot(prot));
      }
    } else {
      each_row<kItems>(items, [&](int i) {
        const int j = j0 + 64 * i;
        const bool prot = j < n && pos[j] >= first;
        here += __popcll(__ballot(prot));
        if constexpr (kItems == kLdsKeys) {
          guarded |= (uint64_t)prot << i;
          keys_lds[i * kSelThreads + tid] = j < n ? rank_key(acc[j]) : 0u;
        }
      });
    }
    const int np = total(here, 0, skip_x, skip_y).x;
    // candidates: the unprotected rows (the protected ones all stay), or the protected ones where these are too many
    among_protected = np >= b;
    need = among_protected ? b : b - np;
    if constexpr (kItems > 0) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) reg[i] = (((guarded >> i) & 1) != 0) == among_protected ? reg[i] : 0u;
    }
  }
  // key of row i as a candidate (0: it is none), and whether it stays anyhow
  auto row_of = [&](int i, bool& anyhow) -> uint32_t {
    const int j = j0 + 64 * i;
    if (all) {
      anyhow = j < n;
      return 0u;
    }
    bool prot;
    if constexpr (kItems == kReadKeys) prot = j < n && pos[j] >= first;
    else prot = (guarded >> i) & 1;
    anyhow = prot && !among_protected;
    if constexpr (kItems > 0) return reg[i];
    else if constexpr (kItems == kLdsKeys) return prot == among_protected ? keys_lds[i * kSelThreads + tid] : 0u;
    else return j < n && prot == among_protected ? rank_key(acc[j]) : 0u;
  };

  uint32_t threshold = 0xffffffffu;  // candidates above it stay, and the first `ties` at it (no key is that high)
  int ties = 0;
  if (need > 0) {
    uint32_t found = 0;  // the leading bytes of the need-th largest key
    int left = need;     // its rank among the candidates that share them
    bool exact = false;
    for (int shift = 24; shift >= 0 && !exact; shift -= 8) {
      each_row<kItems>(items, [&](int i) {
        bool anyhow;
        const uint32_t key = row_of(i, anyhow);
        if (key != 0 && (shift == 24 || key >> (shift + 8) == found))
          atomicAdd(&counts[((key >> shift) & 255u) * kCopies + lane % kCopies], 1);
      });
      __syncthreads();
      if (tid < 256) {  // the copies together, and clear for the next byte
        int4* c = reinterpret_cast<int4*>(counts + tid * kCopies);
        const int4 u = c[0], v = c[1];
        c[0] = c[1] = make_int4(0, 0, 0, 0);
        bins[tid] = ((u.x + u.y) + (u.z + u.w)) + ((v.x + v.y) + (v.z + v.w));
      }
      __syncthreads();
      // every wave: lane l looks at bins 255 - 4l and the three below
      const int4 q = reinterpret_cast<const int4*>(bins)[63 - lane];
      const int upto = wave_scan((q.x + q.y) + (q.z + q.w));
      int above = upto - ((q.x + q.y) + (q.z + q.w));
      const uint64_t hit = __ballot(upto >= left);  // (not empty: a candidate of that rank is there)
      const int owner = __ffsll((unsigned long long)hit) - 1;
      int bin = 255 - 4 * lane, size = q.w;
      if (above + size < left) { above += size; size = q.z; --bin; }
      if (above + size < left) { above += size; size = q.y; --bin; }
      if (above + size < left) { above += size; size = q.x; --bin; }
      left -= __builtin_amdgcn_readlane(above, owner);
      found = (found << 8) | (uint32_t)__builtin_amdgcn_readlane(bin, owner);
      if (__builtin_amdgcn_readlane(size, owner) == left) {  // all of them stay
        exact = true;
        // every candidate from this bin on; the lowest one holds NaN and -inf, and no candidate's key is 0
        threshold = max(found << shift, 1u) - 1;
      }
    }
    if (!exact) {
      threshold = found;
      ties = left;
    }
  }

  // ranks in row order: the ties before this wave's rows, then holes (rows below b that go) and extras (rows behind that stay)
  int ties0 = 0;
  if (ties > 0) {
    int here = 0;
    each_row<kItems>(items, [&](int i) {
      bool anyhow;
      here += __popcll(__ballot(row_of(i, anyhow) == threshold));
    });
    total(here, 0, ties0, skip_y);
  }
  int run;             // ties so far
  uint64_t stays = 0;  // bit i: row i of this lane stays (not kReadKeys)
  auto decide = [&](int i) {
    bool anyhow;
    const uint32_t key = row_of(i, anyhow);
    const uint64_t at = ties > 0 ? __ballot(key == threshold) : 0;
    const bool tie = ties > 0 && key == threshold && run + below(at, lane) < ties;
    run += __popcll(at);
    return anyhow || key > threshold || tie;
  };
  int holes = 0, extras = 0;
  run = ties0;
  each_row<kItems>(items, [&](int i) {
    const int j = j0 + 64 * i;
    const bool stay = decide(i);
    if constexpr (kItems != kReadKeys) stays |= (uint64_t)stay << i;
    holes += __popcll(__ballot(!stay && j < b));
    extras += __popcll(__ballot(stay && j >= b));
  });
  auto stay_of = [&](int i) {
    if constexpr (kItems == kReadKeys) return decide(i);
    else return ((stays >> i) & 1) != 0;
  };
  int hole0, extra0;
  const int moves = total(holes, extras, hole0, extra0).x;
  const int half = a.cols / 2;
  int32_t* source = a.source + (int64_t)r * half;
  int32_t* target = a.target + (int64_t)r * half;
  run = ties0;
  holes = hole0;
  extras = extra0;
  each_row<kItems>(items, [&](int i) {
    const int j = j0 + 64 * i;
    const bool stay = stay_of(i);
    const uint64_t hm = __ballot(!stay && j < b), em = __ballot(stay && j >= b);
    if (!stay && j < b) target[holes + below(hm, lane)] = j;
    if (stay && j >= b) {
      const int at = extras + below(em, lane);
      source[at] = j;
      if constexpr (kItems > 0) fill_lds[at] = j;
    }
    holes += __popcll(hm);
    extras += __popcll(em);
  });
  for (int i = moves + tid; i < half; i += kSelThreads) source[i] = target[i] = -1;
  if (tid == 0) a.out_lengths[r] = b;
  __syncthreads();  // the lists are whole
  run = ties0;
  holes = hole0;
  // where the rows of the new order come from, eight rows of a lane at a time
  for (int i0 = 0; i0 < items; i0 += 8) {
    int from[8];
    float w[8];
    int32_t p[8];
    each_row<8>(8, [&](int e) {
      const int i = i0 + e, j = j0 + 64 * i;
      from[e] = 0;
      if (i >= items) return;  // uniform
      const bool stay = stay_of(i);
      const uint64_t hm = __ballot(!stay && j < b);
      if (j < b) {
        if (stay) from[e] = j;
        else if constexpr (kItems > 0) from[e] = fill_lds[holes + below(hm, lane)];
        else from[e] = source[holes + below(hm, lane)];
      }
      holes += __popcll(hm);
    });
    if (n > 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = acc[from[e]];
        p[e] = pos[from[e]];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = j0 + 64 * (i0 + e);
      if (i0 + e < items && j < a.cols) {
        a.out_account[(int64_t)r * a.cols + j] = j < b ? w[e] : 0.f;
        a.out_positions[(int64_t)r * a.cols + j] = j < b ? p[e] : -1;
      }
    }
  }
}

// ---- moves -----------------------------------------------------------------------------------------------------------
// Row source[r, i] of request r over row target[r, i], for every pair that is not -1. A target lies below the request's new
// length and a source behind it, so no pair touches another's rows.
struct MoveParams {
  uint8_t* cache;
  int64_t page_stride, row_stride;  // bytes (row_stride: bf16 pages)
  int block;
  int64_t num_blocks;
  const int32_t* bt;
  int64_t bt_stride;
  int bt_cols;
  const int32_t* source;
  const int32_t* target;
  int64_t list_st;
  int count;
};

constexpr int kMoveRows = 16;  // moves per wave

// The moves of a wave in pieces of kBytes, kPer of them a row: piece u of row x of a tile lies at(x, u) behind it. Pieces of
// the wave's rows lie lane behind lane, so an instruction moves as many rows as have room in it.
template <int kBytes> struct PieceOf { typedef u32x4 T; };
template <> struct PieceOf<8> { typedef u32x2 T; };
template <> struct PieceOf<4> { typedef uint32_t T; };
template <> struct PieceOf<1> { typedef uint8_t T; };

template <int kBytes, int kPer, class At, int kRows = kMoveRows>
struct MovePieces {
  static constexpr int ITEMS = kRows * kPer, STEPS = (ITEMS + 63) / 64;
  typedef typename PieceOf<kBytes>::T T;
  T v[STEPS];
  // address of item s * 64 + lane of the moves from number `first` on (targets: from kMoveRows on)
  static __device__ __forceinline__ uint8_t* address(uint8_t* cache, uint32_t lo, uint32_t hi, int first, int s, int lane) {
    const int item = min(s * 64 + lane, ITEMS - 1), row = first + item / kPer;
    const uint32_t l = __shfl(lo, row), h = __shfl(hi, row);
    return cache + (int64_t)(((uint64_t)(h & 0x0fffffffu) << 32) | l) + At::at((int)(h >> 28), item % kPer);
  }
  __device__ __forceinline__ void load(uint8_t* cache, uint32_t lo, uint32_t hi, int lane, int first = 0) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) v[s] = *reinterpret_cast<const T*>(address(cache, lo, hi, first, s, lane));
  }
  __device__ __forceinline__ void store(uint8_t* cache, uint32_t lo, uint32_t hi, int lane, uint32_t valid,
                                        int first = 0) const {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      uint8_t* p = address(cache, lo, hi, kMoveRows + first, s, lane);
      const int item = s * 64 + lane;
      if (item < ITEMS && ((valid >> (first + item / kPer)) & 1)) {
        // rows past the caches; scales, many rows' to a line, through them
        if constexpr (kBytes == 16) __builtin_nontemporal_store(v[s], reinterpret_cast<T*>(p));
        else *reinterpret_cast<T*>(p) = v[s];
      }
    }
  }
};

template <int W> struct AtValues {  // compact: 16-byte pieces of K, then of V
  static __device__ __forceinline__ int at(int x, int u) {
    return u < W / 32 ? k_code_at(x, u) : v_code_at(W, x, 16 * (u - W / 32));
  }
};
template <int W> struct AtKeyScales {  // a row's K scales lie side by side: in pieces of up to 16 bytes
  static __device__ __forceinline__ int at(int x, int u) { return 16 * W + x * (W / 32) + 16 * u; }
};
template <int W> struct AtValueScales {
  static __device__ __forceinline__ int at(int x, int u) { return v_scale_at(W, x, u); }
};
struct AtRow {  // bf16
  static __device__ __forceinline__ int at(int, int u) { return 16 * u; }
};

// One wave takes 16 moves. Its lanes first work out where the 16 sources and 16 targets begin, together, and then hand these
// places to the lanes that move the pieces. 121,000 rows of 544 bytes (their pieces fill half of many lines: 200 MB in pieces of 64
// bytes, both ways) out of a cold cache take 40 us, 5.0 TB/s; 49 with ordinary stores, 41 with those of the scales past the
// caches too. 30,000 bf16 rows of 1 KB: 12.5, and 17.6 with ordinary ones.
template <int W, bool kCompact>
__global__ __launch_bounds__(256) void move_rows_kernel(MoveParams a) {
  const int r = blockIdx.y, lane = threadIdx.x & 63;
  const int first = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kMoveRows;
  if (first >= a.count) return;
  int64_t off = 0;  // of the tile (compact) or the row (bf16)
  int x = 0;        // row in the tile
  bool ok = false;
  if (lane < 2 * kMoveRows) {
    const int i = first + lane % kMoveRows;
    const int32_t* list = (lane < kMoveRows ? a.source : a.target) + (int64_t)r * a.list_st;
    const int row = i < a.count ? list[i] : -1;
    if (row >= 0 && row < (int64_t)a.bt_cols * a.block) {
      const int64_t page = a.bt[(int64_t)r * a.bt_stride + row / a.block];
      const int in_page = row % a.block;
      ok = page >= 0 && page < a.num_blocks;
      off = page * a.page_stride + (kCompact ? (in_page >> 4) * compact_tile_bytes(W) : in_page * a.row_stride);
      x = in_page & 15;
    }
  }
  const uint32_t both = (uint32_t)__ballot(ok);
  const uint32_t valid = both & (both >> kMoveRows) & ((1u << kMoveRows) - 1);
  if (valid == 0) return;  // uniform over the wave; there is no barrier
  // (a pair that is skipped reads the first valid one's source, and writes nothing: loads stand under no condition)
  uint32_t lo = (uint32_t)off, hi = (uint32_t)((uint64_t)off >> 32) | ((uint32_t)x << 28);  // (offsets below 2^60)
  const int some = __ffs((int)valid) - 1;
  const uint32_t some_lo = __builtin_amdgcn_readlane(lo, some), some_hi = __builtin_amdgcn_readlane(hi, some);
  if (!((valid >> (lane % kMoveRows)) & 1)) {
    lo = some_lo;
    hi = some_hi;
  }
  if constexpr (kCompact) {
    constexpr int KB = W >= 512 ? 16 : W / 32;
    MovePieces<16, W / 16, AtValues<W>> values;
    MovePieces<KB, W / 32 / KB, AtKeyScales<W>> key_scales;
    MovePieces<1, W / 32, AtValueScales<W>> value_scales;
    values.load(a.cache, lo, hi, lane);
    key_scales.load(a.cache, lo, hi, lane);
    value_scales.load(a.cache, lo, hi, lane);
    values.store(a.cache, lo, hi, lane, valid);
    key_scales.store(a.cache, lo, hi, lane, valid);
    value_scales.store(a.cache, lo, hi, lane, valid);
  } else {
    constexpr int ROWS = W <= 256 ? kMoveRows : W == 512 ? 8 : 4;  // 16 pieces of a lane in flight
#pragma unroll 1
    for (int k = 0; k < kMoveRows; k += ROWS) {
      MovePieces<16, W / 4, AtRow, ROWS> rows;
      rows.load(a.cache, lo, hi, lane, k);
      rows.store(a.cache, lo, hi, lane, valid, k);
    }
  }
}

template <int W, bool kCompact>
void launch_account(const AccountParams& p, int R, int shares, bool chunks, hipStream_t st) {
  const int keys = min((int64_t)p.bt_cols * p.block, (int64_t)p.cols);
  if (!chunks) {
    hipLaunchKernelGGL((account_step_kernel<W, kCompact>), dim3((unsigned)((keys + p.per_wg - 1) / p.per_wg), (unsigned)R),
                       dim3(256), 0, st, p);
    return;
  }
  constexpr int per = 4 * (W <= 512 ? 4 : 2) * kTile;
  hipLaunchKernelGGL((account_chunk_kernel<W, kCompact>),
                     dim3((unsigned)(((p.partial ? p.cols : keys) + per - 1) / per), (unsigned)R, (unsigned)shares),
                     dim3(256), 0, st, p);
  if (p.partial)
    hipLaunchKernelGGL(account_reduce_kernel, dim3((unsigned)((p.cols + 255) / 256), (unsigned)R), dim3(256), 0, st,
                       p.partial, shares, R, p.cols, p.account, p.a_st);
}

template <int W, bool kCompact>
void launch_move(const MoveParams& p, int R, hipStream_t st) {
  constexpr int rows = 4 * kMoveRows;
  hipLaunchKernelGGL((move_rows_kernel<W, kCompact>), dim3((unsigned)((p.count + rows - 1) / rows), (unsigned)R),
                     dim3(256), 0, st, p);
}

int check_pages16(const char* what, int width, const void* cache, int64_t page_stride, int64_t row_stride, int block,
                  int64_t num_blocks) {
  HLA_REQUIRE(known_width(width), HLA_S6_EUNSUPPORTED, "%s: latent width %d not in {128, 256, 512, 1024}", what, width);
  HLA_REQUIRE(block > 0 && block % kTile == 0, HLA_S6_EUNSUPPORTED, "%s: block size %d is not a positive multiple of 16",
              what, block);
  HLA_REQUIRE(num_blocks >= 1, HLA_S6_EINVAL, "%s: empty cache", what);
  HLA_REQUIRE(cache && aligned(cache, 16) && page_stride % 8 == 0 && row_stride % 8 == 0, HLA_S6_EINVAL,
              "%s: cache rows must be 16-byte aligned (strides multiple of 8 elements)", what);
  return HLA_S6_OK;
}

}  // namespace
}  // namespace hla

extern "C" int hla_s6_attention_weights(const void* q, int32_t num_tokens, int32_t num_heads, int32_t width, int64_t q_st,
                                        int64_t q_sh, const void* cache, int32_t compact, int64_t page_stride,
                                        int64_t row_stride, int32_t block_size, int64_t num_blocks,
                                        const int32_t* block_table, int64_t bt_stride, int32_t bt_cols,
                                        const int32_t* query_start_loc, int32_t num_reqs, const int32_t* ctx,
                                        const float* lse, float scale, float* account, int64_t a_st, int32_t cols,
                                        int32_t keys_per_wg, int32_t shares, float* workspace, int64_t workspace_floats,
                                        void* stream) {
  using namespace hla;
  HLA_REQUIRE(num_tokens >= 0 && num_reqs >= 0 && num_reqs <= 65535 && bt_cols >= 0 && cols >= 0, HLA_S6_EINVAL,
              "attention_weights: bad token count, request count (0..65535) or table width");
  HLA_REQUIRE(num_heads == kHeads, HLA_S6_EUNSUPPORTED, "attention_weights: %d query heads (the kernel is built for 16)",
              num_heads);
  int rc = compact ? check_cache("attention_weights", width, cache, page_stride, block_size, num_blocks)
                   : check_pages16("attention_weights", width, cache, page_stride, row_stride, block_size, num_blocks);
  if (rc != HLA_S6_OK || num_tokens == 0 || num_reqs == 0 || cols == 0 || bt_cols == 0) return rc;
  HLA_REQUIRE(q && block_table && query_start_loc && ctx && lse && account, HLA_S6_EINVAL,
              "attention_weights: null pointer argument");
  HLA_REQUIRE(aligned(q, 16) && q_st % 8 == 0 && q_sh % 8 == 0, HLA_S6_EINVAL,
              "attention_weights: q needs 16-byte aligned rows (unit last stride, strides multiple of 8)");
  HLA_REQUIRE(a_st >= cols, HLA_S6_EINVAL, "attention_weights: account rows overlap");
  HLA_REQUIRE(shares >= 0 && shares <= 64, HLA_S6_EINVAL, "attention_weights: shares must be in [0, 64]");
  HLA_REQUIRE(shares > 0 || (keys_per_wg > 0 && keys_per_wg % 64 == 0 && keys_per_wg <= kMaxStepKeys), HLA_S6_EINVAL,
              "attention_weights: keys per workgroup must be a positive multiple of 64, at most %d", kMaxStepKeys);
  if (shares > 1) {
    const int64_t need = (int64_t)shares * num_reqs * cols;
    HLA_REQUIRE(workspace && workspace_floats >= need, HLA_S6_EWORKSPACE,
                "attention_weights: workspace needs %lld floats, has %lld", (long long)need, (long long)workspace_floats);
  }
  AccountParams p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.cache = static_cast<const uint8_t*>(cache);
  p.cache16 = static_cast<const uint16_t*>(cache);
  p.page_stride = page_stride;
  p.row_stride = row_stride;
  p.block = block_size;
  p.num_blocks = num_blocks;
  p.bt = block_table;
  p.bt_stride = bt_stride;
  p.bt_cols = bt_cols;
  p.qsl = query_start_loc;
  p.ctx = ctx;
  p.lse = lse;
  p.T = num_tokens;
  p.scale = scale;
  p.account = account;
  p.a_st = a_st;
  p.cols = cols;
  p.per_wg = keys_per_wg;
  p.partial = shares > 1 ? workspace : nullptr;
  const hipStream_t st = as_stream(stream);
  const bool chunks = shares > 0;
#define HLA_ACCOUNT(W)                                                      \
  compact ? launch_account<W, true>(p, num_reqs, shares, chunks, st)        \
          : launch_account<W, false>(p, num_reqs, shares, chunks, st)
  switch (width) {
    case 128: HLA_ACCOUNT(128); break;
    case 256: HLA_ACCOUNT(256); break;
    case 512: HLA_ACCOUNT(512); break;
    default: HLA_ACCOUNT(1024); break;
  }
#undef HLA_ACCOUNT
  return check_launch("attention_weights");
}

extern "C" int hla_s6_select_rows(const float* account, int64_t a_st, const int32_t* positions, int64_t p_st,
                                  const int32_t* lengths, int32_t num_reqs, int32_t cols, int32_t budget,
                                  const int32_t* budgets, const int32_t* protect_from, int32_t* out_lengths,
                                  float* out_account, int32_t* out_positions, int32_t* source, int32_t* target,
                                  void* stream) {
  using namespace hla;
  HLA_REQUIRE(num_reqs >= 0 && cols >= 0 && (budgets || budget >= 0), HLA_S6_EINVAL,
              "select_rows: bad request count, row count or budget");
  if (num_reqs == 0) return HLA_S6_OK;
  HLA_REQUIRE(lengths && protect_from && out_lengths, HLA_S6_EINVAL, "select_rows: null pointer argument");
  HLA_REQUIRE(cols == 0 || (account && positions && out_account && out_positions), HLA_S6_EINVAL,
              "select_rows: null pointer argument");
  HLA_REQUIRE(cols < 2 || (source && target), HLA_S6_EINVAL, "select_rows: null list");
  HLA_REQUIRE(a_st >= cols && p_st >= cols, HLA_S6_EINVAL, "select_rows: rows overlap");
  SelectParams p = {account, a_st, positions, p_st, lengths, budget, budgets, protect_from, cols,
                    out_lengths, out_account, out_positions, source, target};
  const hipStream_t st = as_stream(stream);
  const dim3 grid((unsigned)num_reqs), block(kSelThreads);
  const int items = (cols + kSelThreads - 1) / kSelThreads;
  if (items <= 2) hipLaunchKernelGGL(select_rows_kernel<2>, grid, block, 0, st, p);
  else if (items <= 8) hipLaunchKernelGGL(select_rows_kernel<8>, grid, block, 0, st, p);
  else if (items <= kMaxLdsItems) hipLaunchKernelGGL(select_rows_kernel<kLdsKeys>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(select_rows_kernel<kReadKeys>, grid, block, 0, st, p);
  return check_launch("select_rows");
}

extern "C" int hla_s6_move_rows(void* cache, int32_t width, int32_t compact, int64_t page_stride, int64_t row_stride,
                                int32_t block_size, int64_t num_blocks, const int32_t* block_table, int64_t bt_stride,
                                int32_t bt_cols, const int32_t* source, const int32_t* target, int64_t list_st,
                                int32_t count, int32_t num_reqs, void* stream) {
  using namespace hla;
  HLA_REQUIRE(num_reqs >= 0 && num_reqs <= 65535 && count >= 0 && bt_cols >= 0, HLA_S6_EINVAL,
              "move_rows: bad request count (0..65535), list length or table width");
  int rc = compact ? check_cache("move_rows", width, cache, page_stride, block_size, num_blocks)
                   : check_pages16("move_rows", width, cache, page_stride, row_stride, block_size, num_blocks);
  if (rc != HLA_S6_OK || num_reqs == 0 || count == 0 || bt_cols == 0) return rc;
  HLA_REQUIRE(block_table && source && target, HLA_S6_EINVAL, "move_rows: null pointer argument");
  HLA_REQUIRE(list_st >= count, HLA_S6_EINVAL, "move_rows: lists overlap");
  MoveParams p = {static_cast<uint8_t*>(cache), compact ? page_stride : 2 * page_stride, 2 * row_stride, block_size,
                  num_blocks, block_table, bt_stride, bt_cols, source, target, list_st, count};
  const hipStream_t st = as_stream(stream);
#define HLA_MOVE(W) compact ? launch_move<W, true>(p, num_reqs, st) : launch_move<W, false>(p, num_reqs, st)
  switch (width) {
    case 128: HLA_MOVE(128); break;
    case 256: HLA_MOVE(256); break;
    case 512: HLA_MOVE(512); break;
    default: HLA_MOVE(1024); break;
  }
#undef HLA_MOVE
  return check_launch("move_rows");
}
