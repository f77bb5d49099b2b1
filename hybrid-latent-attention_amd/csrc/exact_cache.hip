// Attention of new tokens, single ones and chunks, over a whole exact (per-head K / V) paged cache, and the store into it.
//
// A cache page holds `block` rows of every KV head, [K | V] of 2d values in bf16 or e4m3; G query heads read one KV head.
//   o[t, h] = sum_j softmax_j(scale q[t, h] . K[j]) V[j], j over the rows [max(0, n - window), n) of n = ctx[t].
//
// A workgroup takes a share of the rows of one KV head for up to 16 of its query heads. The rows of all tokens, one token behind
// the other, are cut in shares of equal length: every workgroup has as much to stream, however ragged the lengths are. What a
// share holds of a token is a part, whole tokens are written at once, and exact_join_kernel joins the parts of the others. (With
// rows enough for the device, or short ones, a workgroup takes all rows of a token.) Each wave walks tiles of its own:
//   * a tile's K and V rows come by direct copies into LDS, a KB each, NB - 1 tiles ahead (the stream is what bounds the
//     kernel: 2d values per row and head are read once and meet 4 G d flops); the 16-byte pieces of a row lie swizzled, which
//     spreads both ways of reading them below over the banks;
//   * S^T[keys x 16 heads] = K Q^T on 16x16x32 bf16 products: K is the A operand (a row's pieces as they lie), Q^T stays in
//     registers; heads past the group's are zero columns, whose work is cheaper than the bytes;
//   * softmax in the exp2 domain, fp32, with a running maximum that is raised only when a score exceeds it by 2^8;
//   * O^T[d x 16 heads] += V^T P^T: P^T comes out of the scores' registers as the B operand, V^T is read by the transposing
//     LDS loads. bf16 tiles have 16 keys (16x16x16 products), e4m3 ones 32, in the order of keys that the two halves of the
//     scores have (16x16x32), and e4m3 values become bf16, exactly, on their way into the operands.
// P goes into its product as two bf16 parts, upper half and rounded rest (2^-16 of a weight is left; one part alone would add about
// two thirds of the output's own rounding to it: 0.0024 relative to the 64-bit result, now 0.0017). Up to 8 query heads have their
// rests in the 8 columns that would be zero: the scores of a head are made twice, for free. With more heads, or
// tokens, both parts are keys of one product of twice the keys, V twice in its operand (bf16), or of two products (e4m3).
//
// Large steps of many tokens per request (chunks) put the heads of 16 / G or 32 / G tokens in the columns: 4 x 512 tokens on
// 8160 rows, 16 heads, 370 to 410 us, 320 to 360 TFLOP/s (matrix units 23 %, vector units 53 %, LDS 17 %: two waves per SIMD, each a
// chain of them, on 16 keys at a time; K and V cross the caches once per group).
//
// Single tokens beside chunks (exact_alone_kernel lists them) keep their shares, in a launch behind that of the groups.
//
// Bound by HBM: 64 tokens of 4096 rows and 16 heads (2.1 GB) 320 us, 6.7 TB/s, the vector units at 15 %; a call is its bytes at
// that rate and about 11 us (launch, lengths, table entries, first rows, joining waves, the second launch). Past the caches
// (kOnce) 7 % faster. Two workgroups of four waves per CU, a tile of each wave on its way: three waves, eight, or one workgroup
// with twice the tiles measured the same or slower, so did dealing the heads of a share to one XCD.
#include "common.h"

namespace hla {
namespace {

constexpr int kMaxTile = 16;     // query heads per workgroup
constexpr int kMaxShares = 1024;
constexpr int kCus = 256;
constexpr float kRaise = 8.f;    // log2 by which a score may exceed the running maximum
constexpr int kStep = 64;        // rows that shares are counted in
// steps below which a share is not worth a workgroup of its own (its partial is written and read once more)
constexpr int kMinSteps = 2;

struct ExactCacheParams {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint8_t* cache;
  int64_t page_stride, head_stride, row_stride;  // bytes
  int block;
  int64_t num_blocks;
  const int32_t* bt;
  int64_t bt_stride;
  int bt_cols, bt_count;
  const int64_t* bt_rows;
  const int32_t* ctx;
  int window;
  float scale_log2;
  const float *k_scale, *v_scale;
  int T, H, KH, G, tiles;  // tiles: workgroups of query heads per KV head
  int shares;              // 0: a workgroup takes all rows of a token, or (grouped) of 16 / G or 32 / G tokens; beside groups: see alone
  int grouped;             // workgroups among which the requests of a group are dealt; 0: a token by itself
  bool shared;             // several tokens read the same rows
  float *ws_o, *ws_lse;    // [shares][2][H][D], [shares][2][H]
  int32_t* split;          // [T][2]: first and last share of a token's rows
  int32_t* alone;          // null, or where shares take the tokens alone and groups the others: [1 + T], how many are alone, and which
  uint16_t* out;
  int64_t o_st, o_sh;
  float* lse;  // [H][T]
};

template <int kDim, bool kE4m3, bool kWide>
struct ExactGeo {
  static constexpr int D = kDim;
  static constexpr bool kE4 = kE4m3;
  static constexpr int ES = kE4 ? 1 : 2;
  static constexpr int KEYS = kE4 ? 32 : 16;
  static constexpr int RB = 2 * D * ES;          // bytes of a row, K and V
  static constexpr int CPR = RB / 16;            // pieces of 16 bytes in it
  static constexpr int RPI = 64 / CPR;           // rows per copy of a wave
  static constexpr int NI = KEYS / RPI;          // copies per tile
  static constexpr int TILE = KEYS * RB;         // bytes of a tile
  static constexpr int NB = !kE4 && TILE <= 4096 ? 4 : 2;
  static constexpr int WAVES = (TILE > 8192 ? 2 : 4) * (kWide ? 2 : 1);   // two workgroups per CU by their LDS, or a wide one
  // (two are what LDS holds; said to the compiler, it keeps the sums out of the accumulation registers, from which it would copy
  // them to others and back in every tile)
  static constexpr int kWavesPerSimd = D <= 128 ? 2 : 1;
  static constexpr int BATCH = 64 / KEYS;        // tiles whose row addresses are worked out at a time
  static_assert(NB <= BATCH, "page ids are requested a batch ahead and waited for with the tile before");
};

// Where the pieces of row x of a tile lie: piece c at c ^ swizzle(x). Both reads go over 256 bytes of banks at a time: K by 16
// lanes that take one piece of rows 0..15 (or 16..31), V by 32 lanes that take 32 bytes of rows 0..7 or 8..15 (bf16), or 16
// bytes of rows 0..7 and 16..23, or 8..15 and 24..31 (e4m3). Rows of 128 bytes share the 256.
template <class G>
__device__ __forceinline__ int swizzle(int x) {
  if (!G::kE4) return ((x & 7) << 1) | ((x >> 3) & 1);
  if (G::CPR == 8) return ((x >> 1) & 3) | ((((x >> 3) ^ (x >> 4)) & 1) << 2);
  return (x & 7) | ((((x >> 3) ^ (x >> 4)) & 1) << 3);
}

// Waits that no memory access moves across, in either direction: for the copies into LDS but the N newest, and for LDS reads
template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// 8 e4m3 values (two words) as 8 bf16, exactly
__device__ __forceinline__ u32x4 e4m3_to_bf16(uint32_t lo, uint32_t hi) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  return u32x4{__builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false)),
               __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true)),
               __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false)),
               __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true))};
}

// A weight in two bf16 parts: its upper half, and the rest rounded. The rest of a weight that is not 0 is not 0 and not negative,
// so that an infinity in V stays one.
__device__ __forceinline__ uint32_t upper_halves(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ uint32_t rests(float a, float b, uint32_t upper) {
  return pack2(fmaxf(a - lo_bf(upper), a * 0x1p-40f), fmaxf(b - hi_bf(upper), b * 0x1p-40f));
}

// Rows of a token: [first, n)
__device__ __forceinline__ void token_rows(const ExactCacheParams& a, int t, int& first, int& n) {
  n = (int)min((int64_t)max(a.ctx[t], 0), min((int64_t)a.bt_cols * a.block, (int64_t)INT32_MAX - kStep));
  first = a.window > 0 ? max(0, n - a.window) : 0;
}

// Its row of the table
__device__ __forceinline__ int64_t table_row(const ExactCacheParams& a, int t) {
  return a.bt_rows ? min(max(a.bt_rows[t], (int64_t)0), (int64_t)a.bt_count - 1) : t;
}

// Whether a token has rows and its neighbours none of the same table row
__device__ __forceinline__ bool is_alone(const ExactCacheParams& a, int t) {
  int first, n;
  token_rows(a, t, first, n);
  if (n == 0) return false;
  const int64_t row = table_row(a, t);
  for (int i = max(t - 1, 0); i <= min(t + 1, a.T - 1); ++i) {
    token_rows(a, i, first, n);
    if (i != t && n > 0 && table_row(a, i) == row) return false;
  }
  return true;
}

// The tokens that shares take: all, or (kAlone) those alone
template <bool kAlone>
__device__ __forceinline__ int shared_tokens(const ExactCacheParams& a) { return kAlone ? a.alone[0] : a.T; }
template <bool kAlone>
__device__ __forceinline__ int shared_token(const ExactCacheParams& a, int i) { return kAlone ? a.alone[1 + i] : i; }

// Steps of the rows of the i-th of them
template <bool kAlone>
__device__ __forceinline__ int token_steps(const ExactCacheParams& a, int i) {
  int first, n;
  token_rows(a, shared_token<kAlone>(a, i), first, n);
  return (n - first + kStep - 1) / kStep;
}

// Share k of the steps of all tokens, one token behind the other: a share is ceil(total / shares) of them, kMinSteps at least.
// `left` steps of it (0: none) begin at step `at` of the t-th token, whose first step is the `before`-th of all.
template <bool kAlone>
__device__ __forceinline__ void find_share(const ExactCacheParams& a, int k, int threads, int64_t* sums, int64_t* found, int& t,
                                           int& at, int64_t& left, int64_t& before, int64_t& share) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tokens = shared_tokens<kAlone>(a), seg = (tokens + threads - 1) / threads;
  const int t0 = min(tokens, tid * seg), t1 = min(tokens, t0 + seg);
  int64_t mine = 0;
  for (int i = t0; i < t1; ++i) mine += token_steps<kAlone>(a, i);
  int64_t x = mine;
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  if (lane == 63) sums[wave] = x;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < threads / 64; ++w) {
    if (w < wave) x += sums[w];
    total += sums[w];
  }
  total = uniform64(total);
  share = max((total + a.shares - 1) / a.shares, (int64_t)kMinSteps);
  const int64_t begin = k * share;
  left = min(share, total - begin);
  if (left <= 0) return;
  int64_t base = x - mine;
  if (begin >= base && begin < x)   // one thread's tokens hold it
    for (int i = t0; i < t1; ++i) {
      const int steps = token_steps<kAlone>(a, i);
      if (begin < base + steps) {
        found[0] = i;
        found[1] = base;
        break;
      }
      base += steps;
    }
  __syncthreads();
  t = __builtin_amdgcn_readfirstlane((int)found[0]);
  before = uniform64(found[1]);
  at = (int)(begin - before);
}

// What the 16 columns of the scores are
enum Columns {
  kHeads,    // query heads of a token
  kTwice,    // up to 8 of them, and the same again
  kTokens16, // those of several tokens, which share the rows of a request (the queries of a chunk)
  kTokens32, // the same with 32 columns
};

// kOnce: rows are read by one workgroup and stream past the caches; kAlone: shares of the tokens alone, beside groups of the others
// (a kernel of its own: told apart within one, every step in shares took 0.5 to 3 us longer)
template <class G, bool kOnce, Columns kColumns, bool kAlone = false>
__global__ __launch_bounds__(64 * G::WAVES, G::kWavesPerSimd) void exact_cache_kernel(ExactCacheParams a) {
  constexpr int D = G::D;
  constexpr bool kE4 = G::kE4;
  constexpr int KEYS = G::KEYS, RB = G::RB, CPR = G::CPR, RPI = G::RPI, NI = G::NI, NB = G::NB, WAVES = G::WAVES;
  constexpr int CT = D / 16;       // 16-column tiles of O^T
  constexpr int OS = D + 4;        // LDS row stride of a wave's partial output, in floats
  constexpr bool kTokens = kColumns >= kTokens16;
  constexpr int COLS = kColumns == kTokens32 ? 32 : 16, Y = COLS / 16;   // columns of the scores, 16 per product
  constexpr int kTiles = WAVES * NB * G::TILE, kJoin = WAVES * COLS * OS * 4;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kTiles > kJoin ? kTiles : kJoin];
  __shared__ int64_t offsets[WAVES][64];
  __shared__ int32_t page_ids[WAVES][64];
  __shared__ float stats[WAVES][2][COLS];
  __shared__ int64_t sums[WAVES], found[2];

  const int tid = threadIdx.x, lane = tid & 63, x = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // heads innermost: workgroups dispatched one behind the other read the same rows' heads
  const int parts = a.KH * a.tiles, part = blockIdx.x % parts;
  // a group's requests (runs of tokens with one table row) are dealt to `turns` workgroups
  const int groups = kTokens ? (a.T + COLS / a.G - 1) / (COLS / a.G) : 0;
  const int k = kTokens ? (int)(blockIdx.x / parts) % groups : (int)(blockIdx.x / parts);
  const int turn = kTokens ? (int)(blockIdx.x / parts) / groups : 0;
  const int kh = part / a.tiles, j0 = part % a.tiles * kMaxTile;
  const int heads = min(kMaxTile, a.G - j0), h0 = kh * a.G + j0;
  const uint8_t* cache = a.cache + kh * a.head_stride;
  // column x: head `head` of token k; with several, column 16 y + x: that of token t_group + (16 y + x) / G
  const int group = kTokens ? COLS / a.G : 1, t_group = k * group, t_end = min(a.T, t_group + group);
  int head[Y], token[Y];
#pragma unroll
  for (int y = 0; y < Y; ++y) {
    head[y] = kColumns == kTwice ? x & 7 : kTokens ? (16 * y + x) % a.G : x;
    token[y] = t_group + (kTokens ? (16 * y + x) / a.G : 0);
  }

  // lane i: what token t_group + i reads and sees; a bit for every token that begins a run (tokens alone, where shares take them,
  // are in none)
  int64_t lane_row = 0;
  int lane_first = 0, lane_n = 0;
  uint32_t heads_of_runs = 0;
  if constexpr (kTokens) {
    const int i = t_group + lane;
    bool runs = i < t_end;
    if (runs) {
      lane_row = table_row(a, i);
      token_rows(a, i, lane_first, lane_n);
      if (a.alone && is_alone(a, i)) {
        lane_row = ~(int64_t)i;
        runs = false;
      }
    }
    const int64_t before = __shfl_up(lane_row, 1);
    heads_of_runs = (uint32_t)__ballot(runs && (lane == 0 || lane_row != before));
    for (int skip = 0; skip < turn; ++skip) heads_of_runs &= heads_of_runs - 1;
    if (!heads_of_runs) return;
  }

  int t = kTokens ? t_group + __ffs((int)heads_of_runs) - 1 : t_group, at = 0;
  int64_t left_steps = INT32_MAX, before = 0, share = 1;
  if (a.shares) {
    find_share<kAlone>(a, k, 64 * WAVES, sums, found, t, at, left_steps, before, share);
    if (left_steps <= 0) return;
  }
  for (;;) {   // the tokens of the share, or the requests of the group
    // tokens [t, t_last) of a request: rows [first, n) are seen by any of them, [all_first, all_n) by all that see any
    int first, n, t_last = t + 1, all_first, all_n, my_first[Y] = {}, my_n[Y] = {};
    int64_t row;
    const int my_token = kAlone ? __builtin_amdgcn_readfirstlane(shared_token<kAlone>(a, t)) : t;   // (of one)
    if constexpr (kTokens) {
      const int at_lane = t - t_group;
      row = __shfl(lane_row, at_lane);
      const uint64_t others = __ballot(lane > at_lane && (t_group + lane >= t_end || lane_row != row));
      t_last = min(t_end, t_group + (others ? __ffsll((unsigned long long)others) - 1 : 64));
      const bool sees = lane >= at_lane && t_group + lane < t_last && lane_n > lane_first;
      first = sees ? lane_first : INT32_MAX;
      n = sees ? lane_n : 0;
      all_first = sees ? lane_first : 0;
      all_n = sees ? lane_n : INT32_MAX;
      for (int off = COLS / 2; off > 0; off >>= 1) {   // (a group is in the first COLS lanes)
        first = min(first, __shfl_xor(first, off));
        n = max(n, __shfl_xor(n, off));
        all_first = max(all_first, __shfl_xor(all_first, off));
        all_n = min(all_n, __shfl_xor(all_n, off));
      }
      n = __builtin_amdgcn_readfirstlane(n);
      first = min(__builtin_amdgcn_readfirstlane(first), n);
      all_first = __builtin_amdgcn_readfirstlane(all_first);
      all_n = __builtin_amdgcn_readfirstlane(all_n);
#pragma unroll
      for (int y = 0; y < Y; ++y) {
        const int f = __shfl(lane_first, token[y] - t_group), c = __shfl(lane_n, token[y] - t_group);
        if (token[y] >= t && token[y] < t_last) {
          my_first[y] = f;
          my_n[y] = c;
        }
      }
    } else {
      token_rows(a, my_token, first, n);
      row = table_row(a, my_token);
      all_first = first;
      all_n = n;
    }
    const int steps = (n - first + kStep - 1) / kStep;
    const int taken = (int)min((int64_t)steps - at, left_steps);
    const int lo = first + at * kStep, hi = (int)min((int64_t)n, (int64_t)lo + (int64_t)taken * kStep);
    const bool whole = taken == steps;
    if (a.shares && part == 0 && tid == 0 && at == 0 && steps > 0) {
      a.split[2 * t] = k;
      a.split[2 * t + 1] = (int)((before + steps - 1) / share);
    }
    if (lo >= hi && !a.shares) {
      for (int u = t; u < t_last; ++u) {
        for (int i = tid; i < heads * (D / 8); i += 64 * WAVES)
          st16(a.out + (int64_t)u * a.o_st + (int64_t)(h0 + i / (D / 8)) * a.o_sh + i % (D / 8) * 8, u32x4{0u, 0u, 0u, 0u});
        for (int j = tid; j < heads; j += 64 * WAVES) a.lse[(int64_t)(h0 + j) * a.T + u] = -INFINITY;
      }
    }
    if (lo < hi) {
      const int32_t* btr = a.bt + row * a.bt_stride;
      const int tiles = (hi - lo + KEYS - 1) / KEYS;
      const int mine = tiles > wave ? (tiles - wave + WAVES - 1) / WAVES : 0;  // tiles wave, wave + WAVES, ...

      // row of lane `lane` in the batch of tiles b: rows past the last are the last one again
      auto batch_row = [&](int b) {
        return (int)min((int64_t)hi - 1, lo + ((int64_t)wave + (int64_t)(b * G::BATCH + lane / KEYS) * WAVES) * KEYS + lane % KEYS);
      };
      auto fetch_ids = [&](int b) { copy4_to_lds_v(btr + (uint32_t)batch_row(b) / (uint32_t)a.block, page_ids[wave]); };
      auto work_out = [&](int b) {
        const int64_t page = min(max((int64_t)page_ids[wave][lane], (int64_t)0), a.num_blocks - 1);
        offsets[wave][lane] = page * a.page_stride + (uint32_t)batch_row(b) % (uint32_t)a.block * a.row_stride;
        wait_reads();   // (other lanes' writes, read by the requests)
      };
      const uint8_t* buf0 = lds + wave * (NB * G::TILE);
      const int in_copy = lane / CPR, piece = lane % CPR;
      const uint32_t at_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)buf0;
      // tile i of the wave on its way into buffer i % NB
      auto request = [&](int i) {
        const uint32_t buf = at_lds + i % NB * G::TILE;
#pragma unroll
        for (int c = 0; c < NI; ++c) {
          const int r = RPI * c + in_copy;
          const uint8_t* src = cache + offsets[wave][i % G::BATCH * KEYS + r] + 16 * (piece ^ swizzle<G>(r));
          copy16_to_lds_rfl_v<kOnce>(src, buf + 1024 * c);
        }
      };

      // Q^T: the columns of step s that lane group g holds are those of K's pieces
      const float scale = a.scale_log2 * (kE4 && a.k_scale ? a.k_scale[kh] : 1.f);
      u32x4 qo[Y][D / 32];
      const uint32_t flip = scale < 0.f ? 0x80008000u : 0u;   // scores of -q, so that the largest one has the largest weight
#pragma unroll
      for (int y = 0; y < Y; ++y) {
        const bool used = kTokens ? token[y] >= t && token[y] < t_last : head[y] < heads;
        const uint16_t* qp = a.q + (int64_t)(kTokens && used ? token[y] : my_token) * a.q_st + (int64_t)(h0 + (used ? head[y] : 0)) * a.q_sh;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
          const int col = kE4 ? 16 * (g + 4 * (s / 2)) + 8 * (s % 2) : 32 * s + 8 * g;
          qo[y][s] = used ? ld16(qp + col) ^ flip : u32x4{0u, 0u, 0u, 0u};
        }
      }
      const float factor = scale == 0.f ? 0x1p-126f : fabsf(scale);   // (a masked score stays -inf)

      float m[Y], l[Y];
      floatx4 o[CT][Y];
#pragma unroll
      for (int y = 0; y < Y; ++y) {
        m[y] = -INFINITY;
        l[y] = 0.f;
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c][y] = floatx4{0.f, 0.f, 0.f, 0.f};
      }

      if (mine > 0) {
        fetch_ids(0);
        wait_copies<0>();
        work_out(0);
        if (mine > G::BATCH) fetch_ids(1);
        for (int i = 0; i < NB - 1 && i < mine; ++i) request(i);   // (NB - 1 <= BATCH)
      }
      for (int i = 0; i < mine; ++i) {
        const int ahead = i + NB - 1;
        if (ahead < mine) {
          if (ahead % G::BATCH == 0 && ahead > 0) {
            // the ids were requested a batch ago, before copies that have been waited for
            work_out(ahead / G::BATCH);
            if ((ahead / G::BATCH + 1) * G::BATCH < mine) {
              wait_reads();   // page_ids has been read
              fetch_ids(ahead / G::BATCH + 1);
            }
          }
          wait_reads();       // so has the buffer
          request(ahead);
          wait_copies<NI * (NB - 1)>();
        } else {
          wait_copies<0>();
        }
        const uint8_t* buf = buf0 + i % NB * G::TILE;

        constexpr int KB = KEYS / 16;
        floatx4 s[Y][KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
#pragma unroll
          for (int y = 0; y < Y; ++y) s[y][b] = floatx4{0.f, 0.f, 0.f, 0.f};
          const int key = 16 * b + x;
#pragma unroll
          for (int c = 0; c < CPR / 8; ++c) {
            const u32x4 v = ld16(buf + key * RB + 16 * ((4 * c + g) ^ swizzle<G>(key)));
            if (kE4) {
              const u32x4 lower = e4m3_to_bf16(v[0], v[1]), upper = e4m3_to_bf16(v[2], v[3]);
#pragma unroll
              for (int y = 0; y < Y; ++y) s[y][b] = mfma16x16x32(upper, qo[y][2 * c + 1], mfma16x16x32(lower, qo[y][2 * c], s[y][b]));
            } else {
#pragma unroll
              for (int y = 0; y < Y; ++y) s[y][b] = mfma16x16x32(v, qo[y][c], s[y][b]);
            }
          }
        }
        const int row0 = lo + (wave + i * WAVES) * KEYS, left = hi - row0;   // keys of the tile
        const bool mixed = kTokens && (row0 < all_first || row0 + KEYS > all_n);   // some tokens see some of them
        if (kTokens) {
          if (mixed) {
#pragma unroll
            for (int y = 0; y < Y; ++y)
#pragma unroll
              for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const int j = row0 + 16 * b + 4 * g + r;
                  if (j < my_first[y] || j >= my_n[y]) s[y][b][r] = -INFINITY;
                }
          }
        } else if (left < KEYS) {
          // rows past the last repeat it: no weight, and values of 0 (0 * inf is not)
#pragma unroll
          for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (16 * b + 4 * g + r >= left) s[0][b][r] = -INFINITY;
          for (int j = left * CPR + lane; j < KEYS * CPR; j += 64) st16(const_cast<uint8_t*>(buf) + 16 * j, u32x4{0u, 0u, 0u, 0u});
          wait_reads();
        }
        u32x2 p[Y][KB], p2[Y][KB];   // the column's part of P; with 16 heads p2 has the rests
#pragma unroll
        for (int y = 0; y < Y; ++y) {
          float top = -INFINITY;
#pragma unroll
          for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, s[y][b][r]);
          top = wave_max16x4(top) * factor;
          if (__any(top > m[y] + kRaise)) {
            const float raised = fmaxf(m[y], top);
            const float alpha = raised == -INFINITY ? 1.f : fast_exp2(m[y] - raised);
            m[y] = raised;
            l[y] *= alpha;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
              for (int r = 0; r < 4; ++r) o[c][y][r] *= alpha;
          }
          const float from = m[y] == -INFINITY ? 0.f : m[y];   // (nothing but scores of -inf so far: weights of zero)
#pragma unroll
          for (int b = 0; b < KB; ++b) {
            float w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) l[y] += w[r] = fast_exp2(fmaf(s[y][b][r], factor, -from));
            p[y][b] = u32x2{upper_halves(w[0], w[1]), upper_halves(w[2], w[3])};
            p2[y][b] = u32x2{rests(w[0], w[1], p[y][b][0]), rests(w[2], w[3], p[y][b][1])};
            if (kColumns == kTwice && x >= 8) p[y][b] = p2[y][b];
          }
        }
        // V^T of 16 columns, as the A operand
        // e4m3: lane x of group g reads half a piece of key 4g + x/2 (x < 8) or 16 + 4g + x/2 - 4; bf16: of key 4g + x/4
        const int key = kE4 ? (x < 8 ? 0 : 12) + 4 * g + (x >> 1) : 4 * g + (x >> 2);
        const uint8_t* vr = buf + key * RB + 8 * (x & 1);
        auto add = [&](floatx4 (&to)[Y], int c, const uint32_t* seen, bool both) {
          if constexpr (kE4) {
            typedef int int2v __attribute__((ext_vector_type(2)));
            int2v v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (__attribute__((address_space(3))) int2v*)(vr + 16 * ((CPR / 2 + c) ^ swizzle<G>(key))));
            if (seen) v = int2v{(int)(v[0] & seen[0]), (int)(v[1] & seen[1])};
            const u32x4 vt = e4m3_to_bf16((uint32_t)v[0], (uint32_t)v[1]);
#pragma unroll
            for (int y = 0; y < Y; ++y) {
              to[y] = mfma16x16x32(vt, u32x4{p[y][0][0], p[y][0][1], p[y][1][0], p[y][1][1]}, to[y]);
              if (both) to[y] = mfma16x16x32(vt, u32x4{p2[y][0][0], p2[y][0][1], p2[y][1][0], p2[y][1][1]}, to[y]);
            }
          } else {
            u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) short4v*)(vr + 16 * ((CPR / 2 + 2 * c + ((x >> 1) & 1)) ^ swizzle<G>(key)))));
            if (seen) v = u32x2{v[0] & seen[0], v[1] & seen[1]};
#pragma unroll
            for (int y = 0; y < Y; ++y) {
              // both parts of P as keys of one product, V twice
              if (both) to[y] = mfma16x16x32(u32x4{v[0], v[1], v[0], v[1]}, u32x4{p[y][0][0], p[y][0][1], p2[y][0][0], p2[y][0][1]}, to[y]);
              else to[y] = mfma16x16x16(__builtin_bit_cast(short4v, v), __builtin_bit_cast(short4v, p[y][0]), to[y]);
            }
          }
        };
        bool apart = false;
        if (kTokens && mixed) {
          // rows that a token does not see may hold anything, and 0 * NaN is not 0: is there an infinity or NaN?
          uint32_t bad = 0;
          for (int i = lane; i < KEYS * CPR / 2; i += 64) {
            const u32x4 v = ld16(buf + i / (CPR / 2) * RB + 16 * ((CPR / 2 + i % (CPR / 2)) ^ swizzle<G>(i / (CPR / 2))));
#pragma unroll
            for (int e = 0; e < 4; ++e)
              bad |= kE4 ? ((v[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((v[e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
          }
          apart = __any(bad != 0);
        }
        if (kTokens && apart) {   // a token at a time, its rows and its columns
          for (int u = t; u < t_last; ++u) {
            const int f = __shfl(lane_first, u - t_group), c1 = __shfl(lane_n, u - t_group);
            uint32_t seen[2];   // of keys 4g .. and 16 + 4g .. (a byte each), or of 4g, 4g + 1 and 4g + 2, 4g + 3 (a half each)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              seen[w] = 0;
#pragma unroll
              for (int e = 0; e < (kE4 ? 4 : 2); ++e) {
                const int j = row0 + 4 * g + (kE4 ? 16 * w : 2 * w) + e;
                if (j >= f && j < c1) seen[w] |= (kE4 ? 0xffu : 0xffffu) << (kE4 ? 8 : 16) * e;
              }
            }
#pragma unroll
            for (int c = 0; c < CT; ++c) {
              floatx4 more[Y] = {};
              add(more, c, seen, true);
#pragma unroll
              for (int y = 0; y < Y; ++y)
                if (token[y] == u) o[c][y] += more[y];
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < CT; ++c) add(o[c], c, nullptr, kColumns != kTwice);
        }
      }

      // the waves' parts together
#pragma unroll
      for (int y = 0; y < Y; ++y) {
        l[y] = wave_sum16x4(l[y]);
        if (g == 0) {
          stats[wave][0][16 * y + x] = m[y];
          stats[wave][1][16 * y + x] = l[y];
        }
      }
      __syncthreads();   // (and every wave has read its last tile)
      float* joined = reinterpret_cast<float*>(lds);
#pragma unroll
      for (int y = 0; y < Y; ++y) {
        float top = -INFINITY;
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stats[w][0][16 * y + x]);
        const float f = m[y] == -INFINITY ? 0.f : fast_exp2(m[y] - top);
        // (a NaN among the scores is in l, and where m is -inf nothing but zeros and NaN are in o)
        if (kTokens || head[y] < heads) {
#pragma unroll
          for (int c = 0; c < CT; ++c) *reinterpret_cast<floatx4*>(joined + (wave * COLS + 16 * y + x) * OS + 16 * c + 4 * g) = o[c][y] * f;
        }
      }
      __syncthreads();
      const int j_first = (t - t_group) * heads, j_count = (t_last - t) * heads;   // its columns (the tokens' ones)
      for (int i = tid; i < (kTokens ? j_count : heads) * (D / 4); i += 64 * WAVES) {
        const int j = (kTokens ? j_first : 0) + i / (D / 4), col = i % (D / 4) * 4;
        const int u = kTokens ? t_group + j / heads : my_token, h = h0 + (kTokens ? j % heads : j);
        float top = -INFINITY, sum = 0.f;
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stats[w][0][j]);
        floatx4 v = floatx4{0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < WAVES; ++w) {
          const float mw = stats[w][0][j];
          sum += stats[w][1][j] * (mw == -INFINITY ? 0.f : fast_exp2(mw - top));
          v += *reinterpret_cast<floatx4*>(joined + (w * COLS + j) * OS + col);
          if (kColumns == kTwice) v += *reinterpret_cast<floatx4*>(joined + (w * COLS + j + 8) * OS + col);
        }
        bool none = sum == 0.f;
        if (kTokens) {
          int f, c;
          token_rows(a, u, f, c);
          none = none || c <= f;   // (its columns took part in what the others see)
        }
        // (weights of 0, of which a NaN in V made NaN: no weight at all gives 0, but a part may yet be joined to others)
        if (none && whole) v = floatx4{0.f, 0.f, 0.f, 0.f};
        const float inv = none ? 0.f : (kE4 && a.v_scale ? a.v_scale[kh] : 1.f) / sum;
        const float lse = none ? -INFINITY : (top + log2f(sum)) * kLn2;
        if (!whole) {   // rows that began in an earlier share, or that go on in the next
          const int64_t place = ((int64_t)2 * k + (at == 0)) * a.H + h;
          *reinterpret_cast<floatx4*>(a.ws_o + place * D + col) = v * inv;
          if (col == 0) a.ws_lse[place] = lse;
        } else {
          *reinterpret_cast<u32x2*>(a.out + (int64_t)u * a.o_st + (int64_t)h * a.o_sh + col) =
              u32x2{pack2(v[0] * inv, v[1] * inv), pack2(v[2] * inv, v[3] * inv)};
          if (col == 0) a.lse[(int64_t)h * a.T + u] = lse;
        }
      }
    }
    if constexpr (kTokens) {
      for (int skip = 0; skip < a.grouped; ++skip) heads_of_runs &= heads_of_runs - 1;
      if (!heads_of_runs) return;
      t = t_group + __ffs((int)heads_of_runs) - 1;
    } else {
      left_steps -= taken;
      if (!a.shares || left_steps <= 0) return;
      before += steps;
      at = 0;
      ++t;           // (steps are left, so a token with rows follows)
    }
    __syncthreads(); // the parts in LDS have been read
  }
}

// The tokens alone in a list, for shares beside groups
__global__ __launch_bounds__(1024) void exact_alone_kernel(ExactCacheParams a) {
  __shared__ int sums[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int count = 0;
  for (int t0 = 0; t0 < a.T; t0 += 1024) {
    const bool alone = t0 + tid < a.T && is_alone(a, t0 + tid);
    const uint64_t mask = __ballot(alone);
    if (lane == 0) sums[wave] = __popcll(mask);
    __syncthreads();
    int at = count;
    for (int w = 0; w < 16; ++w) {
      at += w < wave ? sums[w] : 0;
      count += sums[w];
    }
    if (alone) a.alone[1 + at + __popcll(mask & ((1ull << lane) - 1))] = t0 + tid;
    __syncthreads();
  }
  if (tid == 0) a.alone[0] = count;
}

// The parts of one (token, head) joined by their lse, where its rows lie in several shares; tokens without rows. One workgroup
// for a token, or, of the tokens alone, for every gridDim.x / H-th; D / 4 threads per part.
template <int D, bool kAlone>
__global__ __launch_bounds__(256) void exact_join_kernel(ExactCacheParams a) {
  constexpr int PER = D / 4, ROWS = 256 / PER;
  __shared__ float weight[kMaxShares];
  __shared__ floatx4 sums[ROWS][PER];
  __shared__ float red[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x % a.H, tokens = shared_tokens<kAlone>(a);
  int i = blockIdx.x / a.H;
  if (i >= tokens) return;
  do {
    const int t = shared_token<kAlone>(a, i);
    int first, n;
    token_rows(a, t, first, n);
    int k0 = 0, count = 0;
    if (n > first) {
      k0 = a.split[2 * i];
      count = a.split[2 * i + 1] - k0 + 1;
      if (count == 1) continue;   // written by its workgroup
    }
    // part s: the rows' end of share k0 (s = 0), or their beginning in share k0 + s
    const int64_t place = ((int64_t)2 * k0 + 1) * a.H + h;
    auto where = [&](int s) { return place + (s ? (2 * (int64_t)s - 1) * a.H : 0); };
    float top = -INFINITY;
    for (int s = tid; s < count; s += 256) top = fmaxf(top, weight[s] = a.ws_lse[where(s)]);
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    if (lane == 0) red[0][wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    float w = 0.f;
    for (int s = tid; s < count; s += 256) {
      // (a part with a NaN lse has a NaN weight; one with nothing but scores of -inf has a weight of 0, and its NaN, if V has any, stay)
      const float mine = weight[s];
      w += weight[s] = mine == -INFINITY ? 0.f : fast_exp2((mine - top) * kLog2e);
    }
    for (int off = 32; off > 0; off >>= 1) w += __shfl_xor(w, off);
    if (lane == 0) red[1][wave] = w;
    __syncthreads();
    const float sum = red[1][0] + red[1][1] + red[1][2] + red[1][3];
    floatx4 v = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = tid / PER; s < count; s += ROWS)
      v += *reinterpret_cast<const floatx4*>(a.ws_o + where(s) * D + tid % PER * 4) * weight[s];
    sums[tid / PER][tid % PER] = v;
    __syncthreads();
    if (tid >= PER) continue;   // (what is in LDS has been read before it is written again: barriers lie between)
    for (int r = 1; r < ROWS; ++r) v += sums[r][tid];
    const bool none = sum == 0.f;
    if (none) v = floatx4{0.f, 0.f, 0.f, 0.f};
    const float inv = none ? 0.f : 1.f / sum;
    *reinterpret_cast<u32x2*>(a.out + (int64_t)t * a.o_st + (int64_t)h * a.o_sh + 4 * tid) =
        u32x2{pack2(v[0] * inv, v[1] * inv), pack2(v[2] * inv, v[3] * inv)};
    if (tid == 0) a.lse[(int64_t)h * a.T + t] = none ? -INFINITY : top + logf(sum);
  } while (kAlone && (i += gridDim.x / a.H) < tokens);
}

// Groups of tokens: 32 columns take half as many reads of K and V, where there are two workgroups per CU all the same (4 x 512
// tokens on 8160 rows of 16 heads 555 -> 454 us, with P in two products; of 256 workgroups with them 61, of 512 without 53). With
// d = 256 the registers do not suffice for them (463 -> 817).
bool groups_of_32(const ExactCacheParams& p, int dim) {
  const int group = kMaxTile * 2 / p.G;
  return dim <= 128 && p.grouped && ((int64_t)p.T + group - 1) / group * p.KH >= 2 * kCus;
}

int64_t exact_workgroups(const ExactCacheParams& p, int dim) {
  const int group = !p.grouped ? 1 : (groups_of_32(p, dim) ? 2 : 1) * kMaxTile / p.G;
  return (p.shares ? p.shares : ((int64_t)p.T + group - 1) / group) * (p.grouped ? p.grouped : 1) * p.KH * p.tiles;
}

// The two halves of a step with shares beside groups
ExactCacheParams groups_of(ExactCacheParams p) {
  p.shares = 0;
  return p;
}
ExactCacheParams alone_of(ExactCacheParams p) {
  p.grouped = 0;
  return p;
}

template <int D, bool kE4>
void launch_exact_cache(const ExactCacheParams& p, hipStream_t st) {
  const bool more = groups_of_32(p, D);
  const unsigned grid = (unsigned)exact_workgroups(p, D);
  // past the caches where no other workgroup reads the rows (a chunk of 64 tokens on 8160 rows, 8 KV heads for 32: 128 us, past them 145)
  const bool once = p.tiles == 1 && !p.shared;
  // whole tokens for at most a workgroup per CU: twice the waves (one token of 16 heads, 993 rows: 17.4 us with 4, 11.7 with 8)
  const bool wide = !p.shares && !p.grouped && (int64_t)p.T * p.KH * p.tiles <= kCus;
  using G = ExactGeo<D, kE4, false>;
  using W = ExactGeo<D, kE4, true>;
  void (*const kernels[10])(ExactCacheParams) = {
      exact_cache_kernel<G, false, kHeads>, exact_cache_kernel<G, false, kTwice>, exact_cache_kernel<G, true, kHeads>,
      exact_cache_kernel<G, true, kTwice>,  exact_cache_kernel<W, false, kHeads>, exact_cache_kernel<W, false, kTwice>,
      exact_cache_kernel<W, true, kHeads>,  exact_cache_kernel<W, true, kTwice>,  exact_cache_kernel<G, false, kTokens16>,
      exact_cache_kernel<G, false, D <= 128 ? kTokens32 : kTokens16>};
  hipLaunchKernelGGL(kernels[p.grouped ? 8 + more : 4 * wide + 2 * once + (p.G <= 8)], dim3(grid), dim3(64 * (wide ? W::WAVES : G::WAVES)),
                     0, st, p);
  if (p.shares)
    hipLaunchKernelGGL((exact_join_kernel<D, false>), dim3((unsigned)((int64_t)p.T * p.H)), dim3(256), 0, st, p);
}

// Shares beside groups: the groups in a launch of their own, then the tokens alone
template <int D, bool kE4>
void launch_exact(const ExactCacheParams& p, hipStream_t st) {
  if (!p.shares || !p.grouped) return launch_exact_cache<D, kE4>(p, st);
  launch_exact_cache<D, kE4>(groups_of(p), st);
  hipLaunchKernelGGL(exact_alone_kernel, dim3(1), dim3(1024), 0, st, p);
  using G = ExactGeo<D, kE4, false>;   // (groups have at most 8 heads, and a table row of its own is read once)
  hipLaunchKernelGGL((exact_cache_kernel<G, true, kTwice, true>), dim3((unsigned)exact_workgroups(alone_of(p), D)),
                     dim3(64 * G::WAVES), 0, st, alone_of(p));
  const int tokens = min(p.T, max(1, 4096 / p.H));
  hipLaunchKernelGGL((exact_join_kernel<D, true>), dim3((unsigned)(tokens * p.H)), dim3(256), 0, st, p);
}

// ---- store -------------------------------------------------------------------------------------------------------
// Rows into slots, a thread per 8 values (16 bytes in); e4m3: x / scale, clamped to +-448, to the nearest, ties to even. Bound by
// HBM: 8192 tokens of 16 heads, 134 MB both ways, 23.8 us, 5.6 TB/s (a large copy 5.1: some rows are in the last cache), with stores
// past the caches; with plain ones 30.
struct ExactStoreParams {
  const uint16_t *key, *value;
  int64_t k_st, k_sh, v_st, v_sh;
  int T, KH, D;
  const int64_t* slots;
  const float *k_scale, *v_scale;
  uint8_t* cache;
  int64_t page_stride, head_stride, row_stride;  // bytes
  int block;
  int64_t num_blocks;
};

__device__ __forceinline__ uint32_t four_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

template <bool kE4>
__global__ __launch_bounds__(256) void exact_store_kernel(ExactStoreParams a) {
  const int per_half = a.D / 8, per_token = 2 * per_half * a.KH;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.T * per_token) return;
  const int t = (int)(i / per_token), at = (int)(i % per_token);
  const int c = at % per_half, half = at / per_half & 1, h = at / (2 * per_half);
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.num_blocks * a.block) return;
  const u32x4 v = ld16(half ? a.value + t * a.v_st + h * a.v_sh + 8 * c : a.key + t * a.k_st + h * a.k_sh + 8 * c);
  uint8_t* dst = a.cache + slot / a.block * a.page_stride + slot % a.block * a.row_stride + h * a.head_stride;
  if (!kE4) {
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(dst + 2 * (half * a.D + 8 * c)));
    return;
  }
  const float* scales = half ? a.v_scale : a.k_scale;
  const float s = scales ? scales[h] : 1.f;
  float f[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = lo_bf(v[e]) / s;
    f[2 * e + 1] = hi_bf(v[e]) / s;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = f[e] > 448.f ? 448.f : f[e] < -448.f ? -448.f : f[e];   // (NaN stays)
  __builtin_nontemporal_store(u32x2{four_e4m3(f[0], f[1], f[2], f[3]), four_e4m3(f[4], f[5], f[6], f[7])},
                              reinterpret_cast<u32x2*>(dst + half * a.D + 8 * c));
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Checks of a cache; strides in elements
int check_exact_cache(const char* what, const void* cache, int e4m3, int dim, int kv_heads, int64_t page_stride,
                      int64_t head_stride, int64_t row_stride, int block, int64_t num_blocks) {
  const int es = e4m3 ? 1 : 2;
  HLA_REQUIRE(dim == 64 || dim == 128 || dim == 256, HLA_S6_EUNSUPPORTED, "%s: head dim %d not in {64, 128, 256}", what, dim);
  HLA_REQUIRE(kv_heads >= 1 && kv_heads <= 1 << 20, HLA_S6_EINVAL, "%s: %d KV heads", what, kv_heads);
  HLA_REQUIRE(block >= 1 && num_blocks >= 1, HLA_S6_EINVAL, "%s: bad block size or page count", what);
  HLA_REQUIRE(cache && aligned16(cache), HLA_S6_EINVAL, "%s: the cache must be 16-byte aligned", what);
  HLA_REQUIRE(page_stride >= 0 && head_stride >= 0 && row_stride >= 0 && page_stride * es % 16 == 0 &&
                  head_stride * es % 16 == 0 && row_stride * es % 16 == 0,
              HLA_S6_EINVAL, "%s: page, head and row strides must be multiples of 16 bytes", what);
  HLA_REQUIRE((kv_heads == 1 || head_stride >= 2 * dim) && (block == 1 || row_stride >= 2 * dim), HLA_S6_EINVAL,
              "%s: rows overlap (strides smaller than 2 x %d values)", what, dim);
  return HLA_S6_OK;
}

}  // namespace
}  // namespace hla

extern "C" int hla_s6_exact_attention(const void* q, int32_t num_tokens, int32_t num_heads, int32_t head_dim, int64_t q_st,
                                      int64_t q_sh, const void* cache, int32_t e4m3, int32_t kv_heads, int64_t page_stride,
                                      int64_t head_stride, int64_t row_stride, int32_t block_size, int64_t num_blocks,
                                      const int32_t* block_table, int64_t bt_stride, int32_t bt_cols, int32_t bt_count,
                                      const int64_t* bt_rows, const int32_t* ctx, int32_t window, float scale,
                                      const float* k_scale, const float* v_scale, int32_t shares,
                                      int32_t grouped, float* workspace, int64_t workspace_floats, void* out, int64_t o_st, int64_t o_sh,
                                      float* lse, int32_t shared_rows, void* stream) {
  using namespace hla;
  HLA_REQUIRE(num_tokens >= 0, HLA_S6_EINVAL, "exact_attention: negative token count");
  int rc = check_exact_cache("exact_attention", cache, e4m3, head_dim, kv_heads, page_stride, head_stride, row_stride,
                             block_size, num_blocks);
  if (rc != HLA_S6_OK) return rc;
  HLA_REQUIRE(num_heads >= kv_heads && num_heads % kv_heads == 0, HLA_S6_EINVAL,
              "exact_attention: %d query heads over %d KV heads", num_heads, kv_heads);
  HLA_REQUIRE(shares >= 0 && shares <= kMaxShares, HLA_S6_EINVAL, "exact_attention: %d shares (0..%d)", shares, kMaxShares);
  HLA_REQUIRE(window >= 0 && bt_cols >= 0, HLA_S6_EINVAL, "exact_attention: bad window or table");
  HLA_REQUIRE(e4m3 || (!k_scale && !v_scale), HLA_S6_EINVAL, "exact_attention: scales belong to e4m3 caches");
  if (num_tokens == 0) return HLA_S6_OK;
  HLA_REQUIRE(bt_count >= (bt_rows ? 1 : num_tokens), HLA_S6_EINVAL, "exact_attention: %d table rows", bt_count);
  HLA_REQUIRE(q && ctx && out && lse && (block_table || bt_cols == 0), HLA_S6_EINVAL, "exact_attention: null pointer argument");
  HLA_REQUIRE(aligned16(q) && q_st % 8 == 0 && q_sh % 8 == 0 && aligned16(out) && o_st % 8 == 0 && o_sh % 8 == 0,
              HLA_S6_EINVAL, "exact_attention: rows of q and out must be 16-byte aligned");
  ExactCacheParams p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.cache = static_cast<const uint8_t*>(cache);
  const int es = e4m3 ? 1 : 2;
  p.page_stride = page_stride * es;
  p.head_stride = head_stride * es;
  p.row_stride = row_stride * es;
  p.block = block_size;
  p.num_blocks = num_blocks;
  p.bt = block_table;
  p.bt_stride = bt_stride;
  p.bt_cols = bt_cols;
  p.bt_count = bt_count;
  p.bt_rows = bt_rows;
  p.ctx = ctx;
  p.window = window;
  p.scale_log2 = scale * kLog2e;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.T = num_tokens;
  p.H = num_heads;
  p.KH = kv_heads;
  p.G = num_heads / kv_heads;
  p.tiles = (p.G + kMaxTile - 1) / kMaxTile;
  p.shares = shares;
  p.grouped = grouped;
  p.shared = shared_rows != 0;
  HLA_REQUIRE(grouped >= 0 && grouped <= kMaxTile && (!grouped || ((shares == 0 || bt_rows) && p.G <= kMaxTile / 2)), HLA_S6_EINVAL,
              "exact_attention: groups of tokens need table rows per request or shares 0, at most %d query heads per KV head and at "
              "most %d turns", kMaxTile / 2, kMaxTile);
  // (KH * tiles is at most H, so that workgroups are counted in 64 bits; none of a grid has more than 256 threads but one of few)
  const bool both = shares && grouped;
  HLA_REQUIRE((int64_t)p.T * p.H <= INT32_MAX && launchable(exact_workgroups(both ? groups_of(p) : p, head_dim), 256) &&
                  (!both || launchable(exact_workgroups(alone_of(p), head_dim), 256)) &&
                  (!shares || both || launchable((int64_t)p.T * p.H, 256)), HLA_S6_EINVAL, "exact_attention: too many rows");
  if (shares) {
    const int64_t rows = (int64_t)2 * shares * p.H, need = rows * (head_dim + 1) + (both ? 3 * (int64_t)p.T + 1 : 2 * (int64_t)p.T);
    HLA_REQUIRE(workspace && workspace_floats >= need, HLA_S6_EWORKSPACE,
                "exact_attention: workspace overflow: %lld floats, have %lld", (long long)need, (long long)workspace_floats);
    HLA_REQUIRE(aligned16(workspace), HLA_S6_EINVAL, "exact_attention: workspace must be 16-byte aligned");
    p.ws_o = workspace;
    p.ws_lse = workspace + rows * head_dim;
    p.split = reinterpret_cast<int32_t*>(p.ws_lse + rows);
    if (both) p.alone = p.split + 2 * (int64_t)p.T;
  }
  p.out = static_cast<uint16_t*>(out);
  p.o_st = o_st;
  p.o_sh = o_sh;
  p.lse = lse;
  const hipStream_t st = as_stream(stream);
#define HLA_EXACT(D) e4m3 ? launch_exact<D, true>(p, st) : launch_exact<D, false>(p, st)
  switch (head_dim) {
    case 64: HLA_EXACT(64); break;
    case 128: HLA_EXACT(128); break;
    default: HLA_EXACT(256); break;
  }
#undef HLA_EXACT
  return check_launch("exact_attention");
}

extern "C" int hla_s6_exact_store(const void* key, int64_t k_st, int64_t k_sh, const void* value, int64_t v_st, int64_t v_sh,
                                  int32_t num_tokens, int32_t kv_heads, int32_t head_dim, const int64_t* slots,
                                  const float* k_scale, const float* v_scale, void* cache, int32_t e4m3,
                                  int64_t page_stride, int64_t head_stride, int64_t row_stride, int32_t block_size,
                                  int64_t num_blocks, void* stream) {
  using namespace hla;
  HLA_REQUIRE(num_tokens >= 0, HLA_S6_EINVAL, "exact_store: negative token count");
  int rc = check_exact_cache("exact_store", cache, e4m3, head_dim, kv_heads, page_stride, head_stride, row_stride, block_size,
                             num_blocks);
  if (rc != HLA_S6_OK) return rc;
  HLA_REQUIRE(e4m3 || (!k_scale && !v_scale), HLA_S6_EINVAL, "exact_store: scales belong to e4m3 caches");
  if (num_tokens == 0) return HLA_S6_OK;
  HLA_REQUIRE(key && value && slots, HLA_S6_EINVAL, "exact_store: null pointer argument");
  HLA_REQUIRE(aligned16(key) && aligned16(value) && k_st % 8 == 0 && k_sh % 8 == 0 && v_st % 8 == 0 && v_sh % 8 == 0,
              HLA_S6_EINVAL, "exact_store: rows of key and value must be 16-byte aligned");
  const int es = e4m3 ? 1 : 2;
  ExactStoreParams p = {static_cast<const uint16_t*>(key), static_cast<const uint16_t*>(value), k_st, k_sh, v_st, v_sh,
                        num_tokens, kv_heads, head_dim, slots, k_scale, v_scale, static_cast<uint8_t*>(cache),
                        page_stride * es, head_stride * es, row_stride * es, block_size, num_blocks};
  const int64_t blocks = ((int64_t)num_tokens * kv_heads * (head_dim / 4) + 255) / 256;
  HLA_REQUIRE(launchable(blocks, 256), HLA_S6_EINVAL, "exact_store: too many rows");
  const hipStream_t st = as_stream(stream);
  if (e4m3) hipLaunchKernelGGL(exact_store_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL(exact_store_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, st, p);
  return check_launch("exact_store");
}
