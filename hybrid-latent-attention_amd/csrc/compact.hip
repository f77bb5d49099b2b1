// The compact latent cache (compact.h): row commit, row load and paged history attention over 4-bit rows.
#include <type_traits>

#include "compact.h"
#include "split_plan.h"

namespace hla {
namespace {

// ---- commit ------------------------------------------------------------------------------------------------------
// One thread per eight columns of a row, four threads per block of 32. The block's scale exponent is the smallest e with
// max|x| <= 7 * 2^e: the largest value then takes its nearest representable one (up to 7 * 2^e it is nearer to 6 * 2^e
// than to 8 * 2^e). Values go to the nearest E2M1 number, ties to the even one (v_cvt_scalef32_pk_fp4_bf16); a block with
// a value that is not finite gets scale byte 255 and reads as NaN.
struct StoreParams {
  const uint16_t* key;
  const uint16_t* value;
  int64_t k_st, v_st;
  const int64_t* slots;
  uint8_t* cache;
  int64_t page_stride;
  int block;
  int64_t num_slots;
  int64_t units;  // threads of work: T * 2 W / 8
};

__device__ __forceinline__ uint32_t abs_max2(uint32_t m, uint32_t pair) {
  return max(m, max(pair & 0x7fffu, (pair >> 16) & 0x7fffu));
}

template <int W, bool VEC>
__global__ __launch_bounds__(256) void compact_store_kernel(StoreParams a) {
  constexpr int PER = W / 4;  // threads per row
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= a.units) return;  // whole rows of threads: PER is a multiple of 4, and 256 of PER or PER of 256
  const int64_t t = u / PER;
  const int i = (int)(u % PER);
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.num_slots) return;  // the same for all four threads of a block
  const bool is_v = i >= PER / 2;
  const int col = (is_v ? i - PER / 2 : i) * 8;
  const uint16_t* src = (is_v ? a.value + t * a.v_st : a.key + t * a.k_st) + col;
  u32x4 x;
  if (VEC) {
    x = ld16(src);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (uint32_t)src[2 * e] | ((uint32_t)src[2 * e + 1] << 16);
  }
  uint32_t most = 0;  // bit patterns of non-negative bf16 order as integers
#pragma unroll
  for (int e = 0; e < 4; ++e) most = abs_max2(most, x[e]);
  most = max(most, (uint32_t)__shfl_xor((int)most, 1));
  most = max(most, (uint32_t)__shfl_xor((int)most, 2));
  const bool finite = most < 0x7f80u;
  const int e0 = (int)(most >> 7) - 129 + ((most & 127u) > 96u ? 1 : 0);  // 7 = 1.75 * 4: fraction 96 / 128
  const int exponent = min(max(e0, kMinExponent), kMaxExponent);
  const uint32_t byte = finite ? (uint32_t)(exponent + 127) : 255u;
  const float scale = __uint_as_float((uint32_t)(exponent + 127) << 23);
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  uint32_t code = 0;
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, (uint32_t)x[0]), scale, 0);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, (uint32_t)x[1]), scale, 1);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, (uint32_t)x[2]), scale, 2);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, (uint32_t)x[3]), scale, 3);
  if (!finite) code = 0;
  const int in_page = (int)(slot % a.block), r = in_page & 15, b = col >> 5;
  uint8_t* tile = a.cache + (slot / a.block) * a.page_stride + (in_page >> 4) * compact_tile_bytes(W);
  const int at = is_v ? v_code_at(W, r, col >> 1) : k_code_at(r, b) + ((col & 31) >> 1);
  *reinterpret_cast<uint32_t*>(tile + at) = code;
  if ((i & 3) == 0) tile[is_v ? v_scale_at(W, r, b) : k_scale_at(W, r, b)] = (uint8_t)byte;
}

// ---- load --------------------------------------------------------------------------------------------------------
// out[r, j, :] = row j of request r in bf16 for j < lengths[r], 0 behind it (without lengths: of a step's tokens, and
// nothing behind it). One thread per eight columns: 4 bytes in, 16 out. HBM-bound by the writes (64 W bytes of every 81 W).
// They go past the caches (16 x 4096 rows at W = 512: 27.5 us, 6.2 TB/s; through them 43), but for a step's, which the attention
// reads next (4 x 512 tokens on 7000 to 8160: 562 us with it, past the caches 609).
struct LoadParams {
  const uint8_t* cache;
  int64_t page_stride;
  int block;
  int64_t num_blocks;
  const int32_t* bt;
  int64_t bt_stride;
  int bt_cols;
  const int32_t* lengths;  // or null: the largest ctx of the request's tokens
  const int32_t* qsl;
  const int32_t* ctx;
  int T, R;
  uint16_t* out;
  int64_t o_sr, o_sj;  // elements per request and per row
  int max_rows;
};

// the largest ctx of request r's tokens, and of those outside all chunks (padding, which may name any request)
__device__ int most_ctx(const LoadParams& a, int r) {
  __shared__ int red[4];
  int most = 0;
  auto take = [&](int t0, int t1) {
    for (int t = max(t0, 0) + (int)threadIdx.x; t < min(t1, a.T); t += 256) most = max(most, a.ctx[t]);
  };
  take(a.qsl[r], a.qsl[r + 1]);
  take(0, a.qsl[0]);
  take(a.qsl[a.R], a.T);
  for (int off = 32; off > 0; off >>= 1) most = max(most, __shfl_xor(most, off));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
  __syncthreads();
  return max(max(red[0], red[1]), max(red[2], red[3]));
}

template <int W, bool kLengths>
__global__ __launch_bounds__(256) void compact_load_kernel(LoadParams a) {
  constexpr int PER = W / 4;                         // threads per row
  constexpr int ROWS = PER <= 256 ? 256 / PER : 1;   // rows per pass of the workgroup
  const int r = blockIdx.y, i = threadIdx.x % PER;
  const int n = (int)min((int64_t)max(kLengths ? a.lengths[r] : most_ctx(a, r), 0), (int64_t)a.bt_cols * a.block);
  const int32_t* btr = a.bt + (int64_t)r * a.bt_stride;
  const bool is_v = i >= PER / 2;
  const int col = (is_v ? i - PER / 2 : i) * 8, b = col >> 5;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t j = ((int64_t)blockIdx.x * 4 + p) * ROWS + threadIdx.x / PER;
    if (j >= a.max_rows || (j >= n && !kLengths)) return;
    u32x4 x = {0u, 0u, 0u, 0u};
    if (j < n) {
      const int64_t page = clamp_page(btr[j / a.block], a.num_blocks);
      const int in_page = (int)(j % a.block), x16 = in_page & 15;
      const uint8_t* tile = a.cache + page * a.page_stride + (in_page >> 4) * compact_tile_bytes(W);
      const int at = is_v ? v_code_at(W, x16, col >> 1) : k_code_at(x16, b) + ((col & 31) >> 1);
      const uint32_t code = *reinterpret_cast<const uint32_t*>(tile + at);
      const uint32_t scale = tile[is_v ? v_scale_at(W, x16, b) : k_scale_at(W, x16, b)];
      x = eight_bf16(code, scale_of(scale, 0));
    }
    u32x4* to = reinterpret_cast<u32x4*>(a.out + (int64_t)r * a.o_sr + j * a.o_sj + (is_v ? W : 0) + col);
    if constexpr (kLengths) __builtin_nontemporal_store(x, to);
    else *to = x;
  }
}

// ---- history attention ---------------------------------------------------------------------------------------------
// One workgroup of four waves per (token, split). Every wave walks its own 32 rows of each 128 (two tiles), alone:
//   * S^T[32 keys x 16 heads] = K Q^T on v_mfma_f32_16x16x32_bf16. A lane's 16 bytes of K are one block of 32 columns of
//     one row, four k-steps of eight values; Q^T is read with the same order of columns, so nothing is moved.
//   * online softmax in the exp2 domain: a lane holds 8 keys of one head, and P^T stays where it is: the order of keys in
//     the next product's contraction is free, and is taken to be the one the scores come out in.
//   * O^T[columns x 16 heads] += V^T P^T: a lane loads the same 8 keys' values of W / 16 consecutive columns (one scale
//     per key and 32 columns); two keys' values of a column are joined by one v_perm_b32 per pair. Product c of a wave
//     takes column c of every lane's range.
// No row passes through LDS (from W = 512 on the query does) until the waves' partials are joined at the end. At W = 1024 two
// waves share 32 keys, each with all of K and half of the columns of V.
// Bound by HBM where a row is read once: 64 rows of 8160 at W = 512 50 us, 5.7 TB/s with a fixed part of about 11 us (launch,
// work list, page ids and query, first rows, join); by the conversions (8 clocks a pair of values) where rows come out of L2.
struct CompactParams {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint8_t* cache;
  int64_t page_stride;
  int block;
  int64_t num_blocks;
  const int32_t* bt;
  int64_t bt_stride;
  int bt_cols, bt_count;
  const int64_t* bt_rows;
  const int32_t* ctx;
  float scale_log2;
  int num_splits, T;
  float* ws_o;    // [T][S][16][W]
  float* ws_lse;  // [T][S][16]
  const int32_t* plan;
  uint16_t* out;  // one split: the final output and lse
  int64_t o_st, o_sh;
  float* lse;
};

template <int W>
struct VTile {  // one tile of V: rows 4g .. 4g + 3, CPL columns per lane (m, g)
  Words<CompactGeo<W>::VD> code[4];
  uint32_t scale;  // of the four rows
};

template <int W, bool kOnce>
__device__ __forceinline__ void load_v(const uint8_t* tile, int m, int g, int half, VTile<W>& v) {
  using G = CompactGeo<W>;
  const int col = half * (W / G::CH) + m * G::CPL;
  v.scale = *reinterpret_cast<const uint32_t*>(tile + 16 * W + W / 2 + (col / 32) * 16 + 4 * g);
#pragma unroll
  for (int r = 0; r < 4; ++r) v.code[r] = load_words<G::VD, kOnce>(tile + 8 * W + (r * 4 + g) * (W / 2) + col / 2);
}

// Columns 2 kByte and 2 kByte + 1 of dword d of every lane's range: eight keys each, two products
template <int W, int kByte>
__device__ __forceinline__ void pv_pair(const VTile<W> (&v)[2], const float (&f)[8], u32x4 p, int d, floatx4& even,
                                        floatx4& odd) {
  uint32_t x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = two_bf16<kByte>(v[e / 4].code[e % 4].w[d], f[e]);
  u32x4 lo, hi;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    lo[e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x05040100u);
    hi[e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x07060302u);
  }
  even = mfma16x16x32(lo, p, even);
  odd = mfma16x16x32(hi, p, odd);
}

// The workgroup's item of the step's work list, without a plan, worked out by every wave for itself (no barrier): rows are
// cut in chunks of max(ceil(longest / S), ceil(2 total / (T S))) tiles, at least kMinChunk (kMinChunkSmall in small steps):
// split_chunk's first value, which fits every row in its S slots, and then grow in a few larger steps where that function
// takes single tiles. Lane l looks after rows [l, l + 1) * ceil(T / 64). (With split_chunk and find_item, six barriers, a
// call of 992 rows took 1.2 us longer, one of 32 ragged rows in two slots each 133 us longer.)
__device__ __forceinline__ void wave_item(const int32_t* ctx, int T, int64_t cap, int S, int b, int lane, int& chunk,
                                          int& t, int& s) {
  const int seg = (T + 63) / 64, r0 = min(T, lane * seg), r1 = min(T, r0 + seg);
  const int one = r0 < r1 ? row_tiles(ctx[r0], cap) : 0;  // the only one where T <= 64
  int longest = one;
  int64_t sum = one;
  for (int r = r0 + 1; r < r1; ++r) {
    const int tiles = row_tiles(ctx[r], cap);
    longest = max(longest, tiles);
    sum += tiles;
  }
  longest = wave_max(longest);
  sum = ((int64_t)wave_total((int)(sum >> 12)) << 12) + wave_total((int)(sum & 4095));
  const int64_t slots = (int64_t)T * S;
  const int least = min(longest, sum < kSmallStepTiles ? kMinChunkSmall : kMinChunk);
  chunk = (int)max((int64_t)max(1, least), max((int64_t)(longest + S - 1) / S, (2 * sum + slots - 1) / slots));
  int mine, upto;
  for (int turn = 0;; ++turn) {  // the tails of ragged rows: larger chunks until at most T S / 2 items are left
    mine = (one + chunk - 1) / chunk;
    for (int r = r0 + 1; r < r1; ++r) mine += (row_tiles(ctx[r], cap) + chunk - 1) / chunk;
    upto = wave_scan(mine);
    const int items = __builtin_amdgcn_readlane(upto, 63);
    if (items <= slots / 2 || turn == 6 || chunk >= longest) break;
    chunk = min(longest, max(chunk + 1, (int)((int64_t)chunk * items / (slots / 2))));
  }
  const uint64_t owner = __ballot(b >= upto - mine && b < upto);
  if (owner == 0) {  // past the end of the list
    t = -1;
    return;
  }
  int row = r0, slot = b - (upto - mine);
  for (int r = r0; r < r1; ++r) {  // (lanes that do not own the item run on, to no effect)
    const int used = (row_tiles(ctx[r], cap) + chunk - 1) / chunk;
    if (slot < used) break;
    slot -= used;
    row = r + 1;
  }
  const int src = __ffsll((unsigned long long)owner) - 1;
  t = __builtin_amdgcn_readlane(row, src);
  s = __builtin_amdgcn_readlane(slot, src);
}

// The log-sum-exp of a slot: NaN goes in as infinity, which makes the row NaN in the reductions over slots. (They take the
// largest of a row's first, past NaN, and would find a row empty whose every slot is NaN.)
__device__ __forceinline__ float slot_lse(float lse) { return lse != lse ? INFINITY : lse; }

template <int W, bool kOnce>
__global__ __launch_bounds__(256, W <= 512 ? 2 : 1) void compact_history_kernel(CompactParams a) {
  using G = CompactGeo<W>;
  __shared__ float m_lds[4][16], l_lds[4][16];
  constexpr int C2 = G::CPL / 8;  // half of a lane's columns, in fours
  __shared__ floatx4 o_lds[4][G::CH][G::G - 1][C2][64];
  __shared__ u32x4 q_lds[QOperand<W>::kLds ? G::KC * 4 : 1][64];

  const int tid = threadIdx.x, lane = tid & 63, h = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = wave % G::CH, set = wave / G::CH;
  const int S = a.num_splits, b = blockIdx.x;
  const int64_t cap = (int64_t)a.bt_cols * a.block;
  int t = b, s = 0, chunk = 0;
  int ctx_of_lane = 0;  // of row `lane`, and its table row: on their way with the work list, in steps of up to 64 rows
  int64_t row_of_lane = 0;
  const bool from_lanes = S > 1 && !a.plan && a.T <= 64;
  if (from_lanes && lane < a.T) {
    ctx_of_lane = a.ctx[lane];
    row_of_lane = a.bt_rows ? a.bt_rows[lane] : lane;
  }
  if (S > 1) {
    if (a.plan) {
      chunk = a.plan[0];
      t = a.plan[1 + a.T + b];
      s = a.plan[1 + a.T + (int)split_workgroups(a.T, S) + b];
    } else {
      wave_item(a.ctx, a.T, cap, S, b, lane, chunk, t, s);
    }
    if (b < a.T) {  // slots of row b past its work
      const int used = a.plan ? min(max(a.plan[1 + b], 0), S) : used_slots(a.ctx[b], cap, chunk);
      float* l0 = a.ws_lse + ((int64_t)b * S + used) * kHeads;
      for (int i = tid; i < (S - used) * kHeads; i += 256) l0[i] = -INFINITY;
    }
  }
  if (t < 0 || t >= a.T || s < 0 || s >= S) return;  // (past the end of the list; or no plan of this step's)
  t = __builtin_amdgcn_readfirstlane(t);
  s = __builtin_amdgcn_readfirstlane(s);
  const int n = (int)min((int64_t)max(from_lanes ? __builtin_amdgcn_readlane(ctx_of_lane, t) : a.ctx[t], 0), cap);
  const int tiles = (n + kTile - 1) / kTile;
  chunk = S == 1 ? tiles : min(max(chunk, 1), tiles);  // (whatever a plan holds: tiles of this row, and no overflow)
  const int j_begin = (int)min((int64_t)s * chunk, (int64_t)tiles), j_end = min(tiles, j_begin + chunk);
  const int64_t part_row = ((int64_t)t * S + s) * kHeads;

  if (j_begin >= j_end) {  // a row without history
    if (!a.out) {
      if (tid < kHeads) a.ws_lse[part_row + tid] = -INFINITY;
      return;
    }
    for (int i = tid; i < kHeads * W / 4; i += 256)
      *reinterpret_cast<uint2*>(a.out + (int64_t)t * a.o_st + (int64_t)(i / (W / 4)) * a.o_sh + i % (W / 4) * 4) =
          uint2{0u, 0u};
    if (tid < kHeads) a.lse[(int64_t)tid * a.T + t] = -INFINITY;
    return;
  }

  const int64_t named = from_lanes ? (int64_t)(((uint64_t)__builtin_amdgcn_readlane((uint32_t)((uint64_t)row_of_lane >> 32), t) << 32) |
                                               (uint32_t)__builtin_amdgcn_readlane((uint32_t)row_of_lane, t))
                                   : a.bt_rows ? a.bt_rows[t] : (int64_t)t;
  const int64_t table_row = min(max(named, (int64_t)0), (int64_t)a.bt_count - 1);
  const int32_t* btr = a.bt + table_row * a.bt_stride;
  const int limit = min(n, j_end * kTile);
  // Tile addresses of the wave's next 32 steps, worked out by its lanes together: lane 2i + e holds the byte offset of tile e
  // of step i. (A page id read by the scalar unit in every step put its latency, a trip to L2 or HBM, into each of them.)
  const int stride = 2 * G::G;
  uint32_t off_lo, off_hi;
  auto look_up = [&](int j0) {
    const int row = min(j0 + (lane >> 1) * stride + (lane & 1), j_end - 1) * kTile;  // (past the chunk: its last tile, masked)
    const int64_t page = clamp_page(btr[row / a.block], a.num_blocks);
    const int64_t off = page * a.page_stride + (row % a.block) / kTile * compact_tile_bytes(W);
    off_lo = (uint32_t)off;
    off_hi = (uint32_t)((uint64_t)off >> 32);
  };
  auto tile_at = [&](int i) {
    const uint32_t lo = __builtin_amdgcn_readlane(off_lo, i), hi = __builtin_amdgcn_readlane(off_hi, i);
    return a.cache + (int64_t)(((uint64_t)hi << 32) | lo);
  };

  floatx4 acc[G::CPL];
#pragma unroll
  for (int c = 0; c < G::CPL; ++c) acc[c] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  KTile<W> k[2];
  VTile<W> v[2];
  // page ids, then the query, then the first rows, each on its way while the one before is waited for
  int j = j_begin + 2 * set;
  look_up(j);
  QOperand<W> q;
  q.template fetch<4>(a.q + (int64_t)t * a.q_st + (int64_t)h * a.q_sh, g, wave);
  const uint8_t *t0 = tile_at(0), *t1 = tile_at(1);
  if (j < j_end) {
    load_k<W, kOnce>(t0, h, g, k[0]);
    load_k<W, kOnce>(t1, h, g, k[1]);
    load_v<W, kOnce>(t0, h, g, half, v[0]);
    load_v<W, kOnce>(t1, h, g, half, v[1]);
  }
  q.template share<4>(wave, lane, q_lds);
  // (the last step by itself: behind a branch that may have skipped the next one's loads the compiler can only wait for all of
  // them, K of the next step with V of this one: 64 rows of 8160, 77 us and 3.7 TB/s; loads of the last tiles over again in
  // its place hold up the end)
  int step = 1;
  auto one_step = [&](auto last) {
    floatx4 s0, s1;
    scores<W>(k, q, lane, s0, s1);
    if constexpr (!last.value || W < 256) {
      if ((step & 31) == 0) look_up(j + stride);
      t0 = tile_at(2 * (step & 31));
      t1 = tile_at(2 * (step & 31) + 1);
      load_k<W, kOnce>(t0, h, g, k[0]);
      load_k<W, kOnce>(t1, h, g, k[1]);
    }
    float sc[8], f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sc[e] = s0[e] * a.scale_log2;
      sc[4 + e] = s1[e] * a.scale_log2;
      f[e] = scale_of(v[0].scale, e);
      f[4 + e] = scale_of(v[1].scale, e);
    }
    const int key = j * kTile + 4 * g;
    if ((j + 2) * kTile > limit) {  // hide the keys past the end, and their scales, which may be those of NaN
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (key + (e / 4) * kTile + e % 4 >= limit) {
          sc[e] = -INFINITY;
          f[e] = 0.f;
        }
    }
    float mx = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
    mx = wave_max16x4(mx);
    // the running maximum is raised only past 2^8, so most steps leave the accumulators alone
    const bool raise = mx > m + 8.f;
    if (__any(raise)) {
      const float m_new = raise ? mx : m;
      const float alpha = raise ? fast_exp2(m - m_new) : 1.f;
      l *= alpha;
      m = m_new;
#pragma unroll
      for (int c = 0; c < G::CPL; ++c) acc[c] = acc[c] * alpha;
    }
    const float m_use = m == -INFINITY ? 0.f : m;
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = fast_exp2(sc[e] - m_use);
    l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    // P in bf16, as in the bf16 cache's kernels: half a step of 2^-8 per weight, independent from key to key
    const u32x4 pb = {pack2(p[0], p[1]), pack2(p[2], p[3]), pack2(p[4], p[5]), pack2(p[6], p[7])};
#pragma unroll
    for (int d = 0; d < G::VD; ++d) {
      pv_pair<W, 0>(v, f, pb, d, acc[8 * d + 0], acc[8 * d + 1]);
      pv_pair<W, 1>(v, f, pb, d, acc[8 * d + 2], acc[8 * d + 3]);
      pv_pair<W, 2>(v, f, pb, d, acc[8 * d + 4], acc[8 * d + 5]);
      pv_pair<W, 3>(v, f, pb, d, acc[8 * d + 6], acc[8 * d + 7]);
    }
    if constexpr (!last.value || W < 256) {
      load_v<W, kOnce>(t0, h, g, half, v[0]);
      load_v<W, kOnce>(t1, h, g, half, v[1]);
    }
  };
  if constexpr (W >= 256) {  // (at 128, where four waves a SIMD hide it, the second body costs more: 64 rows of 8160 27 us and 33
                             // with it; 22.6 since slots are joined by compact_join_kernel)
    for (; j + stride < j_end; j += stride, ++step) one_step(std::false_type{});
    if (j < j_end) one_step(std::true_type{});
  } else {
    for (; j < j_end; j += stride, ++step) one_step(std::false_type{});
  }

  // Join the sets of keys: every wave at the common maximum, then, half of each lane's columns at a time, set i mod G adds up
  // accumulator element i of all of them and writes it.
  l = wave_sum16x4(l);
  if (g == 0) {
    m_lds[wave][h] = m;
    l_lds[wave][h] = l;
  }
  __syncthreads();
  float top = -INFINITY, total = 0.f;
#pragma unroll
  for (int x = 0; x < G::G; ++x) top = fmaxf(top, m_lds[x * G::CH][h]);
#pragma unroll
  for (int x = 0; x < G::G; ++x) total += l_lds[x * G::CH][h] * fast_exp2(m_lds[x * G::CH][h] - top);
  const float mine = fast_exp2(m - top);
  const float inv = 1.0f / total;
  if (wave == 0 && g == 0) {
    const float lse = (top + log2f(total)) * kLn2;
    if (a.out) a.lse[(int64_t)h * a.T + t] = lse;
    else a.ws_lse[part_row + h] = slot_lse(lse);
  }
  // (all sets at work in each part, the reads of a part on their way together, and no barrier that waits for the stores: with
  // one set after the other this took 3.2 us at W = 512)
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    if (part > 0) lds_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int owner = i % G::G;
      if (set == owner) continue;
      const int at = set < owner ? set : set - 1;
#pragma unroll
      for (int c = 0; c < C2; ++c) {
        const int b = 4 * (part * C2 + c);
        o_lds[i][half][at][c][lane] = floatx4{acc[b][i], acc[b + 1][i], acc[b + 2][i], acc[b + 3][i]} * mine;
      }
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (set != i % G::G) continue;
      floatx4 o[C2];
#pragma unroll
      for (int c = 0; c < C2; ++c) {
        const int b = 4 * (part * C2 + c);
        o[c] = floatx4{acc[b][i], acc[b + 1][i], acc[b + 2][i], acc[b + 3][i]} * mine;
#pragma unroll
        for (int x = 0; x < G::G - 1; ++x) o[c] += o_lds[i][half][x][c][lane];
        o[c] = o[c] * inv;
      }
      const int col = half * (W / G::CH) + G::CPL * (4 * g + i) + 4 * part * C2;
      if (a.out) {
#pragma unroll
        for (int c = 0; c < C2; ++c)
          *reinterpret_cast<uint2*>(a.out + (int64_t)t * a.o_st + (int64_t)h * a.o_sh + col + 4 * c) =
              uint2{pack2(o[c][0], o[c][1]), pack2(o[c][2], o[c][3])};
      } else {
#pragma unroll
        for (int c = 0; c < C2; ++c) *reinterpret_cast<floatx4*>(a.ws_o + (part_row + h) * W + col + 4 * c) = o[c];
      }
    }
  }
}

// Two tokens of one request, same rows: the conversion of a row to bf16, which is what bounds the kernel above where rows
// come out of L2 (8 clocks per pair of values, as long as the two 16 x 16 products that a token has for them), serves both.
// One workgroup of four waves per (pair of tokens, split); 32 columns of the products are the pair's 2 x 16 heads, so S^T and
// O^T come from v_mfma_f32_32x32x16_bf16. A wave takes 256 columns of 32 rows: W / 256 waves share a set of rows, add their
// parts of the scores through LDS (one barrier a step, the parts in two buffers), and go on with the softmax each for itself.
// The queries lie in LDS. O^T needs 128 accumulators a lane at every width. Tokens of a pair that differ in request or
// length go through their rows one after the other: a product spreads a NaN in one's rows to the other's sums.
// 4 x 512 tokens on 8160 rows: w = 512 668 us (820 TFLOP/s; a token per workgroup 765), w = 256 322 (458), w = 1024 2025 (2645).
// Four tokens per workgroup convert half as often, but need registers that spill (w = 512: twice as long).
template <int W>
struct PairGeo {
  static constexpr int CH = W / 256;     // waves per set of rows
  static constexpr int G = 4 / CH;       // sets
  static constexpr int FRAGS = W / 16;   // steps of Q, 16 columns each
};
struct PairRows {  // what a lane holds of 32 rows
  u32x4 k[4];
  uint32_t k_scale[2];
  uint32_t v[2][8];
  uint32_t v_scale[2][2];
};
template <int W>
__device__ __forceinline__ void pair_load_k(const uint8_t* t0, const uint8_t* t1, int n, int f, int slice, PairRows& r) {
  const uint8_t* tile = n < 16 ? t0 : t1;
  const int x = n & 15;
  // scales of blocks b = 8 slice + 2i + f: [b % 4][b / 4], two pairs of neighbours
  const uint8_t* sp = tile + 16 * W + x * (W / 32) + 2 * slice;
  r.k_scale[0] = *reinterpret_cast<const uint16_t*>(sp + f * (W / 128));
  r.k_scale[1] = *reinterpret_cast<const uint16_t*>(sp + (2 + f) * (W / 128));
#pragma unroll
  for (int i = 0; i < 4; ++i) r.k[i] = ld16(tile + k_code_at(x, 8 * slice + 2 * i + f));
}
template <int W>
__device__ __forceinline__ void pair_load_v(const uint8_t* t0, const uint8_t* t1, int n, int f, int slice, PairRows& r) {
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const uint8_t* tile = m ? t1 : t0;
    const uint8_t* sp = tile + 16 * W + W / 2 + (8 * slice + n / 4) * 16 + 4 * f;
    r.v_scale[m][0] = *reinterpret_cast<const uint32_t*>(sp);
    r.v_scale[m][1] = *reinterpret_cast<const uint32_t*>(sp + 8);
#pragma unroll
    for (int e = 0; e < 8; ++e)  // rows 4f + e, then 8 + 4f + e - 4
      r.v[m][e] = *reinterpret_cast<const uint32_t*>(tile + 8 * W + (4 * (e & 3) + 2 * (e >> 2) + f) * (W / 2) + 128 * slice + 4 * n);
  }
}
// columns 2 kByte and 2 kByte + 1 of the lane's eight for the 16 keys of tile m
template <int kByte>
__device__ __forceinline__ void pair_pv(const PairRows& r, int m, const float (&f)[8], u32x4 p, floatx16& even, floatx16& odd) {
  uint32_t x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = two_bf16<kByte>(r.v[m][e], f[e]);
  u32x4 lo, hi;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    lo[e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x05040100u);
    hi[e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x07060302u);
  }
  even = mfma32x32x16(lo, p, even);
  odd = mfma32x32x16(hi, p, odd);
}
template <int W>
__global__ __launch_bounds__(256, W <= 512 ? 2 : 1) void compact_pair_kernel(CompactParams a) {
  using P = PairGeo<W>;
  constexpr int JOIN = P::G > 1 ? 2 * P::CH * 4 * (P::G - 1) * 2 : 0, SUMS = P::CH > 1 ? 2 * 4 * 4 : 0;
  __shared__ u32x4 q_lds[P::FRAGS][64];
  __shared__ floatx4 x_lds[JOIN > SUMS ? JOIN : SUMS][64];  // parts of the scores; then of the outputs
  __shared__ float m_lds[4][32], l_lds[4][32];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, f = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), slice = wave % P::CH, set = wave / P::CH;
  const int S = a.num_splits, s = blockIdx.y;
  const int ta = 2 * blockIdx.x, tb = min(ta + 1, a.T - 1);
  const int64_t cap = (int64_t)a.bt_cols * a.block;
  const int mine = n < 16 ? ta : tb, h = n & 15;
#pragma unroll
  for (int i = 0; i < P::FRAGS / 4; ++i) {
    const int x = wave * (P::FRAGS / 4) + i;
    q_lds[x][lane] = ld16(a.q + (int64_t)mine * a.q_st + (int64_t)h * a.q_sh + 32 * (x / 4 * 2 + f) + 8 * (x % 4));
  }
  __syncthreads();
  const int64_t ra = a.bt_rows ? a.bt_rows[ta] : ta, rb = a.bt_rows ? a.bt_rows[tb] : tb;
  const int na = a.ctx[ta], nb = a.ctx[tb];
  const bool both = ra == rb && na == nb;
#pragma unroll 1
  for (int pass = 0; pass < (both ? 1 : 2); ++pass) {  // (uniform over the workgroup, all but in_pass and what hangs on it)
    const int rows = (int)min((int64_t)max(pass ? nb : na, 0), cap);
    const int tiles = (rows + kTile - 1) / kTile, chunk = (tiles + S - 1) / S;
    const int j_begin = s * chunk, j_end = min(tiles, j_begin + chunk);
    const int limit = min(rows, j_end * kTile);
    const bool in_pass = both || (n < 16) == (pass == 0);
    floatx16 acc[8];
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[t][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    if (j_begin < j_end) {
      const int64_t table_row = min(max(pass ? rb : ra, (int64_t)0), (int64_t)a.bt_count - 1);
      const int32_t* btr = a.bt + table_row * a.bt_stride;
      constexpr int stride = 2 * P::G;
      uint32_t off_lo, off_hi;
      auto look_up = [&](int j0) {  // as in compact_history_kernel
        const int row = min(j0 + (lane >> 1) * stride + (lane & 1), j_end - 1) * kTile;
        const int64_t page = clamp_page(btr[row / a.block], a.num_blocks);
        const int64_t off = page * a.page_stride + (row % a.block) / kTile * compact_tile_bytes(W);
        off_lo = (uint32_t)off;
        off_hi = (uint32_t)((uint64_t)off >> 32);
      };
      auto tile_at = [&](int i) {
        const uint32_t lo = __builtin_amdgcn_readlane(off_lo, i), hi = __builtin_amdgcn_readlane(off_hi, i);
        return a.cache + (int64_t)(((uint64_t)hi << 32) | lo);
      };
      int j = j_begin + 2 * set;  // past the end in the last step of some sets: rows loaded again, and hidden
      look_up(j);
      PairRows r;
      const uint8_t *t0 = tile_at(0), *t1 = tile_at(1);
      pair_load_k<W>(t0, t1, n, f, slice, r);
      pair_load_v<W>(t0, t1, n, f, slice, r);
      for (int step = 1; j_begin + (step - 1) * stride < j_end; j += stride, ++step) {
        floatx16 sc;
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float scale = scale_of(r.k_scale[i & 1], i >> 1);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            sc = mfma32x32x16(eight_bf16(r.k[i][c], scale), q_lds[16 * slice + 4 * i + c][lane], sc);
        }
        if ((step & 31) == 0) look_up(j + stride);
        t0 = tile_at(2 * (step & 31));
        t1 = tile_at(2 * (step & 31) + 1);
        pair_load_k<W>(t0, t1, n, f, slice, r);
        if constexpr (P::CH > 1) {
          floatx4(*to)[64] = x_lds + ((step & 1) * 4 + wave) * 4;
#pragma unroll
          for (int e = 0; e < 4; ++e) to[e][lane] = floatx4{sc[4 * e], sc[4 * e + 1], sc[4 * e + 2], sc[4 * e + 3]};
          __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));  // LDS alone: the rows on their way stay on it
          plain_barrier();
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // every wave of the set adds in the same order
            const floatx4(*from)[64] = x_lds + ((step & 1) * 4 + set * P::CH) * 4;
            floatx4 v = from[e][lane];
#pragma unroll
            for (int c = 1; c < P::CH; ++c) v += from[4 * c + e][lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[4 * e + i] = v[i];
          }
        }
        float vf[2][8];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          sc[e] *= a.scale_log2;
          vf[e / 8][e % 8] = scale_of(r.v_scale[e / 8][e / 4 % 2], e % 4);
        }
        if ((j + 2) * kTile > limit || !both) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool seen = j * kTile + e / 4 * 8 + 4 * f + e % 4 < limit;
            if (!seen) vf[e / 8][e % 8] = 0.f;
            if (!seen || !in_pass) sc[e] = -INFINITY;
          }
        }
        float mx = sc[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, sc[e]);
        mx = xor32_max(mx);
        const bool raise = mx > m + 8.f;
        if (__any(raise)) {
          const float m_new = raise ? mx : m;
          const float alpha = raise ? fast_exp2(m - m_new) : 1.f;
          l *= alpha;
          m = m_new;
#pragma unroll
          for (int t = 0; t < 8; ++t) acc[t] = acc[t] * alpha;
        }
        const float m_use = m == -INFINITY ? 0.f : m;
        float p[16], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = fast_exp2(sc[e] - m_use);
#pragma unroll
        for (int e = 0; e < 16; e += 4) sum += (p[e] + p[e + 1]) + (p[e + 2] + p[e + 3]);
        l += sum;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const u32x4 pb = {pack2(p[8 * x], p[8 * x + 1]), pack2(p[8 * x + 2], p[8 * x + 3]),
                            pack2(p[8 * x + 4], p[8 * x + 5]), pack2(p[8 * x + 6], p[8 * x + 7])};
          pair_pv<0>(r, x, vf[x], pb, acc[0], acc[1]);
          pair_pv<1>(r, x, vf[x], pb, acc[2], acc[3]);
          __builtin_amdgcn_sched_barrier(0);
          pair_pv<2>(r, x, vf[x], pb, acc[4], acc[5]);
          pair_pv<3>(r, x, vf[x], pb, acc[6], acc[7]);
          __builtin_amdgcn_sched_barrier(0);
        }
        pair_load_v<W>(t0, t1, n, f, slice, r);
      }
    }
    // Join the sets. Element 4j + i of accumulator t is column 256 slice + 8 m' + t with m' = 8j + 4f + i; set i % G writes it.
    {
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
      l = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    }
    if (f == 0) { m_lds[wave][n] = m; l_lds[wave][n] = l; }
    __syncthreads();
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int x = 0; x < P::G; ++x) top = fmaxf(top, m_lds[x * P::CH][n]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int x = 0; x < P::G; ++x) total += l_lds[x * P::CH][n] * fast_exp2(m_lds[x * P::CH][n] - base);
    const float own = fast_exp2(m - base), inv = total == 0.f ? 0.f : 1.0f / total;
    const bool store = in_pass && (n < 16 || ta + 1 < a.T);
    const int64_t part = ((int64_t)mine * S + s) * kHeads + h;
    if (wave == 0 && f == 0 && store) {
      const float lse = total == 0.f ? -INFINITY : (top + log2f(total)) * kLn2;
      if (a.out) a.lse[(int64_t)h * a.T + mine] = lse;
      else a.ws_lse[part] = slot_lse(lse);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (P::G > 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (set != i % P::G) {
            const int at = set < i % P::G ? set : set - 1;
#pragma unroll
            for (int c = 0; c < 2; ++c)
              x_lds[((((j & 1) * P::CH + slice) * 4 + i) * (P::G - 1) + at) * 2 + c][lane] =
                  floatx4{acc[4 * c][4 * j + i], acc[4 * c + 1][4 * j + i], acc[4 * c + 2][4 * j + i], acc[4 * c + 3][4 * j + i]} * own;
          }
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (set != i % P::G) continue;
        const int col = 256 * slice + 8 * (8 * j + 4 * f + i);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          floatx4 o = floatx4{acc[4 * c][4 * j + i], acc[4 * c + 1][4 * j + i], acc[4 * c + 2][4 * j + i], acc[4 * c + 3][4 * j + i]} * own;
#pragma unroll
          for (int x = 0; x < P::G - 1; ++x) o += x_lds[((((j & 1) * P::CH + slice) * 4 + i) * (P::G - 1) + x) * 2 + c][lane];
          o = o * inv;
          if (!store) continue;
          if (a.out)
            *reinterpret_cast<uint2*>(a.out + (int64_t)mine * a.o_st + (int64_t)h * a.o_sh + col + 4 * c) = uint2{pack2(o[0], o[1]), pack2(o[2], o[3])};
          else
            *reinterpret_cast<floatx4*>(a.ws_o + part * W + col + 4 * c) = o;
        }
      }
    }
    if (pass == 0 && !both) __syncthreads();  // (the next pass writes what this one may still read)
  }
}

// The slots of (token t, head h) joined by their log-sum-exp, columns [4 L z, 4 L (z + 1)): groups of L lanes take every NG-th
// slot, kAhead of them on their way together, and their sums meet in LDS, in order. Bound by latency: slots' lse, then their
// partials. A slot without rows costs a read of the first one's partial, which is in the cache. 64 rows of 8160 in 8 slots: 4.9
// us (reading the empty slots as well: 6.4), 8 of 32736 in 64: 4.4.
template <int W, int L, int NG, int kAhead>
__global__ __launch_bounds__(L* NG) void compact_join_kernel(CompactParams a) {
  constexpr int THREADS = L * NG, WAVES = THREADS / 64;
  __shared__ float lse_lds[kMaxSplits];
  __shared__ float top_lds[WAVES], den_lds[NG];
  __shared__ floatx4 acc_lds[NG][L];
  const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, i = tid % L, q = tid / L, S = a.num_splits;
  const int col = blockIdx.z * 4 * L + 4 * i;
  const float* ls = a.ws_lse + (int64_t)t * S * kHeads + h;
  float top = -INFINITY;
  for (int s = tid; s < S; s += THREADS) {
    const float v = ls[(int64_t)s * kHeads];
    lse_lds[s] = v;
    top = fmaxf(top, v);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  if (tid % 64 == 0) top_lds[tid / 64] = top;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < WAVES; ++x) top = fmaxf(top, top_lds[x]);
  uint16_t* out = a.out + (int64_t)t * a.o_st + (int64_t)h * a.o_sh + col;
  if (top == -INFINITY) {  // uniform over the workgroup
    if (q == 0) *reinterpret_cast<uint2*>(out) = uint2{0u, 0u};
    if (tid == 0 && blockIdx.z == 0) a.lse[(int64_t)h * a.T + t] = -INFINITY;
    return;
  }
  const float* base = a.ws_o + ((int64_t)t * S * kHeads + h) * W + col;
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  float den = 0.f;
  for (int s0 = q; s0 < S; s0 += kAhead * NG) {
    floatx4 o[kAhead];
    float w[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int s = s0 + u * NG;
      const float v = s < S ? lse_lds[s] : -INFINITY;
      w[u] = fast_exp2((v - top) * kLog2e);  // (infinity for a NaN: NaN)
      o[u] = *reinterpret_cast<const floatx4*>(base + (int64_t)(v == -INFINITY ? 0 : s) * kHeads * W);
      if (v == -INFINITY) w[u] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const floatx4 x = w[u] == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : o[u];  // (the first slot's may be anything)
      den += w[u];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(x[e], w[u], acc[e]);
    }
  }
  acc_lds[q][i] = acc;
  if (i == 0) den_lds[q] = den;
  __syncthreads();
  if (q != 0) return;
#pragma unroll
  for (int x = 1; x < NG; ++x) {
    acc += acc_lds[x][i];
    den += den_lds[x];
  }
  acc = acc * (1.0f / den);
  *reinterpret_cast<uint2*>(out) = uint2{pack2(acc[0], acc[1]), pack2(acc[2], acc[3])};
  if (tid == 0 && blockIdx.z == 0) a.lse[(int64_t)h * a.T + t] = (top * kLog2e + log2f(den)) * kLn2;
}

template <int W>
void launch_join(const CompactParams& p, hipStream_t st) {
  // many slots come with few tokens: more groups, and more workgroups a head (1 token, 512 slots: 21.7 us for the call, 39.6
  // with two workgroups a head; with few slots these are too many: 16 tokens of 32 slots 21.1, this way 22.8)
  constexpr int L = W >= 256 ? 64 : 32;
  if (p.num_splits >= 64)
    hipLaunchKernelGGL((compact_join_kernel<W, 16, 16, 8>), dim3((unsigned)p.T, kHeads, W / 64), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((compact_join_kernel<W, L, 256 / L, 4>), dim3((unsigned)p.T, kHeads, W / (4 * L)), dim3(256), 0, st, p);
}

template <int W>
void launch_history(const CompactParams& p, int tokens_per_group, bool shared_rows, hipStream_t st) {
  if constexpr (W >= 256) {
    if (tokens_per_group == 2) {
      hipLaunchKernelGGL((compact_pair_kernel<W>), dim3((unsigned)((p.T + 1) / 2), (unsigned)p.num_splits), dim3(256), 0, st,
                         p);
      return;
    }
  }
  const dim3 grid(split_workgroups(p.T, p.num_splits));
  // rows that one token reads stream past the caches from W = 512 on (64 rows of 8160: 68.5 -> 60.5 us, 8 of 32736: 41.9 ->
  // 37.0); at 256 and below, where a lane's V pieces are shorter than a cached line's share, not (32 rows of up to 8160 at
  // 256: 20.0 -> 20.6)
  if (W >= 512 && !shared_rows)
    hipLaunchKernelGGL((compact_history_kernel<W, (W >= 512)>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((compact_history_kernel<W, false>), grid, dim3(256), 0, st, p);
}

template <int W>
void launch_store(const StoreParams& p, bool vec, hipStream_t st) {
  const dim3 grid((unsigned)((p.units + 255) / 256));
  if (vec) hipLaunchKernelGGL((compact_store_kernel<W, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((compact_store_kernel<W, false>), grid, dim3(256), 0, st, p);
}

template <int W>
void launch_load(const LoadParams& p, int R, hipStream_t st) {
  constexpr int rows = 4 * (W / 4 <= 256 ? 256 / (W / 4) : 1);
  const dim3 grid((unsigned)((p.max_rows + rows - 1) / rows), (unsigned)R);
  if (p.lengths) hipLaunchKernelGGL((compact_load_kernel<W, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((compact_load_kernel<W, false>), grid, dim3(256), 0, st, p);
}

}  // namespace
}  // namespace hla

extern "C" int hla_s6_compact_store(const void* key, int64_t k_st, const void* value, int64_t v_st, int32_t num_tokens,
                                    int32_t width, const int64_t* slots, void* cache, int64_t page_stride,
                                    int32_t block_size, int64_t num_blocks, void* stream) {
  using namespace hla;
  HLA_REQUIRE(num_tokens >= 0, HLA_S6_EINVAL, "compact_store: negative token count");
  int rc = check_cache("compact_store", width, cache, page_stride, block_size, num_blocks);
  if (rc != HLA_S6_OK || num_tokens == 0) return rc;
  HLA_REQUIRE(key && value && slots, HLA_S6_EINVAL, "compact_store: null pointer argument");
  StoreParams p = {};
  p.key = static_cast<const uint16_t*>(key);
  p.value = static_cast<const uint16_t*>(value);
  p.k_st = k_st;
  p.v_st = v_st;
  p.slots = slots;
  p.cache = static_cast<uint8_t*>(cache);
  p.page_stride = page_stride;
  p.block = block_size;
  p.num_slots = num_blocks * block_size;
  p.units = (int64_t)num_tokens * (width / 4);
  const bool vec = aligned(key, 16) && aligned(value, 16) && k_st % 8 == 0 && v_st % 8 == 0;
  const hipStream_t st = as_stream(stream);
  switch (width) {
    case 128: launch_store<128>(p, vec, st); break;
    case 256: launch_store<256>(p, vec, st); break;
    case 512: launch_store<512>(p, vec, st); break;
    default: launch_store<1024>(p, vec, st); break;
  }
  return check_launch("compact_store");
}

extern "C" int hla_s6_compact_load(const void* cache, int32_t width, int64_t page_stride, int32_t block_size,
                                   int64_t num_blocks, const int32_t* block_table, int64_t bt_stride, int32_t bt_cols,
                                   const int32_t* lengths, const int32_t* query_start_loc, const int32_t* ctx,
                                   int32_t num_tokens, int32_t num_reqs, int32_t max_rows, void* out, int64_t o_sr,
                                   int64_t o_sj, void* stream) {
  using namespace hla;
  HLA_REQUIRE(num_reqs >= 0 && num_reqs <= 65535 && max_rows >= 0 && bt_cols >= 0, HLA_S6_EINVAL,
              "compact_load: bad request count (0..65535), row count or table width");
  int rc = check_cache("compact_load", width, cache, page_stride, block_size, num_blocks);
  if (rc != HLA_S6_OK || num_reqs == 0 || max_rows == 0) return rc;
  HLA_REQUIRE((lengths || (query_start_loc && ctx)) && out && (block_table || bt_cols == 0), HLA_S6_EINVAL,
              "compact_load: null pointer argument");
  HLA_REQUIRE(aligned(out, 16) && o_sr % 8 == 0 && o_sj % 8 == 0 && o_sj >= 2 * width, HLA_S6_EINVAL,
              "compact_load: output rows must be 16-byte aligned and apart");
  LoadParams p = {};
  p.cache = static_cast<const uint8_t*>(cache);
  p.page_stride = page_stride;
  p.block = block_size;
  p.num_blocks = num_blocks;
  p.bt = block_table;
  p.bt_stride = bt_stride;
  p.bt_cols = bt_cols;
  p.lengths = lengths;
  p.qsl = query_start_loc;
  p.ctx = ctx;
  p.T = num_tokens;
  p.R = num_reqs;
  p.out = static_cast<uint16_t*>(out);
  p.o_sr = o_sr;
  p.o_sj = o_sj;
  p.max_rows = max_rows;
  const hipStream_t st = as_stream(stream);
  switch (width) {
    case 128: launch_load<128>(p, num_reqs, st); break;
    case 256: launch_load<256>(p, num_reqs, st); break;
    case 512: launch_load<512>(p, num_reqs, st); break;
    default: launch_load<1024>(p, num_reqs, st); break;
  }
  return check_launch("compact_load");
}

extern "C" int hla_s6_compact_history(const void* q, int32_t num_tokens, int32_t num_heads, int32_t width, int64_t q_st,
                                      int64_t q_sh, const void* cache, int64_t page_stride, int32_t block_size,
                                      int64_t num_blocks, const int32_t* block_table, int64_t bt_stride,
                                      int32_t bt_cols, int32_t bt_count, const int64_t* bt_rows, const int32_t* ctx,
                                      float scale, int32_t num_splits, float* workspace, int64_t workspace_floats,
                                      const int32_t* plan, int64_t plan_len, int32_t tokens_per_group,
                                      int32_t shared_rows, void* out, int64_t o_st, int64_t o_sh, float* lse,
                                      void* stream) {
  using namespace hla;
  HLA_REQUIRE(num_tokens >= 0, HLA_S6_EINVAL, "compact_history: negative token count");
  HLA_REQUIRE(num_heads == kHeads, HLA_S6_EUNSUPPORTED, "compact_history: %d query heads (the kernel is built for 16)",
              num_heads);
  int rc = check_cache("compact_history", width, cache, page_stride, block_size, num_blocks);
  if (rc != HLA_S6_OK) return rc;
  HLA_REQUIRE(num_splits >= 1 && num_splits <= kMaxSplits, HLA_S6_EINVAL,
              "compact_history: num_kv_splits must be in [1, %d]", kMaxSplits);
  HLA_REQUIRE(bt_cols >= 0, HLA_S6_EINVAL, "compact_history: bad table width");
  HLA_REQUIRE(tokens_per_group == 1 || (tokens_per_group == 2 && width >= 256), HLA_S6_EINVAL,
              "compact_history: %d tokens per group at width %d", tokens_per_group, width);
  if (num_tokens == 0) return HLA_S6_OK;
  HLA_REQUIRE(bt_count >= (bt_rows ? 1 : num_tokens), HLA_S6_EINVAL, "compact_history: %d table rows", bt_count);
  HLA_REQUIRE(q && (block_table || bt_cols == 0) && ctx && (out == nullptr) == (lse == nullptr), HLA_S6_EINVAL,
              "compact_history: null pointer argument");
  HLA_REQUIRE(aligned(q, 16) && q_st % 8 == 0 && q_sh % 8 == 0, HLA_S6_EINVAL,
              "compact_history: q needs 16-byte aligned rows (unit last stride, strides multiple of 8)");
  HLA_REQUIRE(aligned(out, 8) && o_st % 4 == 0 && o_sh % 4 == 0, HLA_S6_EINVAL,
              "compact_history: output rows must be 8-byte aligned");
  const bool partials = num_splits > 1 || !out;
  if (partials) {
    const int64_t need = (int64_t)num_tokens * num_splits * kHeads * (width + 1);
    HLA_REQUIRE(workspace != nullptr && workspace_floats >= need, HLA_S6_EWORKSPACE,
                "S6 workspace overflow: need %lld floats, have %lld", (long long)need, (long long)workspace_floats);
    HLA_REQUIRE(aligned(workspace, 16), HLA_S6_EINVAL, "compact_history: workspace must be 16-byte aligned");
  }
  HLA_REQUIRE(!plan || num_splits == 1 || plan_len >= plan_ints(num_tokens, num_splits), HLA_S6_EINVAL,
              "compact_history: split plan of %lld ints, need %lld", (long long)plan_len,
              (long long)plan_ints(num_tokens, num_splits));
  CompactParams p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.cache = static_cast<const uint8_t*>(cache);
  p.page_stride = page_stride;
  p.block = block_size;
  p.num_blocks = num_blocks;
  p.bt = block_table;
  p.bt_stride = bt_stride;
  p.bt_cols = bt_cols;
  p.bt_count = bt_count;
  p.bt_rows = bt_rows;
  p.ctx = ctx;
  p.scale_log2 = scale * kLog2e;
  p.num_splits = num_splits;
  p.T = num_tokens;
  p.plan = plan;
  if (partials) {
    p.ws_o = workspace;
    p.ws_lse = workspace + (int64_t)num_tokens * num_splits * kHeads * width;
  } else {
    p.out = static_cast<uint16_t*>(out);
    p.o_st = o_st;
    p.o_sh = o_sh;
    p.lse = lse;
  }
  const hipStream_t st = as_stream(stream);
#define HLA_EACH_WIDTH(call)     \
  switch (width) {               \
    case 128: call(128); break;  \
    case 256: call(256); break;  \
    case 512: call(512); break;  \
    default: call(1024); break;  \
  }
#define HLA_HISTORY(W) launch_history<W>(p, tokens_per_group, shared_rows != 0, st)
#define HLA_JOIN(W) launch_join<W>(p, st)
  HLA_EACH_WIDTH(HLA_HISTORY)
  rc = check_launch("compact_history");
  if (rc != HLA_S6_OK || !out || !partials) return rc;
  p.out = static_cast<uint16_t*>(out);
  p.o_st = o_st;
  p.o_sh = o_sh;
  p.lse = lse;
  HLA_EACH_WIDTH(HLA_JOIN)
#undef HLA_JOIN
#undef HLA_HISTORY
#undef HLA_EACH_WIDTH
  return check_launch("compact_history");
}
