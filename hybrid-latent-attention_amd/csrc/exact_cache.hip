// Attention over a whole exact (per-head K / V) paged cache, one new token per row, and the store into it.
//
// A cache page holds `block` rows of every KV head, [K | V] of 2d values in bf16 or e4m3; G query heads read one KV head.
//   o[t, h] = sum_j softmax_j(scale q[t, h] . K[j]) V[j], j over the rows [max(0, n - window), n) of n = ctx[t].
//
// A workgroup takes the rows of one (token, KV head, up to 16 of its query heads, slot): the token's rows are cut in slots of
// equal length, whose partials exact_join_kernel joins. Each of its waves walks tiles of kKeys rows of its own:
//   * a tile's K and V rows come by direct copies into LDS, a KB each, NB - 1 tiles ahead (the stream is what bounds the
//     kernel: 2d values per row and head are read once and meet 4 G d flops); the 16-byte pieces of a row lie swizzled, so
//     that both ways of reading them below touch every bank once;
//   * S^T[keys x 16 heads] = K Q^T on 16x16x32 bf16 products: K is the A operand (a row's pieces as they lie), Q^T stays in
//     registers; heads past the group's are zero columns, whose work is cheaper than the bytes;
//   * softmax in the exp2 domain, fp32, with a running maximum that is raised only when a score exceeds it by 2^8;
//   * O^T[d x 16 heads] += V^T P^T: P^T comes out of the scores' registers as the B operand, V^T is read by the transposing
//     LDS loads. bf16 tiles have 16 keys (16x16x16 products), e4m3 ones 32, in the order of keys that the two halves of the
//     scores have (16x16x32), and e4m3 values become bf16, exactly, on their way into the operands.
// P is rounded to bf16 for its product (half a step, 2^-9 of each weight; the output is bf16); sums are fp32.
#include <type_traits>

#include "common.h"

namespace hla {
namespace {

constexpr int kMaxTile = 16;     // query heads per workgroup
constexpr int kMaxSlots = 256;
constexpr float kRaise = 8.f;    // log2 by which a score may exceed the running maximum
// rows below which a slot is not worth a workgroup of its own (its partial is written and read once more)
constexpr int kMinRows = 64;

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
  int S;
  int64_t rows_wanted;     // workgroups that the rows of all tokens are spread over
  float *ws_o, *ws_lse;    // [T][H][S][D], [T][H][S]
  uint16_t* out;
  int64_t o_st, o_sh;
  float* lse;  // [H][T]
};

template <int kDim, bool kE4m3>
struct ExactGeo {
  static constexpr int D = kDim;
  static constexpr bool kE4 = kE4m3;
  static constexpr int ES = kE4 ? 1 : 2;
  static constexpr int KEYS = kE4 ? 32 : 16;
  static constexpr int RB = D * ES;              // bytes of a row's K (or V)
  static constexpr int CPR = RB / 16;            // pieces of 16 bytes in them
  static constexpr int RPI = 64 / CPR;           // rows per copy of a wave
  static constexpr int NI = KEYS / RPI;          // copies per tile, K and V each
  static constexpr int TILE = 2 * KEYS * RB;     // bytes of a tile
  static constexpr int NB = !kE4 && TILE <= 4096 ? 4 : 2;
  static constexpr int WAVES = TILE > 8192 ? 2 : 4;
  static constexpr int BATCH = 64 / KEYS;        // tiles whose row addresses are worked out at a time
  static_assert(NB <= BATCH, "page ids are requested a batch ahead and waited for with the tile before");
};

// Where the pieces of row x of a tile lie: piece c at c ^ swizzle(x). Both reads go over 256 bytes of banks at a time: K by 16
// lanes that take one piece of rows 0..15 (or 16..31), V by 32 lanes that take 32 bytes of rows 0..7 or 8..15 (bf16), or 16
// bytes of rows 0..7 and 16..23, or 8..15 and 24..31 (e4m3). Rows share the 256 bytes where they are shorter.
template <class G>
__device__ __forceinline__ int swizzle(int x) {
  if (G::kE4) {
    if (G::CPR == 4) return ((x >> 2) & 1) | ((((x >> 3) ^ (x >> 4)) & 1) << 1);
    if (G::CPR == 8) return ((x >> 1) & 3) | ((((x >> 3) ^ (x >> 4)) & 1) << 2);
    return (x & 7) | ((((x >> 3) ^ (x >> 4)) & 1) << 3);
  }
  if (G::CPR == 8) return (((x >> 1) & 3) << 1) | ((x >> 3) & 1);
  return ((x & 7) << 1) | ((x >> 3) & 1);
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

// Rows of a token: [first, n)
__device__ __forceinline__ void token_rows(const ExactCacheParams& a, int t, int& first, int& n) {
  n = (int)min((int64_t)max(a.ctx[t], 0), min((int64_t)a.bt_cols * a.block, (int64_t)INT32_MAX));
  first = a.window > 0 ? max(0, n - a.window) : 0;
}

// Rows per slot, the same for every token: no token has more than S slots, and the rows of all tokens and heads make about
// rows_wanted workgroups, however many rows the longest has. Each wave works it out by itself.
__device__ __forceinline__ int slot_rows(const ExactCacheParams& a, int lane, int step) {
  int64_t most = 0, sum = 0;
  for (int t = lane; t < a.T; t += 64) {
    int first, n;
    token_rows(a, t, first, n);
    most = max(most, (int64_t)(n - first));
    sum += n - first;
  }
  for (int off = 32; off > 0; off >>= 1) {
    most = max(most, __shfl_xor(most, off));
    sum += __shfl_xor(sum, off);
  }
  const int64_t share = (sum * a.KH * a.tiles + a.rows_wanted - 1) / a.rows_wanted;
  const int64_t rows = max(max((most + a.S - 1) / a.S, share), (int64_t)kMinRows);
  return (int)min((rows + step - 1) / step * step, (int64_t)INT32_MAX / 2);
}

template <class G>
__global__ __launch_bounds__(64 * G::WAVES) void exact_cache_kernel(ExactCacheParams a) {
  constexpr int D = G::D;
  constexpr bool kE4 = G::kE4;
  constexpr int KEYS = G::KEYS, RB = G::RB, CPR = G::CPR, RPI = G::RPI, NI = G::NI, NB = G::NB, WAVES = G::WAVES;
  constexpr int CT = D / 16;       // 16-column tiles of O^T
  constexpr int OS = D + 4;        // LDS row stride of a wave's partial output, in floats
  constexpr int kTiles = WAVES * NB * G::TILE, kJoin = WAVES * 16 * OS * 4;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kTiles > kJoin ? kTiles : kJoin];
  __shared__ int64_t offsets[WAVES][64];
  __shared__ int32_t page_ids[WAVES][64];
  __shared__ float stats[WAVES][2][16];

  const int tid = threadIdx.x, lane = tid & 63, x = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // item: heads innermost (workgroups dispatched one behind the other read the same rows' heads), then slots, then tokens
  int item = blockIdx.x;
  const int part = item % (a.KH * a.tiles);
  item /= a.KH * a.tiles;
  const int slot = item % a.S, t = item / a.S;
  const int kh = part / a.tiles, j0 = part % a.tiles * kMaxTile;
  const int heads = min(kMaxTile, a.G - j0), h0 = kh * a.G + j0;

  int first, n;
  token_rows(a, t, first, n);
  int lo = first, hi = n;
  if (a.S > 1) {
    const int rows = slot_rows(a, lane, WAVES * KEYS);
    lo = (int)min((int64_t)n, first + (int64_t)slot * rows);
    hi = (int)min((int64_t)n, (int64_t)lo + rows);
  }
  const int64_t base = (int64_t)t * a.H + h0;  // row of the workgroup's first head in [T][H]
  if (lo >= hi) {
    if (a.S > 1) {
      for (int j = tid; j < heads; j += 64 * WAVES) a.ws_lse[(base + j) * a.S + slot] = -INFINITY;
    } else {
      for (int i = tid; i < heads * (D / 8); i += 64 * WAVES)
        st16(a.out + (int64_t)t * a.o_st + (int64_t)(h0 + i / (D / 8)) * a.o_sh + i % (D / 8) * 8, u32x4{0u, 0u, 0u, 0u});
      for (int j = tid; j < heads; j += 64 * WAVES) a.lse[(int64_t)(h0 + j) * a.T + t] = -INFINITY;
    }
    return;
  }

  const int64_t row = a.bt_rows ? min(max(a.bt_rows[t], (int64_t)0), (int64_t)a.bt_count - 1) : t;
  const int32_t* btr = a.bt + row * a.bt_stride;
  const uint8_t* cache = a.cache + kh * a.head_stride;
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
  // tile i of the wave on its way into buffer i % NB
  auto request = [&](int i) {
    const uint8_t* buf = buf0 + i % NB * G::TILE;
#pragma unroll
    for (int c = 0; c < NI; ++c) {
      const int r = RPI * c + in_copy;
      const uint8_t* src = cache + offsets[wave][i % G::BATCH * KEYS + r] + 16 * (piece ^ swizzle<G>(r));
      copy16_to_lds_rfl_v(src, buf + 1024 * c);
      copy16_to_lds_rfl_v(src + RB, buf + KEYS * RB + 1024 * c);
    }
  };

  // Q^T: the columns of step s that lane group g holds are those of K's pieces
  u32x4 qo[D / 32];
  {
    const uint16_t* qp = a.q + (int64_t)t * a.q_st + (int64_t)(h0 + min(x, heads - 1)) * a.q_sh;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      const int col = kE4 ? 16 * (g + 4 * (s / 2)) + 8 * (s % 2) : 32 * s + 8 * g;
      qo[s] = x < heads ? ld16(qp + col) : u32x4{0u, 0u, 0u, 0u};
    }
  }
  const float scale = a.scale_log2 * (kE4 && a.k_scale ? a.k_scale[kh] : 1.f);

  float m = -INFINITY, l = 0.f;
  floatx4 o[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) o[c] = floatx4{0.f, 0.f, 0.f, 0.f};

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
      wait_copies<2 * NI * (NB - 1)>();
    } else {
      wait_copies<0>();
    }
    const uint8_t *kb = buf0 + i % NB * G::TILE, *vb = kb + KEYS * RB;

    constexpr int KB = KEYS / 16;
    floatx4 s[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      s[b] = floatx4{0.f, 0.f, 0.f, 0.f};
      const int key = 16 * b + x;
#pragma unroll
      for (int c = 0; c < CPR / 4; ++c) {
        const u32x4 v = ld16(kb + key * RB + 16 * ((4 * c + g) ^ swizzle<G>(key)));
        if (kE4) {
          s[b] = mfma16x16x32(e4m3_to_bf16(v[0], v[1]), qo[2 * c], s[b]);
          s[b] = mfma16x16x32(e4m3_to_bf16(v[2], v[3]), qo[2 * c + 1], s[b]);
        } else {
          s[b] = mfma16x16x32(v, qo[c], s[b]);
        }
      }
    }
    const int left = hi - (lo + (wave + i * WAVES) * KEYS);   // keys of the tile
    float top = -INFINITY;
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[b][r] = 16 * b + 4 * g + r < left ? s[b][r] * scale : -INFINITY;
        top = fmaxf(top, s[b][r]);
      }
    top = wave_max16x4(top);
    if (__any(top > m + kRaise)) {
      const float raised = fmaxf(m, top);
      const float alpha = raised == -INFINITY ? 1.f : fast_exp2(m - raised);
      m = raised;
      l *= alpha;
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[c][r] *= alpha;
    }
    const float at = m == -INFINITY ? 0.f : m;   // (nothing but scores of -inf so far: weights of zero)
    u32x2 p[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      float w[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) l += w[r] = fast_exp2(s[b][r] - at);
      p[b] = u32x2{pack2(w[0], w[1]), pack2(w[2], w[3])};
    }
    // the keys of a lane's values of V, in the order of the contraction: 4g .. and, e4m3, 16 + 4g ..
    auto sum_values = [&](auto last) {
      uint32_t seen[2] = {~0u, ~0u};   // rows past the last repeat it: their values count as 0 (0 * inf is not)
      if constexpr (decltype(last)::value) {
        if constexpr (kE4) {
          for (int b = 0; b < 2; ++b) {
            const int k = min(max(left - 16 * b - 4 * g, 0), 4);
            seen[b] = k == 4 ? ~0u : (1u << (8 * k)) - 1;
          }
        } else {
          const int k = min(max(left - 4 * g, 0), 4);
          seen[0] = k >= 2 ? ~0u : k == 1 ? 0xffffu : 0u;
          seen[1] = k >= 4 ? ~0u : k == 3 ? 0xffffu : 0u;
        }
      }
      if constexpr (kE4) {
        const u32x4 pt = u32x4{p[0][0], p[0][1], p[1][0], p[1][1]};
        // lane x of group g reads half a piece of key 4g + x/2 (x < 8) or 16 + 4g + x/2 - 4
        const int key = (x < 8 ? 0 : 12) + 4 * g + (x >> 1);
        const uint8_t* vr = vb + key * RB + 8 * (x & 1);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          typedef int int2v __attribute__((ext_vector_type(2)));
          const int2v v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (__attribute__((address_space(3))) int2v*)(vr + 16 * (c ^ swizzle<G>(key))));
          o[c] = mfma16x16x32(e4m3_to_bf16((uint32_t)v[0] & seen[0], (uint32_t)v[1] & seen[1]), pt, o[c]);
        }
      } else {
        const short4v pt = __builtin_bit_cast(short4v, p[0]);
        const int key = 4 * g + (x >> 2);
        const uint8_t* vr = vb + key * RB + 8 * (x & 1);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const short4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) short4v*)(vr + 16 * ((2 * c + ((x >> 1) & 1)) ^ swizzle<G>(key))));
          const u32x2 w = __builtin_bit_cast(u32x2, v);
          o[c] = mfma16x16x16(__builtin_bit_cast(short4v, u32x2{w[0] & seen[0], w[1] & seen[1]}), pt, o[c]);
        }
      }
    };
    if (left < KEYS) sum_values(std::true_type{});
    else sum_values(std::false_type{});
  }

  // the waves' parts together
  l = wave_sum16x4(l);
  if (g == 0) {
    stats[wave][0][x] = m;
    stats[wave][1][x] = l;
  }
  __syncthreads();   // (and every wave has read its last tile)
  float* joined = reinterpret_cast<float*>(lds);
  {
    float top = -INFINITY;
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stats[w][0][x]);
    const float f = m == -INFINITY ? 0.f : fast_exp2(m - top);
    // (a NaN among the scores is in l, and where m is -inf nothing but zeros and NaN are in o)
    if (x < heads) {
#pragma unroll
      for (int c = 0; c < CT; ++c) *reinterpret_cast<floatx4*>(joined + (wave * 16 + x) * OS + 16 * c + 4 * g) = o[c] * f;
    }
  }
  __syncthreads();
  for (int i = tid; i < heads * (D / 4); i += 64 * WAVES) {
    const int j = i / (D / 4), col = i % (D / 4) * 4;
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stats[w][0][j]);
    floatx4 v = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < WAVES; ++w) {
      const float mw = stats[w][0][j];
      sum += stats[w][1][j] * (mw == -INFINITY ? 0.f : fast_exp2(mw - top));
      v += *reinterpret_cast<floatx4*>(joined + (w * 16 + j) * OS + col);
    }
    const bool none = sum == 0.f;
    const float inv = none ? 0.f : (kE4 && a.v_scale ? a.v_scale[kh] : 1.f) / sum;
    const float lse = none ? -INFINITY : (top + log2f(sum)) * kLn2;
    if (a.S > 1) {
      *reinterpret_cast<floatx4*>(a.ws_o + ((base + j) * a.S + slot) * D + col) = v * inv;
      if (col == 0) a.ws_lse[(base + j) * a.S + slot] = lse;
    } else {
      *reinterpret_cast<u32x2*>(a.out + (int64_t)t * a.o_st + (int64_t)(h0 + j) * a.o_sh + col) =
          u32x2{pack2(v[0] * inv, v[1] * inv), pack2(v[2] * inv, v[3] * inv)};
      if (col == 0) a.lse[(int64_t)(h0 + j) * a.T + t] = lse;
    }
  }
}

// The slots of one (token, head) joined by their lse: one workgroup, D / 4 threads per slot.
template <int D>
__global__ __launch_bounds__(256) void exact_join_kernel(const float* ws_o, const float* ws_lse, int T, int H, int S,
                                                         uint16_t* out, int64_t o_st, int64_t o_sh, float* lse) {
  constexpr int PER = D / 4, ROWS = 256 / PER;
  __shared__ float weight[kMaxSlots];
  __shared__ floatx4 sums[ROWS][PER];
  __shared__ float red[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const float mine = tid < S ? ws_lse[row * S + tid] : -INFINITY;
  float top = mine;
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  if (lane == 0) red[0][wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  // (a slot with a NaN lse has a NaN weight; a slot without rows none, and its partial was not written)
  float w = mine == -INFINITY ? 0.f : fast_exp2((mine - top) * kLog2e);
  if (tid < S) weight[tid] = w;
  for (int off = 32; off > 0; off >>= 1) w += __shfl_xor(w, off);
  if (lane == 0) red[1][wave] = w;
  __syncthreads();
  const float sum = red[1][0] + red[1][1] + red[1][2] + red[1][3];
  floatx4 v = floatx4{0.f, 0.f, 0.f, 0.f};
  const float* src = ws_o + row * S * D + tid % PER * 4;
#pragma unroll 4
  for (int s = tid / PER; s < S; s += ROWS) {
    const float f = weight[s];
    if (f != 0.f) v += *reinterpret_cast<const floatx4*>(src + (int64_t)s * D) * f;
  }
  sums[tid / PER][tid % PER] = v;
  __syncthreads();
  if (tid >= PER) return;
  for (int i = 1; i < ROWS; ++i) v += sums[i][tid];
  const int t = (int)(row / H), h = (int)(row % H);
  const bool none = sum == 0.f;
  const float inv = none ? 0.f : 1.f / sum;
  *reinterpret_cast<u32x2*>(out + (int64_t)t * o_st + (int64_t)h * o_sh + 4 * tid) =
      u32x2{pack2(v[0] * inv, v[1] * inv), pack2(v[2] * inv, v[3] * inv)};
  if (tid == 0) lse[(int64_t)h * T + t] = none ? -INFINITY : top + logf(sum);
}

template <int D, bool kE4>
void launch_exact_cache(const ExactCacheParams& p, hipStream_t st) {
  const unsigned grid = (unsigned)((int64_t)p.T * p.S * p.KH * p.tiles);
  using G = ExactGeo<D, kE4>;
  hipLaunchKernelGGL(exact_cache_kernel<G>, dim3(grid), dim3(64 * G::WAVES), 0, st, p);
  if (p.S > 1)
    hipLaunchKernelGGL(exact_join_kernel<D>, dim3((unsigned)((int64_t)p.T * p.H)), dim3(256), 0, st, p.ws_o, p.ws_lse, p.T,
                       p.H, p.S, p.out, p.o_st, p.o_sh, p.lse);
}

// ---- store -------------------------------------------------------------------------------------------------------
// Rows into slots, a thread per 8 values (16 bytes in); e4m3: x / scale, clamped to +-448, to the nearest, ties to even.
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
    st16(dst + 2 * (half * a.D + 8 * c), v);
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
  *reinterpret_cast<u32x2*>(dst + half * a.D + 8 * c) =
      u32x2{four_e4m3(f[0], f[1], f[2], f[3]), four_e4m3(f[4], f[5], f[6], f[7])};
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
                                      const float* k_scale, const float* v_scale, int32_t num_splits, int32_t workgroups,
                                      float* workspace, int64_t workspace_floats, void* out, int64_t o_st, int64_t o_sh,
                                      float* lse, void* stream) {
  using namespace hla;
  HLA_REQUIRE(num_tokens >= 0, HLA_S6_EINVAL, "exact_attention: negative token count");
  int rc = check_exact_cache("exact_attention", cache, e4m3, head_dim, kv_heads, page_stride, head_stride, row_stride,
                             block_size, num_blocks);
  if (rc != HLA_S6_OK) return rc;
  HLA_REQUIRE(num_heads >= kv_heads && num_heads % kv_heads == 0, HLA_S6_EINVAL,
              "exact_attention: %d query heads over %d KV heads", num_heads, kv_heads);
  HLA_REQUIRE(num_splits >= 1 && num_splits <= kMaxSlots, HLA_S6_EINVAL, "exact_attention: %d splits (1..%d)", num_splits,
              kMaxSlots);
  HLA_REQUIRE(window >= 0 && bt_cols >= 0 && workgroups >= 1, HLA_S6_EINVAL, "exact_attention: bad window, table or grid");
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
  p.S = num_splits;
  p.rows_wanted = workgroups;
  HLA_REQUIRE((int64_t)p.T * p.S * p.KH * p.tiles <= INT32_MAX && (int64_t)p.T * p.H <= INT32_MAX, HLA_S6_EINVAL,
              "exact_attention: too many rows");
  if (p.S > 1) {
    const int64_t rows = (int64_t)p.T * p.H * p.S;
    HLA_REQUIRE(workspace && workspace_floats >= rows * (head_dim + 1), HLA_S6_EWORKSPACE,
                "exact_attention: workspace of %lld floats, need %lld", (long long)workspace_floats,
                (long long)(rows * (head_dim + 1)));
    HLA_REQUIRE(aligned16(workspace), HLA_S6_EINVAL, "exact_attention: workspace must be 16-byte aligned");
    p.ws_o = workspace;
    p.ws_lse = workspace + rows * head_dim;
  }
  p.out = static_cast<uint16_t*>(out);
  p.o_st = o_st;
  p.o_sh = o_sh;
  p.lse = lse;
  const hipStream_t st = as_stream(stream);
#define HLA_EXACT(D) e4m3 ? launch_exact_cache<D, true>(p, st) : launch_exact_cache<D, false>(p, st)
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
  HLA_REQUIRE(blocks <= INT32_MAX, HLA_S6_EINVAL, "exact_store: too many rows");
  const hipStream_t st = as_stream(stream);
  if (e4m3) hipLaunchKernelGGL(exact_store_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL(exact_store_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, st, p);
  return check_launch("exact_store");
}
