// The compact latent cache: rows [K | V] of 2 x W values in 4 bits each.
//
// A value is E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) times a power of two that a block of 32 columns
// shares: one byte, exponent + 127, which as the exponent field of an fp32 number is what the gfx950 conversions take
// (v_cvt_scalef32_pk_bf16_fp4: two values and their scale to two bf16 in one instruction, exact; a byte of 255 gives
// NaN). 17 W bytes hold a tile of 16 rows, in the order in which the matrix instructions read them. With x the row in the
// tile, b a block and two columns per byte (the even one in the low half):
//   K values [b / 4][x][b % 4][16 bytes]   8 W bytes: lane (x, g) of a wave loads block 4i + g of row x, so one load
//                                          instruction of 16 bytes per lane covers 1 KB of consecutive bytes
//   V values [x % 4][x / 4][W / 2 bytes]   8 W bytes: lane (m, g) loads row 4g + r, columns m * W / 16 and on
//   K scales [x][b % 4][b / 4]             W / 2 bytes: the W / 128 scales of lane (x, g) side by side
//   V scales [b][x]                        W / 2 bytes: the scales of rows 4g .. 4g + 3 side by side
#pragma once

#include "common.h"
#include "split_plan.h"

namespace hla {
namespace {

constexpr int kMinExponent = -120, kMaxExponent = 125;  // of a scale: every value of a block is then a normal bf16 or 0

__device__ __host__ __forceinline__ int64_t compact_tile_bytes(int W) { return 17 * (int64_t)W; }

// byte offsets in a tile: value bytes of block b (K: 16 consecutive bytes; V: column pair c / 2), scales of block b
__device__ __forceinline__ int k_code_at(int x, int b) { return (b >> 2) * 1024 + x * 64 + (b & 3) * 16; }
__device__ __forceinline__ int v_code_at(int W, int x, int byte) {
  return 8 * W + ((x & 3) * 4 + (x >> 2)) * (W >> 1) + byte;
}
__device__ __forceinline__ int k_scale_at(int W, int x, int b) {
  return 16 * W + x * (W >> 5) + (b & 3) * (W >> 7) + (b >> 2);
}
__device__ __forceinline__ int v_scale_at(int W, int x, int b) { return 16 * W + (W >> 1) + b * 16 + x; }

// scale byte i of a word as the fp32 number that the conversions take
__device__ __forceinline__ float scale_of(uint32_t word, int i) {
  return __uint_as_float(((word >> (8 * i)) & 255u) << 23);
}

// the two values of byte kByte of a word, as two bf16 (the even column in the low half)
template <int kByte>
__device__ __forceinline__ uint32_t two_bf16(uint32_t word, float scale) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, kByte));
}
// the eight values of a word
__device__ __forceinline__ u32x4 eight_bf16(uint32_t word, float scale) {
  return u32x4{two_bf16<0>(word, scale), two_bf16<1>(word, scale), two_bf16<2>(word, scale),
               two_bf16<3>(word, scale)};
}

// Inclusive sums and the maximum over a wave's lanes on DPP moves (within rows of 16, then row to row): no LDS round trip
template <int kCtrl, int kRows>
__device__ __forceinline__ int dpp_from(int v) {
  return __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_from<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v += dpp_from<0x112, 0xf>(v);
  v += dpp_from<0x114, 0xf>(v);
  v += dpp_from<0x118, 0xf>(v);
  v += dpp_from<0x142, 0xa>(v);  // row_bcast 15 into rows 1 and 3
  v += dpp_from<0x143, 0xc>(v);  // row_bcast 31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }
__device__ __forceinline__ int wave_max(int v) {  // of values that are not negative
  v = max(v, dpp_from<0x111, 0xf>(v));
  v = max(v, dpp_from<0x112, 0xf>(v));
  v = max(v, dpp_from<0x114, 0xf>(v));
  v = max(v, dpp_from<0x118, 0xf>(v));
  v = max(v, dpp_from<0x142, 0xa>(v));
  v = max(v, dpp_from<0x143, 0xc>(v));
  return __builtin_amdgcn_readlane(v, 63);
}

// page id of a table entry, in the cache whatever the entry holds
__device__ __forceinline__ int64_t clamp_page(int32_t page, int64_t num_blocks) {
  return min(max((int64_t)page, (int64_t)0), num_blocks - 1);
}

// A barrier that waits for this wave's accesses to LDS, and for none to memory
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
  plain_barrier();
}

template <int W, int NW = 4>
struct CompactGeo {
  static constexpr int KC = W / 128;              // 16-byte K pieces per lane and tile
  static constexpr int CH = W > 512 ? W / 512 : 1;  // waves that share a set of keys
  static constexpr int G = NW / CH;               // sets of keys per workgroup of NW waves
  static constexpr int CPL = W / CH / 16;         // V columns per lane
  static constexpr int VD = CPL / 8;              // dwords of V per lane and row
};

// 16 bytes, past the caches where nothing reads them again
template <bool kOnce>
__device__ __forceinline__ u32x4 ld_row(const void* p) {
  if constexpr (kOnce) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  else return ld16(p);
}

template <int N> struct Words { uint32_t w[N]; };

// N dwords from p (N * 4 bytes aligned)
template <int N, bool kOnce>
__device__ __forceinline__ Words<N> load_words(const uint8_t* p) {
  Words<N> r;
  if constexpr (N == 4) {
    const u32x4 v = ld_row<kOnce>(p);
    r.w[0] = v[0]; r.w[1] = v[1]; r.w[2] = v[2]; r.w[3] = v[3];
  } else if constexpr (N == 2) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    r.w[0] = v[0]; r.w[1] = v[1];
  } else {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  return r;
}

template <int W>
struct KTile {  // one tile of K: block 4i + g of row x per lane (x, g)
  u32x4 code[CompactGeo<W>::KC];
  uint32_t scale[(CompactGeo<W>::KC + 3) / 4];
};

template <int W, bool kOnce>
__device__ __forceinline__ void load_k(const uint8_t* tile, int x, int g, KTile<W>& k) {
  constexpr int KC = CompactGeo<W>::KC;
  const uint8_t* sp = tile + 16 * W + x * (W / 32) + g * KC;
  if constexpr (KC == 1) k.scale[0] = *sp;
  else if constexpr (KC == 2) k.scale[0] = *reinterpret_cast<const uint16_t*>(sp);
  else {
#pragma unroll
    for (int i = 0; i < KC / 4; ++i) k.scale[i] = reinterpret_cast<const uint32_t*>(sp)[i];
  }
#pragma unroll
  for (int i = 0; i < KC; ++i) k.code[i] = ld_row<kOnce>(tile + i * 1024 + x * 64 + g * 16);
}

// Q^T as the B operand in the column order of the K pieces: step 4i + j of lane (h, g) takes columns 32 (4i + g) + 8j
// .. + 8. In registers, or, from W = 512 on, where these would be 64 and more, in LDS (every wave of a workgroup reads the
// same; at 512 the history kernel then fits 256 registers and two workgroups a CU).
template <int W>
struct QOperand {
  static constexpr int N = CompactGeo<W>::KC * 4;
  static constexpr bool kLds = W >= 512;
  u32x4 r[kLds ? N / 4 : N];
  const u32x4 (*lds)[64];
  // the loads, before those of the first rows; with kLds each of the NW waves its share
  template <int NW>
  __device__ __forceinline__ void fetch(const uint16_t* q, int g, int wave) {
#pragma unroll
    for (int s = 0; s < (kLds ? N / NW : N); ++s) {
      const int x = kLds ? wave * (N / NW) + s : s;
      r[s] = ld16(q + 32 * (x / 4 * 4 + g) + 8 * (x % 4));
    }
  }
  // kLds: puts the shares together
  template <int NW>
  __device__ __forceinline__ void share(int wave, int lane, u32x4 (*buf)[64]) {
    if constexpr (kLds) {
#pragma unroll
      for (int s = 0; s < N / NW; ++s) buf[wave * (N / NW) + s][lane] = r[s];
      __syncthreads();
      lds = buf;
    }
  }
  __device__ __forceinline__ u32x4 at(int s, int lane) const {
    if constexpr (kLds) return lds[s][lane];
    else return r[s];
  }
};

// S^T of two tiles: column h of lane (h, g) holds keys 4g .. 4g + 3 of each. Each step of Q serves both; the products of
// the tiles alternate, so that neither waits for its own last one.
template <int W>
__device__ __forceinline__ void scores(const KTile<W> (&k)[2], const QOperand<W>& q, int lane, floatx4& s0, floatx4& s1) {
  s0 = s1 = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < CompactGeo<W>::KC; ++i) {
    const float f0 = scale_of(k[0].scale[i / 4], i % 4), f1 = scale_of(k[1].scale[i / 4], i % 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u32x4 qj = q.at(4 * i + j, lane);
      s0 = mfma16x16x32(eight_bf16(k[0].code[i][j], f0), qj, s0);
      s1 = mfma16x16x32(eight_bf16(k[1].code[i][j], f1), qj, s1);
    }
    // (no conversions ahead of their products, whose operands would not fit the registers)
    if constexpr (QOperand<W>::kLds) __builtin_amdgcn_sched_barrier(0);
  }
}

// ---- host checks ---------------------------------------------------------------------------------------------------
inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

inline bool known_width(int w) { return w == 128 || w == 256 || w == 512 || w == 1024; }

// Checks of a compact cache's geometry, shared by its entry points
int check_cache(const char* what, int width, const void* cache, int64_t page_stride, int block, int64_t num_blocks) {
  HLA_REQUIRE(known_width(width), HLA_S6_EUNSUPPORTED, "%s: latent width %d not in {128, 256, 512, 1024}", what, width);
  HLA_REQUIRE(block > 0 && block % kTile == 0, HLA_S6_EUNSUPPORTED, "%s: block size %d is not a positive multiple of 16",
              what, block);
  HLA_REQUIRE(num_blocks >= 1, HLA_S6_EINVAL, "%s: empty cache", what);
  HLA_REQUIRE(cache && aligned(cache, 16) && page_stride % 16 == 0 &&
                  page_stride >= block / kTile * compact_tile_bytes(width),
              HLA_S6_EINVAL, "%s: pages must be 16-byte aligned, whole and apart", what);
  return HLA_S6_OK;
}

}  // namespace
}  // namespace hla
