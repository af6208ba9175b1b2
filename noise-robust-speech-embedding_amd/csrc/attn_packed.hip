// Attention over packed sequences: rows of all sequences one behind another (or each sequence in its
// own padded stretch), grouped heads, full or causal, with an optional gated relative-position bias.
// For row i and key j of one sequence, query head h, key head h / G:
//   s_ij = scale q_i.k_j + g_i b[j - i]      P = softmax_j(s)      o_i = sum_j P_ij v_j
//   dV_j = sum_i P_ij dO_i   dP_ij = dO_i.v_j   dS = P (dP - delta_i), delta_i = sum_j P_ij dP_ij
//   dQ_i = scale sum_j dS_ij k_j   dK_j = scale sum_i dS_ij q_i   (dK, dV summed over the G heads)
//   dg_i = sum_j dS_ij b[j - i]    db[d] = sum over j - i = d of g_i dS_ij
//
// One workgroup = 4 waves = 128 rows (forward, dQ: queries; dK/dV: keys) of one sequence and head;
// one wave = 32 rows on the 32x32 matrix instructions, whose operand of 32 columns is the wave's own
// rows: S^T = K Q^T, so a softmax row is one lane and its neighbour 32 lanes on, and the
// probabilities leave the accumulators as the next product's operand without a shuffle (its inner
// index is taken in the accumulators' order: key 8 (r / 4) + 4 half + r % 4 for register r). The
// other side streams through LDS in tiles of 64 or 32 rows by LDS-DMA, one tile ahead. Each wave reads
// each tile once for its 32 columns: LDS reads (2 tiles x 4 waves) and matrix cycles are then about even
// at head_dim 128.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "common.h"
#include "overlap.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void_t;

constexpr int BQ = 128;       // keys of a dK/dV workgroup, rows of a forward or dQ one of one stream
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float INF = __builtin_huge_valf();
// Lazy rescaling: a row's probabilities are taken relative to a reference that only moves when a
// score passes it by more than 2^8; f32 sums hold values up to 2^8 as well as values up to 1.
constexpr float RESCALE_TAU = 8.f;
// A score is rounded where it stands relative to the reference, so a reference far below it (a row whose first keys
// are all masked by a large finite bias) would cost it bits of its own. A row has none, and is taken relative to
// zero, until a score passes -2^6: the distance then rounds off less than a score of 2^6 does itself. A row that ends
// without one is swept again relative to its largest score.
constexpr float FLOOR = -64.f;
// Under a bias, a row whose largest score is below -2^14 is taken to be left nothing: its keys are all masked by
// finite values, and what they hide is less than the last f32 bit of an lse, by which the backward rebuilds P.
constexpr float LEAST = -16384.f * LOG2E;

NRSE_DEV float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Rows of a streamed tile, for ST streams: 64 where registers and LDS leave the waves that hide its latency,
// else 32. bf16 at head_dim 128: 32 rows let a third wave onto a SIMD (8192 causal rows, forward 280 -> 260 us;
// 32 rows with two waves: 290). At head_dim 64, 32 rows and a fourth wave: no faster.
constexpr int tile_rows(int row_bytes, int es, int ST) {
  return row_bytes == 128 || (row_bytes == 256 && es == 4 && ST == 1) ? 64 : 32;
}
template <typename T, int D, int KT_>
struct Geo {
  static constexpr int RB = D * (int)sizeof(T);         // bytes of a row
  static constexpr int PANELS = RB / 128;               // a tile is kept in panels of 128-byte rows
  static constexpr int KT = KT_;                        // rows of a streamed tile
  static constexpr int TILE = KT * RB;                  // bytes of a tile
  static constexpr int NS = RB / 32;                    // 16-byte fragments of a row per lane half
  static constexpr int DT = D / 32;                     // 32-wide pieces of the head
  static constexpr int NT = KT / 32;                    // 32-row pieces of a tile
  static constexpr int DMA = KT / 8 * PANELS / 4;       // LDS-DMA instructions per wave and tile
  static constexpr int SEG = 192;                       // bias entries of a workgroup's tile, KT + 127, in 64s
};

// The forward and dQ kernels in ST streams, one or two: the 4 waves are 4 / ST pieces of 32 rows times ST streams,
// and stream i takes every ST-th key tile, its running maximum, sum and output joined with the others' in
// LDS at the end. A workgroup then has 128 / ST rows: more of them, each ST times shorter.
template <typename T, int D, int ST>
struct QGeo : Geo<T, D, tile_rows(D * (int)sizeof(T), (int)sizeof(T), ST)> {
  using B = Geo<T, D, tile_rows(D * (int)sizeof(T), (int)sizeof(T), ST)>;
  static constexpr int BR = 128 / ST;                               // rows of a workgroup
  static_assert(ST == 1 || ST == 2, "streams");
  static constexpr int SEG = ST == 1 ? 192 : 128;                   // >= KT + BR - 1, in 64s
  static_assert(SEG >= B::KT + BR - 1 && SEG * ST <= 256, "a bias entry per thread");
  static constexpr int BUF = 2 * B::TILE;                           // K and V tile
  static constexpr int KV_LDS = ST * 2 * BUF;                       // [ST][2 buffers]
  // of the forward, per SIMD: what the registers leave (more would spill)
  static constexpr int waves(bool bias) {
    return ST == 1 && (B::RB == 128 || (D == 128 && sizeof(T) == 2 && !bias)) ? 3 : 2;
  }
  static constexpr int Q_WAVES = B::RB > 256 ? 1 : 2;               // of dQ (three at 128-byte rows: no faster)
};

// LDS of dQ, and of the forward, which has a float for each row and stream behind it
template <typename G>
__host__ __device__ constexpr size_t lds_q(bool bias) {
  return G::KV_LDS + (bias ? G::KV_LDS / (2 * G::BUF) * 8 * G::SEG * sizeof(float) : 0);
}
template <typename G>
__host__ __device__ constexpr size_t lds_q_fwd(bool bias) { return lds_q<G>(bias) + 128 * sizeof(float); }

// ---------------------------------------------------------------------------------- LDS tiles
// Row r of a panel holds its 16-byte chunk c at position c ^ sw(r), sw(r) the three bits of (r / 2) % 8 in
// reverse. A 16-lane phase of a b128 row read takes one chunk of 8 pairs of rows, r / 2 all different
// mod 8; a transposed read takes 4 chunks of 4 rows, and the lowest bit of r / 2, moved to the top of the
// position, puts one pair of rows on each half of the panel: both then meet every bank once.
// (With two bits, ((r / 2) % 4) * 2, half of the LDS cycles were conflicts.)
NRSE_DEV int sw(int row) { return ((row & 2) << 1) | ((row & 4) >> 1) | ((row & 8) >> 3); }
template <int KT>
NRSE_DEV int loff(int row, int chunk) {
  return (chunk >> 3) * (KT * 128) + row * 128 + (((chunk & 7) ^ sw(row)) << 4);
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// A lane's places in a tile. Everything but the 16-byte chunk's swizzle is a constant offset from
// them (a 32-row piece or a panel does not change it), so a read is one of these plus an immediate.
template <typename T, typename G>
struct Lds {
  int row[4];  // row m, chunk 2 c + half of a panel, c = 0 .. 3
  int col[4];  // inner index down the rows: bf16 see rd_col; f32 see mma_col
  NRSE_DEV void init(int lane) {
    const int m = lane & 31, half = lane >> 5;
#pragma unroll
    for (int c = 0; c < 4; ++c) row[c] = loff<G::KT>(m, 2 * c + half);
    if constexpr (std::is_same_v<T, bf16_t>) {
      const int g = lane >> 4, i = lane & 15;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        col[e] = loff<G::KT>(4 * (g >> 1) + (i >> 2) + 8 * (e >> 1), 4 * (e & 1) + 2 * (g & 1) + ((i & 3) >> 1)) + (i & 1) * 8;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        col[e] = (4 * half) * 128 + (((m >> 2) ^ (half << 1) ^ (e & 1) ^ ((e & 2) << 1)) << 4) + (m & 3) * 4;
    }
  }
  // 16 bytes of row 32 t + m, fragment c
  NRSE_DEV u32x4 rd_row(const char* tile, int t, int c) const {
    return *reinterpret_cast<const u32x4*>(tile + row[c & 3] + (c >> 2) * (G::KT * 128) + 32 * t * 128);
  }
  // bf16 operand with its inner index down the rows: lane (m, half) gets column 32 dt + m of rows
  // r0 + 4 half .. + 3 and r0 + 8 + 4 half .. + 3 (r0 a multiple of 16: the swizzle repeats every 16 rows)
  NRSE_DEV bf16x8 rd_col(const char* tile, int r0, int dt) const {
    const char* a = tile + (dt >> 1) * (G::KT * 128) + r0 * 128;
    const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(a + col[dt & 1]));
    const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(a + col[2 + (dt & 1)]));
    const short8v v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8, v);
  }
};

NRSE_DEV bf16x8 pack8(const float* a) {
  bf16x8 v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (__bf16)a[j];
  return v;
}

// acc += A B over one 16-byte fragment of the inner index (8 bf16 or 4 f32 per lane half)
template <typename T>
NRSE_DEV void mma_row(u32x4 a, u32x4 b, f32x16& acc) {
  if constexpr (std::is_same_v<T, bf16_t>) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[c]), __uint_as_float(b[c]), acc, 0, 0, 0);
  }
}

// acc[dt] += X^T P for a 32-row piece of the tile at `t` (rows r0 ..): X^T from the tile, P the 16
// registers of a 32x32 accumulator (rounded to bf16 for the bf16 product: relative 2^-8 per
// probability at most, as every bf16 operand)
template <typename T, typename G>
NRSE_DEV void mma_col(const Lds<T, G>& L, const char* t, int r0, const float* p, f32x16* acc, int lane) {
  if constexpr (std::is_same_v<T, bf16_t>) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const bf16x8 b = pack8(p + 8 * ks);
#pragma unroll
      for (int dt = 0; dt < G::DT; ++dt)
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(L.rd_col(t, r0 + 16 * ks, dt), b, acc[dt], 0, 0, 0);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      // row r0 + 8 (r / 4) + 4 half + r % 4, column 32 dt + m: of the row's swizzle, half's bit is in col, the
      // lowest bits of r / 2 and r / 4 choose one of its four
      const int at = (r0 + 8 * (r >> 2) + (r & 3)) * 128 + L.col[((r >> 2) & 1) + (r & 2)];
#pragma unroll
      for (int dt = 0; dt < G::DT; ++dt) {
        const float a = *reinterpret_cast<const float*>(t + dt * (G::KT * 128) + at);
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], acc[dt], 0, 0, 0);
      }
    }
  }
}

// The same with P in two bf16 parts, its upper 16 bits and the rest, for dQ: the dS of a row sum to zero, so
// where the keys share a direction dQ is a small difference of large terms, and one rounding of each dS to
// bf16 was most of its error (causal bf16 batch, error over norm: dQ 2.9e-3 in one part, 2.3e-3 in two, 1.7e-3
// of it the output's own rounding). A third more matrix work in this kernel: backward + 4 %.
template <typename T, typename G>
NRSE_DEV void mma_col_split(const Lds<T, G>& L, const char* t, int r0, const float* p, f32x16* acc, int lane) {
  if constexpr (std::is_same_v<T, bf16_t>) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      u32x4 hi;
      float lo[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned a = __float_as_uint(p[8 * ks + 2 * j]), b = __float_as_uint(p[8 * ks + 2 * j + 1]);
        hi[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        lo[2 * j] = p[8 * ks + 2 * j] - __uint_as_float(a & 0xffff0000u);
        lo[2 * j + 1] = p[8 * ks + 2 * j + 1] - __uint_as_float(b & 0xffff0000u);
      }
      const bf16x8 bh = __builtin_bit_cast(bf16x8, hi), bl = pack8(lo);
      bf16x8 a[G::DT];
#pragma unroll
      for (int dt = 0; dt < G::DT; ++dt) {
        a[dt] = L.rd_col(t, r0 + 16 * ks, dt);
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[dt], bh, acc[dt], 0, 0, 0);
      }
#pragma unroll
      for (int dt = 0; dt < G::DT; ++dt) acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[dt], bl, acc[dt], 0, 0, 0);
    }
  } else {
    mma_col<T, G>(L, t, r0, p, acc, lane);
  }
}

// ---------------------------------------------------------------------------------- LDS-DMA
// A wave instruction moves 8 rows of a panel (1 KiB): lane l brings row l / 8, position l % 8, that is
// the logical chunk (l % 8) ^ sw(row), so the swizzle goes into the source address. The descriptor
// is made per tile (64-bit base: a long sequence's rows pass 32 bits of offset) and ends behind the
// tile's last row of the sequence: rows past the end land as zeros and nothing behind them is read.
template <typename T, typename G>
struct Dma {
  const char* base;   // row 0 of the sequence
  long long ld;       // bytes between rows
  int len;
  unsigned even, odd;   // a lane's source, in 8-row groups of even and of odd number
  NRSE_DEV void init(const void* p, long long ld_elems, int len_, int lane) {
    base = (const char*)p;
    ld = ld_elems * (long long)sizeof(T);
    len = len_;
    const int row = lane >> 3;
    even = (unsigned)row * (unsigned)ld + (unsigned)(((lane & 7) ^ sw(row)) << 4);
    odd = (unsigned)row * (unsigned)ld + (unsigned)(((lane & 7) ^ sw(row + 8)) << 4);
  }
  // head: byte offset of the head
  NRSE_DEV void issue(char* tile, int row0, int wave, long long head = 0) const {
    const int n = min(G::KT, len - row0);
    const unsigned ldu = (unsigned)ld;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(base + head + (long long)row0 * ld), 0, n > 0 ? (int)((unsigned)(n - 1) * ldu + G::RB) : 0, 0x00020000);
#pragma unroll
    for (int j = 0; j < G::DMA; ++j) {
      const int k = wave * G::DMA + j;
      const int panel = k % G::PANELS, rg = k / G::PANELS;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(tile + panel * (G::KT * 128) + rg * 1024), 16,
                                               ((rg & 1) ? odd : even) + (unsigned)(rg * 8) * ldu + (unsigned)(panel * 128), 0, 0, 0);
    }
  }
};

// ---------------------------------------------------------------------------------- which rows
// The blocks of all sequences are numbered from the longest sequences' last blocks down: a block's work
// grows with its sequence and, under a causal mask, with its place, so the long ones start first and the short
// ones fill the end. "Longest" by classes, each three quarters of the one before, of 64 sequences at a time, a
// lane each: a place among them is a scan or two. (Against the batch's own order: 16 utterances, backward
// 134 -> 113 us; 6 causal sequences, the longest last in that order, 162 -> 153. An exact order by 64 steps of
// comparing: 64 sequences of 30 rows, forward 8 -> 20 us.) Every workgroup walks the sequences before its own, 64 at a
// time, so with thousands of them the walk is most of the time: 8 heads of 64, sequences of 20 rows, 64 of them 7 us,
// 1000 76, 4000 654. The grid is sized from what the host knows, rows / BR +
// sequences, and what is left over ends at once.
// Bounds are taken from cu_seqlens as they stand in device memory, clamped to the tensors.
struct Block { int seq0, len, row0; bool any; };

// lane i: f over lanes 0 .. i, of values for which 0 is neutral. In rows of 16 lanes, then row 0's last into row 1 and 2's
// into 3, then lane 31's into both of the upper rows.
template <typename F>
NRSE_DEV int wave_scan(int x, F f) {
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true));   // row_shr 1, 2, 4, 8
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, true));   // row_bcast 15, 31
  return f(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, true));
}
struct Add { NRSE_DEV int operator()(int a, int b) const { return a + b; } };
struct Max { NRSE_DEV int operator()(int a, int b) const { return max(a, b); } };

template <int BR>
NRSE_DEV Block find_block(const int* __restrict__ cu, const int* __restrict__ used, int nseq, int rows, int want) {
  const int lane = threadIdx.x & 63;
  int before = 0, from = 0, to = 0, own = rows;
  auto fetch = [&](int base) {   // a lane's sequence of those at `base`; none: an empty one
    const int s = min(base + lane, nseq - 1);
    from = cu[s];
    to = cu[s + 1];
    own = used ? used[s] : rows;
    if (base + lane >= nseq) own = 0;
  };
  if (nseq > 0) fetch(0);
  for (int base = 0; base < nseq; base += 64) {
    const int start = min(max(from, 0), rows);
    const int len = min(min(max(to, start), rows) - start, max(own, 0));
    const int nb = (len + BR - 1) / BR;
    if (nseq > 64) {
      if (base + 64 < nseq) fetch(base + 64);
      const int all = __builtin_amdgcn_readlane(wave_scan(nb, Add()), 63);
      if (want >= before + all) {
        before += all;
        continue;
      }
    }
    int hi = __builtin_amdgcn_readlane(wave_scan(len, Max()), 63);
    for (int c = 0; c < 8; ++c) {
      const int lo = c == 7 ? 0 : hi - (hi >> 2) - 1;
      const int last = before + wave_scan(len <= hi && len > lo ? nb : 0, Add());   // (one behind a lane's last block)
      const unsigned long long hit = __builtin_amdgcn_ballot_w64(last > want);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        return Block{__builtin_amdgcn_readlane(start, l), __builtin_amdgcn_readlane(len, l),
                     (__builtin_amdgcn_readlane(last, l) - 1 - want) * BR, true};
      }
      before = __builtin_amdgcn_readlane(last, 63);
      hi = lo;
    }
  }
  return Block{0, 0, 0, false};
}

// Workgroup i runs on XCD i % 8 (each with its own L2): the XCDs share out the key heads, and where
// there are fewer than 8 the blocks, so that the G query heads of a block and the blocks of a sequence
// meet the same K and V in one L2. The blocks, which get shorter, are dealt out to and fro, so that no XCD
// has the longer one every time (3 causal sequences over 2 key heads, backward 227 -> 214 us).
struct Place { int block, kvh, g; };
__host__ __device__ inline int gcd8(int n) { return (n & 7) == 0 ? 8 : (n & 3) == 0 ? 4 : (n & 1) == 0 ? 2 : 1; }
NRSE_DEV Place place(int nblk, int hkv, int G) {
  const int gc = gcd8(hkv), nsub = 8 / gc;
  const int xcd = blockIdx.x & 7, local = blockIdx.x >> 3;
  const int per = (nblk + nsub - 1) / nsub * G;
  const int r = local % per;
  const int turn = r / G, sub = xcd / gc;
  return Place{turn * nsub + ((turn & 1) ? nsub - 1 - sub : sub), (xcd % gc) * (hkv / gc) + local / per, r % G};
}
inline long long grid_size(long long nblk, int hkv, int G) {
  const int gc = gcd8(hkv), nsub = 8 / gc;
  return 8LL * ((nblk + nsub - 1) / nsub) * G * (hkv / gc);
}

// ---------------------------------------------------------------------------------- the bias
// The entries of the Toeplitz vector that a workgroup's tile touches, as 4 copies shifted by 0 .. 3, so
// that a lane's 4 consecutive entries are one aligned 16-byte read; copy s is rotated by 16 s floats
// inside 64-float blocks, which puts the copies' equal places on different banks.
NRSE_DEV int bv_pos(int j, int s) { return (j & ~63) | ((j + 16 * s) & 63); }
template <int SEG>
NRSE_DEV void bv_store(float* bv, int tid, float v) {
  if (tid < SEG) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (tid >= s) bv[s * SEG + bv_pos(tid - s, s)] = v;
  }
}
NRSE_DEV float bv_load(const float* __restrict__ vec, int nd, int e) {
  const float v = vec[min(max(e, 0), nd - 1)];
  return (e >= 0 && e < nd) ? v : 0.f;
}

template <typename T>
NRSE_DEV void store4(T* p, float a, float b, float c, float d) {
  if constexpr (std::is_same_v<T, bf16_t>) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<bf16x4*>(p) = bf16x4{(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
  }
}

// The lane's number, formed where it is used: what is derived from it does not take registers through a loop.
NRSE_DEV int lane_again() {
  int zero = 0;
  asm volatile("" : "+s"(zero));
  return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero));
}

NRSE_DEV void wait_all_and_meet() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---------------------------------------------------------------------------------- forward
// Bound by the matrix units where there are rows enough (bf16): 8192 causal rows, 16 heads of 128 over 2,
// 256-278 us on several cards = 990-1075 TF (the matrix units busy 65 % of the time, no LDS conflicts, the rest exp and
// sums beside them); long full sequences 1117 TF at 128, 941 at 64. Ragged batches are bound by each workgroup's own
// latency and by the last ones to end: 4096 causal rows in 6 sequences, 16 heads of 128 over 4, 45 us; 16 utterances
// of 149 to 599 rows, 16 heads of 64 with a bias, 31 us (matrix units 21 % busy, waves waiting 48 %). f32 is 16 times
// as much matrix time a product: 1193 rows, 8 heads of 64, 31 us. A few single-token prompts: 6.3 us, the launch.
// The second sweep, where it is needed, doubles a workgroup's time; asking whether it is, a barrier and two LDS reads,
// takes up to 0.3 us of a call.
template <typename T, int D, bool BIAS, bool CAUSAL, int ST>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(QGeo<T, D, ST>::waves(BIAS), QGeo<T, D, ST>::waves(BIAS)))) void fwd_kernel(const nrse_attn_packed_fwd_params p) {
  using G = QGeo<T, D, ST>;
  constexpr int KT = G::KT;
  extern __shared__ __attribute__((aligned(16))) char dyn[];
  float* const bv0 = reinterpret_cast<float*>(dyn + G::KV_LDS);  // [ST][2][4][SEG]
  const int group = p.hq / p.hkv;
  const int nblk = (int)(p.rows / G::BR) + p.nseq;
  const Place pl = place(nblk, p.hkv, group);
  if (pl.block >= nblk) return;
  const Block bl = find_block<G::BR>(p.cu_seqlens, p.seq_lens, p.nseq, (int)p.rows, pl.block);
  if (!bl.any) return;
  const int h = pl.kvh * group + pl.g, len = bl.len;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 31, half = lane >> 5;
  Lds<T, G> L;
  L.init(lane);
  const int st = w / (4 / ST), sub = w % (4 / ST);
  const int q0 = bl.row0 + sub * 32;     // this wave's first row in the sequence
  const int qi = q0 + m;
  const bool live = q0 < len;            // a wave past the end keeps its share of the copies and the barriers
  Dma<T, G> kd, vd;
  kd.init((const T*)p.k + (long long)bl.seq0 * p.k_row + pl.kvh * p.k_head, p.k_row, len, lane);
  vd.init((const T*)p.v + (long long)bl.seq0 * p.v_row + pl.kvh * p.v_head, p.v_row, len, lane);
  const int kend = CAUSAL ? min(len, bl.row0 + G::BR) : len;
  const int ntiles = (kend + KT - 1) / KT, nit = (ntiles + ST - 1) / ST;
  auto issue = [&](int it) {   // start bringing every stream's tile of iteration `it`
#pragma unroll
    for (int i = 0; i < ST; ++i) {
      char* const K = dyn + (i * 2 + (it & 1)) * G::BUF;
      kd.issue(K, (it * ST + i) * KT, w);
      vd.issue(K + G::TILE, (it * ST + i) * KT, w);
    }
  };
  issue(0);
  const int nd = 2 * p.bias_len - 1;
  const float* vec = BIAS ? p.bias_vec + (long long)h * nd : nullptr;
  // segment entry j of the tile at key kb: b[kb - row0 + j - (BR - 1)]; a thread brings one entry of its
  // stream's segment
  const int bst = ST == 1 ? 0 : tid / G::SEG, bt = ST == 1 ? tid : tid % G::SEG;
  const int e0 = p.bias_len - 1 - bl.row0 - (G::BR - 1) + bst * KT + bt;
  float bnext = 0.f;
  if constexpr (BIAS) bv_store<G::SEG>(bv0 + bst * 8 * G::SEG, bt, bv_load(vec, nd, e0));
  u32x4 qf[G::NS];
  const int qc = min(qi, len - 1);       // loads from a row that is there, zeroed after
  auto load_q = [&]() {   // (and again before a second sweep: kept for that, registers ran out at head_dim 128)
    const int ln = lane_again(), i = q0 + (ln & 31);
    const T* qrow = (const T*)p.q + (long long)(bl.seq0 + min(i, len - 1)) * p.q_row + h * p.q_head;
#pragma unroll
    for (int s = 0; s < G::NS; ++s) {
      qf[s] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(qrow) + (2 * s + (ln >> 5)) * 16);
      if (i >= len) qf[s] = u32x4{0, 0, 0, 0};
    }
  };
  load_q();
  const float c1 = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(p.scale * LOG2E)));   // (a scalar register)
  float gl = LOG2E;
  if constexpr (BIAS) {
    if (p.gate) gl = p.gate[h * p.rows + bl.seq0 + qc] * LOG2E;
  }
  const int u0 = 4 * half + G::BR - 1 - (sub * 32 + m);
  const float* const bcopy = bv0 + st * 8 * G::SEG + (u0 & 3) * G::SEG;
  const int uj = u0 - (u0 & 3), us = u0 & 3;

  // thr: RESCALE_TAU once the row has a reference, its largest score (-inf: none) until then
  float mref = 0.f, thr = -INF, lsum;
  f32x16 o[G::DT];

  auto tile = [&](const int it, auto masked_c) {
    constexpr bool MASKED = decltype(masked_c)::value;
    const int kb = (it * ST + st) * KT;
    char* const Kt = dyn + (st * 2 + (it & 1)) * G::BUF;
    char* const Vt = Kt + G::TILE;
    wait_all_and_meet();
    float4 bb[G::NT][4];
    if constexpr (BIAS) {
      // this tile's entries before the next tile's copies are issued (the compiler cannot tell the LDS
      // that they write from what is read here, and would wait for them)
#pragma unroll
      for (int t = 0; t < G::NT; ++t)
#pragma unroll
        for (int a = 0; a < 4; ++a)
          bb[t][a] = *reinterpret_cast<const float4*>(bcopy + (it & 1) * 4 * G::SEG + bv_pos(uj + 32 * t + 8 * a, us));
    }
    if (it + 1 < nit) {
      issue(it + 1);
      if constexpr (BIAS) bnext = bv_load(vec, nd, e0 + (it + 1) * ST * KT);
    }
    if (live && (ST == 1 || kb < kend) && (!CAUSAL || kb <= q0 + 31)) {
      float v[G::NT][16];
      f32x16 sv[G::NT];
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < G::NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) sv[t][r] = 0.f;
#pragma unroll
      for (int c = 0; c < G::NS; ++c)   // (the pieces' products in turn: none waits for the one before it)
#pragma unroll
        for (int t = 0; t < G::NT; ++t) mma_row<T>(L.rd_row(Kt, t, c), qf[c], sv[t]);
      if constexpr (sizeof(T) == 2) {
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < G::NS * G::NT - 4; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
      }
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < G::NT; ++t) {
        const f32x16& s = sv[t];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          if constexpr (BIAS) {
            v[t][4 * a + 0] = fmaf(s[4 * a + 0], c1, fmaf(gl, bb[t][a].x, -mref));
            v[t][4 * a + 1] = fmaf(s[4 * a + 1], c1, fmaf(gl, bb[t][a].y, -mref));
            v[t][4 * a + 2] = fmaf(s[4 * a + 2], c1, fmaf(gl, bb[t][a].z, -mref));
            v[t][4 * a + 3] = fmaf(s[4 * a + 3], c1, fmaf(gl, bb[t][a].w, -mref));
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[t][4 * a + c] = fmaf(s[4 * a + c], c1, -mref);
          }
        }
      }
      if constexpr (MASKED) {
        // keys past the end or, under the causal mask, behind the query
        const int last = CAUSAL ? min(len - 1, qi) : len - 1;
#pragma unroll
        for (int t = 0; t < G::NT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            v[t][r] = kb + 32 * t + 8 * (r >> 2) + 4 * half + (r & 3) <= last ? v[t][r] : -INF;
      }
      float m4[4] = {v[0][0], v[0][1], v[0][2], v[0][3]};   // (four chains: each step waits for its last)
#pragma unroll
      for (int t = 0; t < G::NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 2) m4[(r >> 1) & 3] = fmaxf(fmaxf(m4[(r >> 1) & 3], v[t][r]), v[t][r + 1]);
      const float mx = xor32_max(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
      if (__builtin_amdgcn_ballot_w64(mx > thr)) {
        const bool first = thr < 0.f, low = first && mx <= FLOOR;
        const float sh = low ? 0.f : first ? mx : fmaxf(mx, 0.f);
        const float al = exp2_(-sh);
        thr = low ? fmaxf(thr, mx) : RESCALE_TAU;
        mref += sh;
        lsum *= al;
#pragma unroll
        for (int t = 0; t < G::NT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) v[t][r] -= sh;
#pragma unroll
        for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= al;
      }
#pragma unroll
      for (int t = 0; t < G::NT; ++t) {
        float part[4];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          v[t][r] = exp2_(v[t][r]);
          part[r & 3] = r < 4 ? v[t][r] : part[r & 3] + v[t][r];
        }
        lsum += (part[0] + part[1]) + (part[2] + part[3]);
        mma_col<T, G>(L, Vt, 32 * t, v[t], o, lane);
      }
    }
    if constexpr (BIAS) {
      if (it + 1 < nit) bv_store<G::SEG>(bv0 + (bst * 2 + ((it + 1) & 1)) * 4 * G::SEG, bt, bnext);
    }
  };
  // tiles that every row of the workgroup sees whole, then those with a mask
  const int nfull = min(len, CAUSAL ? bl.row0 + 1 : len) / (KT * ST);
  auto empty = [&]() {
    lsum = 0.f;
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  };
  empty();
  for (bool again = false;; again = true) {
    for (int it = 0; it < nfull; ++it) tile(it, std::false_type{});
    for (int it = nfull; it < nit; ++it) tile(it, std::true_type{});
    if (again) break;
    // once more, where a row of the workgroup has no reference in any stream, but a score to take for one. (Every wave
    // looks at all rows, so that all decide the same.)
    float* const best = reinterpret_cast<float*>(dyn + lds_q_fwd<G>(BIAS)) - 128;   // [ST][BR]
    const int ln = lane_again();
    if (ln < 32) best[st * G::BR + sub * 32 + ln] = q0 + ln < len ? thr : 0.f;
    __syncthreads();
    float b = ST == 1 ? best[ln] : fmaxf(best[ln], best[64 + ln]);
    bool redo = b < 0.f && b > (BIAS ? LEAST : -INF);
    if constexpr (ST == 1) {
      b = best[64 + ln];
      redo |= b < 0.f && b > (BIAS ? LEAST : -INF);
    }
    if (!__builtin_amdgcn_ballot_w64(redo)) break;
    if (thr < 0.f && thr > (BIAS ? LEAST : -INF)) {
      mref = thr;
      thr = RESCALE_TAU;
    }
    empty();
    load_q();
    issue(0);
    if constexpr (BIAS) bv_store<G::SEG>(bv0 + bst * 8 * G::SEG, bt, bv_load(vec, nd, e0));
  }

  float l = xor32_sum(lsum);
  bool none = thr < 0.f;
  if constexpr (ST > 1) {
    // join: out = sum 2^(m_i - M) o_i over the streams, in stream order
    float* const js = reinterpret_cast<float*>(dyn);
    constexpr int PER = (D / 2 + 2) * 64;   // a wave's accumulators, maximum and sum
    float* const at = js + ((st - 1) * (4 / ST) + sub) * PER + lane;
    const float mine = thr < 0.f ? -INF : mref;   // (-inf: relative to zero)
    __syncthreads();
    if (st > 0) {
#pragma unroll
      for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) at[(dt * 16 + r) * 64] = o[dt][r];
      at[(D / 2) * 64] = mine;
      at[(D / 2 + 1) * 64] = l;
    }
    __syncthreads();
    if (st > 0) return;
    const float* from = js + sub * PER + lane;
    float M = mine;
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) M = fmaxf(M, from[i * (4 / ST) * PER + (D / 2) * 64]);
    none = !(M > -INF);
    // (a stream without a reference: relative to zero, and nothing in it where M is below FLOOR)
    const float a0 = none ? 0.f : exp2_(fminf(mref - M, -FLOOR));
    l *= a0;
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] *= a0;
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      const float* const x = from + i * (4 / ST) * PER;
      const float mi = x[(D / 2) * 64];
      const float a = none ? 0.f : exp2_(fminf((mi > -INF ? mi : 0.f) - M, -FLOOR));
      l = fmaf(a, x[(D / 2 + 1) * 64], l);
#pragma unroll
      for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] = fmaf(a, x[(dt * 16 + r) * 64], o[dt][r]);
    }
    mref = none ? 0.f : M;
  }
  const int ln = lane_again(), row = q0 + (ln & 31);
  if (row >= len) return;
  // a row whose bias leaves nothing: zeros; not one of NaN, whose sum is a NaN and no small number (seen by its bits: the
  // compiler is told not to expect NaN)
  none = none && __float_as_uint(l) < 0x40000000u;
  const float inv = 1.f / l;
#pragma unroll
  for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = none ? 0.f : o[dt][r] * inv;   // (a masked key's infinite value may be in its sums)
  T* const orow = (T*)p.out + (long long)(bl.seq0 + row) * p.out_row + h * p.out_head + 4 * (ln >> 5);
#pragma unroll
  for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      store4<T>(orow + 32 * dt + 8 * a, o[dt][4 * a], o[dt][4 * a + 1], o[dt][4 * a + 2], o[dt][4 * a + 3]);
  if (p.lse && ln < 32)
    p.lse[h * p.rows + bl.seq0 + row] = none ? -INF : (mref + __builtin_amdgcn_logf(l)) * LN2;
}

// ---------------------------------------------------------------------------------- backward: dQ, dgate
// The forward's loop with P rebuilt from lse; also delta_i, which the dK/dV kernel reads after it. Here
// delta is rowsum(dO O), from the stored output. The gradients of bias and gate are f32 outputs, and the
// rounding of a bf16 O would be all their error (and a quarter of dK's): for what follows delta is summed again as
// sum_j P dP from the f32 accumulators (EXACT), and dgate = sum P dP b - delta sum P b.
// The forward's batches: 70-74 us (4096 causal rows), 51-53 us (utterances), 46 us (f32). It holds Q, dO, S and dP beside dQ, so
// two waves per SIMD; what bounds it is the latency of one tile's chain of products and exponentials.
template <typename T, int D, bool BIAS, bool CAUSAL, int ST>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(QGeo<T, D, ST>::Q_WAVES, QGeo<T, D, ST>::Q_WAVES))) void bwd_q_kernel(const nrse_attn_packed_bwd_params p) {
  using G = QGeo<T, D, ST>;
  constexpr int KT = G::KT;
  constexpr bool EXACT = BIAS || sizeof(T) == 2;
  extern __shared__ __attribute__((aligned(16))) char dyn[];
  float* const bv0 = reinterpret_cast<float*>(dyn + G::KV_LDS);
  const int group = p.hq / p.hkv;
  const int nblk = (int)(p.rows / G::BR) + p.nseq;
  const Place pl = place(nblk, p.hkv, group);
  if (pl.block >= nblk) return;
  const Block bl = find_block<G::BR>(p.cu_seqlens, p.seq_lens, p.nseq, (int)p.rows, pl.block);
  if (!bl.any) return;
  const int h = pl.kvh * group + pl.g, len = bl.len;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 31, half = lane >> 5;
  Lds<T, G> L;
  L.init(lane);
  const int st = w / (4 / ST), sub = w % (4 / ST);
  const int q0 = bl.row0 + sub * 32;
  const int qi = q0 + m;
  const bool live = q0 < len;
  Dma<T, G> kd, vd;
  kd.init((const T*)p.k + (long long)bl.seq0 * p.k_row + pl.kvh * p.k_head, p.k_row, len, lane);
  vd.init((const T*)p.v + (long long)bl.seq0 * p.v_row + pl.kvh * p.v_head, p.v_row, len, lane);
  const int kend = CAUSAL ? min(len, bl.row0 + G::BR) : len;
  const int ntiles = (kend + KT - 1) / KT, nit = (ntiles + ST - 1) / ST;
  auto issue = [&](int it) {   // start bringing every stream's tile of iteration `it`
#pragma unroll
    for (int i = 0; i < ST; ++i) {
      char* const K = dyn + (i * 2 + (it & 1)) * G::BUF;
      kd.issue(K, (it * ST + i) * KT, w);
      vd.issue(K + G::TILE, (it * ST + i) * KT, w);
    }
  };
  issue(0);
  const int nd = 2 * p.bias_len - 1;
  const float* vec = BIAS ? p.bias_vec + (long long)h * nd : nullptr;
  const int bst = ST == 1 ? 0 : tid / G::SEG, bt = ST == 1 ? tid : tid % G::SEG;
  const int e0 = p.bias_len - 1 - bl.row0 - (G::BR - 1) + bst * KT + bt;
  float bnext = 0.f;
  // (kept finite: P = 0 where the bias is -inf, and 0 * -inf would reach dgate)
  if constexpr (BIAS) bv_store<G::SEG>(bv0 + bst * 8 * G::SEG, bt, fmaxf(bv_load(vec, nd, e0), -3e38f));
  u32x4 qf[G::NS], df[G::NS];
  const int qc = min(qi, len - 1);
  const long long row = bl.seq0 + qc;
  const char* qrow = (const char*)((const T*)p.q + row * p.q_row + h * p.q_head);
  const char* drow = (const char*)((const T*)p.dout + row * p.dout_row + h * p.dout_head);
  const char* orow = (const char*)((const T*)p.out + row * p.out_row + h * p.out_head);
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < G::NS; ++s) {
    const int at = (2 * s + half) * 16;
    qf[s] = *reinterpret_cast<const u32x4*>(qrow + at);
    df[s] = *reinterpret_cast<const u32x4*>(drow + at);
    u32x4 of = *reinterpret_cast<const u32x4*>(orow + at);
    if (qi >= len) qf[s] = df[s] = of = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (std::is_same_v<T, bf16_t>)
        delta += __uint_as_float(df[s][e] << 16) * __uint_as_float(of[e] << 16) +
                 __uint_as_float(df[s][e] & 0xffff0000u) * __uint_as_float(of[e] & 0xffff0000u);
      else
        delta += __uint_as_float(df[s][e]) * __uint_as_float(of[e]);
    }
  }
  delta = xor32_sum(delta);
  const float c1 = p.scale * LOG2E;
  float gl = LOG2E;
  if constexpr (BIAS) {
    if (p.gate) gl = p.gate[h * p.rows + row] * LOG2E;
  }
  float lse2 = p.lse[h * p.rows + row] * LOG2E;
  if (lse2 == -INF) lse2 = INF;  // nothing left in this row: P = 0
  const int u0 = 4 * half + G::BR - 1 - (sub * 32 + m);
  const float* const bcopy = bv0 + st * 8 * G::SEG + (u0 & 3) * G::SEG;
  const int uj = u0 - (u0 & 3), us = u0 & 3;
  float sum_pd = 0.f, sum_pb = 0.f, sum_pdb = 0.f;
  f32x16 dq[G::DT];
#pragma unroll
  for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[dt][r] = 0.f;

  auto tile = [&](const int it, auto masked_c) {
    constexpr bool MASKED = decltype(masked_c)::value;
    const int kb = (it * ST + st) * KT;
    char* const Kt = dyn + (st * 2 + (it & 1)) * G::BUF;
    char* const Vt = Kt + G::TILE;
    wait_all_and_meet();
    float4 bb[G::NT][4];
    if constexpr (BIAS) {
#pragma unroll
      for (int t = 0; t < G::NT; ++t)
#pragma unroll
        for (int a = 0; a < 4; ++a)
          bb[t][a] = *reinterpret_cast<const float4*>(bcopy + (it & 1) * 4 * G::SEG + bv_pos(uj + 32 * t + 8 * a, us));
    }
    if (it + 1 < nit) {
      issue(it + 1);
      if constexpr (BIAS) bnext = fmaxf(bv_load(vec, nd, e0 + (it + 1) * ST * KT), -3e38f);
    }
    if (live && (ST == 1 || kb < kend) && (!CAUSAL || kb <= q0 + 31)) {
      const int last = CAUSAL ? min(len - 1, qi) : len - 1;
#pragma unroll
      for (int t = 0; t < G::NT; ++t) {
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
        for (int c = 0; c < G::NS; ++c) {
          mma_row<T>(L.rd_row(Kt, t, c), qf[c], s);
          mma_row<T>(L.rd_row(Vt, t, c), df[c], dp);
        }
        float ds[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float b = 0.f;
          if constexpr (BIAS) {
            const float4 b4 = bb[t][r >> 2];
            b = (r & 3) == 0 ? b4.x : (r & 3) == 1 ? b4.y : (r & 3) == 2 ? b4.z : b4.w;
          }
          float e = fmaf(s[r], c1, BIAS ? fmaf(gl, b, -lse2) : -lse2);
          if constexpr (MASKED) e = kb + 32 * t + 8 * (r >> 2) + 4 * half + (r & 3) <= last ? e : -INF;
          const float pr = exp2_(e);
          const float pd = pr * dp[r];
          ds[r] = fmaf(-delta, pr, pd);
          if constexpr (EXACT) sum_pd += pd;
          if constexpr (BIAS) {
            sum_pb = fmaf(pr, b, sum_pb);
            sum_pdb = fmaf(pd, b, sum_pdb);
          }
        }
        mma_col_split<T, G>(L, Kt, 32 * t, ds, dq, lane);
      }
    }
    if constexpr (BIAS) {
      if (it + 1 < nit) bv_store<G::SEG>(bv0 + (bst * 2 + ((it + 1) & 1)) * 4 * G::SEG, bt, bnext);
    }
  };
  const int nfull = min(len, CAUSAL ? bl.row0 + 1 : len) / (KT * ST);
  for (int it = 0; it < nfull; ++it) tile(it, std::false_type{});
  for (int it = nfull; it < nit; ++it) tile(it, std::true_type{});

  if constexpr (ST > 1) {   // join: sums, in stream order
    float* const js = reinterpret_cast<float*>(dyn);
    constexpr int PER = (D / 2 + 3) * 64;
    float* const at = js + ((st - 1) * (4 / ST) + sub) * PER + lane;
    __syncthreads();
    if (st > 0) {
#pragma unroll
      for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) at[(dt * 16 + r) * 64] = dq[dt][r];
      if constexpr (EXACT) at[(D / 2) * 64] = sum_pd;
      if constexpr (BIAS) {
        at[(D / 2 + 1) * 64] = sum_pb;
        at[(D / 2 + 2) * 64] = sum_pdb;
      }
    }
    __syncthreads();
    if (st > 0) return;
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      const float* const x = js + (i * (4 / ST) + sub) * PER + lane;
#pragma unroll
      for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[dt][r] += x[(dt * 16 + r) * 64];
      if constexpr (EXACT) sum_pd += x[(D / 2) * 64];
      if constexpr (BIAS) {
        sum_pb += x[(D / 2 + 1) * 64];
        sum_pdb += x[(D / 2 + 2) * 64];
      }
    }
  }
  if constexpr (EXACT) delta = xor32_sum(sum_pd);
  if constexpr (BIAS) {
    sum_pb = xor32_sum(sum_pb);
    sum_pdb = xor32_sum(sum_pdb);
  }
  if (qi >= len) return;
  if (half == 0) {
    p.delta[h * p.rows + row] = delta;
    if constexpr (BIAS) {
      if (p.dgate) p.dgate[h * p.rows + row] = fmaf(-delta, sum_pb, sum_pdb);
    }
  }
  T* const out = (T*)p.dq + row * p.dq_row + h * p.dq_head + 4 * half;
#pragma unroll
  for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      store4<T>(out + 32 * dt + 8 * a, dq[dt][4 * a] * p.scale, dq[dt][4 * a + 1] * p.scale, dq[dt][4 * a + 2] * p.scale,
                dq[dt][4 * a + 3] * p.scale);
}

// ---------------------------------------------------------------------------------- backward: dK, dV, dbias
// One workgroup = 128 keys; the queries of every head of the group stream past (their Q and dO tiles by
// LDS-DMA, lse, delta and gate beside them), so shared heads' gradients are sums in registers, in one
// order. S = Q K^T here: a lane is a key, its registers 16 queries.
//
// dbias: g dS summed along j - i. Register (a, c) of lane (x = lane & 15, kr = (lane >> 4) & 1, half) is
// query 8 a + 4 half + c and key 16 kr + x: shifted by R = 8 (a & 1) + c lanes inside its row of 16, it
// joins diagonal 16 kr + x - 4 half - 16 (a >> 1), or, where the shift ran out of the row, the one 16
// further down. 2 NT + 1 accumulators so hold a tile; all but the last are done with it and go, as 16
// strips (4 waves x 4 lane rows) of 32 NT, to LDS, where the next iteration adds what falls on a diagonal,
// a thread each, in one order, into a ring; what the workgroup will not meet again leaves the ring for
// this block's row of a slab in memory. rows of the slab are added by dbias_kernel: no atomics.
//
// Bound by latency at two waves per SIMD, and by the causal blocks' unequal lengths: the forward's batches take 89-94 us
// (4096 causal rows; matrix units 29 % busy, waves waiting 47 %) + 14 us dkv_kernel, 69-73 us (utterances, with both the
// bias and its gradient), 45 + 7 us (f32); long full sequences 676 TF for the whole backward at head_dim 128, 646 at 64.
constexpr int RING = 256;   // more than the diagonals of an iteration
template <int R>
NRSE_DEV void diag_add(float v, float& lo, float& hi) {
  if constexpr (R == 0) {
    lo += v;
  } else {
    lo += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x100 + R, 0xF, 0xF, true));
    hi += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x110 + 16 - R, 0xF, 0xF, true));
  }
}
__host__ __device__ inline long long slab_row(int bias_len) { return ((bias_len + 63) & ~63) + 192; }

template <typename T, int D>
struct KvGeo : Geo<T, D, (D * (int)sizeof(T) > 128 ? 32 : 64)> {
  // bf16 at head_dim 128: the accumulators and K fill a wave's 256 registers, V's fragments stay in LDS. With a bias
  // even so 42 registers of the compiler's report are spilled, and some of their reloads stand in the loop.
  static constexpr bool VLDS = sizeof(T) == 2 && D == 128;
  static constexpr int WAVES = sizeof(T) == 4 && D == 128 ? 1 : 2;   // per SIMD
  // Streams: where a workgroup's registers and LDS leave a SIMD two waves either way (256-byte rows), 8
  // waves in two streams of query tiles share the keys instead of two workgroups, and end in half the time
  static constexpr int ST = D * (int)sizeof(T) == 256 ? 2 : 1;
  using B = Geo<T, D, (D * (int)sizeof(T) > 128 ? 32 : 64)>;
  static constexpr int W = ST * B::KT;                               // queries of an iteration
  static constexpr int BUF = 2 * B::TILE;                            // Q and dO tile
  static constexpr int SLOTS = 16 * (2 * B::NT + 1);                 // of a diagonal strip
  static constexpr int NDIAG = 132 + 32 * B::NT + B::KT * (ST - 1);  // diagonals of an iteration: 127 down
  static_assert(NDIAG <= RING, "the ring holds an iteration's diagonals");
  // LDS: tiles [ST][2 buffers], V [4], rows [ST][2][3][KT], bias [ST][2][4][SEG], strips [2][ST][16][SLOTS], ring
  static constexpr int V_AT = ST * 2 * BUF, ROWS_AT = V_AT + (VLDS ? 4 * B::TILE : 0),
                       BIAS_AT = ROWS_AT + ST * 6 * B::KT * 4, STRIPS_AT = BIAS_AT + ST * 8 * B::SEG * 4,
                       RING_AT = STRIPS_AT + 2 * ST * 16 * SLOTS * 4, END = RING_AT + RING * 4;
  static constexpr int JOIN = ST > 1 ? 2 * 4 * (D / 2) * 64 * 4 : 0;  // the streams' dK and dV, at the end
};

template <typename T, int D, bool BIAS, bool CAUSAL>
__global__ __launch_bounds__((256 * KvGeo<T, D>::ST)) __attribute__((amdgpu_waves_per_eu(KvGeo<T, D>::WAVES, KvGeo<T, D>::WAVES))) void bwd_kv_kernel(const nrse_attn_packed_bwd_params p, int slices,
                                                                         float* __restrict__ sums) {
  using G = KvGeo<T, D>;
  constexpr int KT = G::KT, NT = G::NT, ST = G::ST, W = G::W;
  extern __shared__ __attribute__((aligned(16))) char dyn[];
  char* const vt0 = dyn + G::V_AT;
  float* const rows0 = reinterpret_cast<float*>(dyn + G::ROWS_AT);
  float* const bv0 = reinterpret_cast<float*>(dyn + G::BIAS_AT);
  float* const strip0 = reinterpret_cast<float*>(dyn + G::STRIPS_AT);
  float* const ring = reinterpret_cast<float*>(dyn + G::RING_AT);
  const int group = p.hq / p.hkv;
  const int nblk = (int)(p.rows / BQ) + p.nseq;
  const Place pl = place(nblk, p.hkv, slices);
  if (pl.block >= nblk) return;
  // a causal block's queries start at its own rows: the first block of a sequence has the most
  Block bl = find_block<BQ>(p.cu_seqlens, p.seq_lens, p.nseq, (int)p.rows, pl.block);
  const int tid = threadIdx.x, lane = tid & 63;
  const bool dbias = BIAS && p.dbias_vec;
  // with a bias a slice is whole heads, or one of `parts` runs of one head's queries: each has its own row of
  // the slab
  const int parts = BIAS && slices > group ? slices / group : 1, piece = BIAS ? pl.g % parts : 0;
  const bool lists = dbias && tid == 0 && pl.kvh == 0 && pl.g < parts;
  int* const meta = dbias ? (int*)p.part + (pl.block * parts + piece) * 4 : nullptr;
  if (!bl.any) {
    if (lists) meta[1] = meta[2] = 0;
    return;
  }
  const int len = bl.len;
  if (CAUSAL) bl.row0 = (len - 1) / BQ * BQ - bl.row0;
  const int st = __builtin_amdgcn_readfirstlane(tid >> 8), w = __builtin_amdgcn_readfirstlane((tid >> 6) & 3);
  const int t8 = tid & 255;
  const int m = lane & 31, half = lane >> 5;
  Lds<T, G> L;
  L.init(lane);
  const int kb0 = bl.row0, k0 = kb0 + w * 32, kj = k0 + m;
  const bool live = k0 < len;
  const int qt0 = CAUSAL ? kb0 / W : 0, qtn = (len + W - 1) / W, nq = qtn - qt0;
  Dma<T, G> qd, od;
  qd.init((const T*)p.q + (long long)bl.seq0 * p.q_row, p.q_row, len, lane);
  od.init((const T*)p.dout + (long long)bl.seq0 * p.dout_row, p.dout_row, len, lane);
  const int h0 = pl.kvh * group;
  const int nd = 2 * p.bias_len - 1;
  float nrow[3] = {INF, 0.f, 1.f}, nbias = 0.f;
  auto fetch = [&](int h, int qt, int buf) {   // start bringing this stream's tile of (h, qt) into buffer buf
    char* const Q = dyn + (st * 2 + buf) * G::BUF;
    const int qb = qt * W + st * KT;
    qd.issue(Q, qb, w, h * p.q_head * (long long)sizeof(T));
    od.issue(Q + G::TILE, qb, w, h * p.dout_head * (long long)sizeof(T));
    if (t8 < KT) {
      const int qi = qb + t8;
      const long long at = h * p.rows + bl.seq0 + min(qi, len - 1);
      const float l = p.lse[at], d = p.delta[at];
      float g = 1.f;
      if constexpr (BIAS) {
        if (p.gate) g = p.gate[at];
      }
      // rows past the end and rows that were left nothing: P = 0
      nrow[0] = (qi < len && l != -INF) ? l * LOG2E : INF;
      nrow[1] = qi < len ? d : 0.f;
      nrow[2] = qi < len ? g : 1.f;
    }
    // segment entry u of the tile: b[kb0 - qb + 127 - u], u = query - key + 127
    if constexpr (BIAS)
      nbias = bv_load(p.bias_vec + (long long)h * nd, nd, kb0 - qb + 127 - t8 + p.bias_len - 1);
  };
  auto keep = [&](int buf) {   // what came by registers
    if (t8 < KT) {
      float* r = rows0 + (st * 2 + buf) * 3 * KT + t8;
      r[0] = nrow[0];
      r[KT] = nrow[1];
      r[2 * KT] = nrow[2];
    }
    if constexpr (BIAS) bv_store<G::SEG>(bv0 + (st * 2 + buf) * 4 * G::SEG, t8, nbias * LOG2E);
  };
  // this slice's share of the group's (head, query tile) pairs
  const int total = group * nq;
  int it0 = (int)((long long)total * pl.g / slices), it1 = (int)((long long)total * (pl.g + 1) / slices);
  int qlo = qt0, qhi = qtn;
  if (BIAS && parts > 1) {
    qlo = qt0 + (int)((long long)nq * piece / parts);
    qhi = qt0 + (int)((long long)nq * (piece + 1) / parts);
    it0 = pl.g / parts * nq + qlo - qt0;
    it1 = it0 + qhi - qlo;
  }
  int g = it0 / nq, qt = qt0 + it0 % nq;
  if (it0 < it1) fetch(h0 + g, qt, it0 & 1);
  Dma<T, G> vd;
  if constexpr (G::VLDS) {
    vd.init((const T*)p.v + (long long)bl.seq0 * p.v_row + pl.kvh * p.v_head, p.v_row, len, lane);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i % ST == st) vd.issue(vt0 + i * G::TILE, kb0 + 32 * i, w);
  }
  const char* const vt = vt0 + w * G::TILE;
  u32x4 kf[G::NS], vf[G::VLDS ? 1 : G::NS];
  const long long krow = bl.seq0 + min(kj, len - 1);
  const char* kp = (const char*)((const T*)p.k + krow * p.k_row + pl.kvh * p.k_head);
  const char* vp = (const char*)((const T*)p.v + krow * p.v_row + pl.kvh * p.v_head);
#pragma unroll
  for (int s = 0; s < G::NS; ++s) {
    kf[s] = *reinterpret_cast<const u32x4*>(kp + (2 * s + half) * 16);
    if (kj >= len) kf[s] = u32x4{0, 0, 0, 0};
    if constexpr (!G::VLDS) {
      vf[s] = *reinterpret_cast<const u32x4*>(vp + (2 * s + half) * 16);
      if (kj >= len) vf[s] = u32x4{0, 0, 0, 0};
    }
  }
  keep(it0 & 1);
  const float c1 = p.scale * LOG2E;
  const int u0 = 4 * half + 127 - (w * 32 + m);
  const float* const bcopy = bv0 + st * 8 * G::SEG + (u0 & 3) * G::SEG;
  const int uj = u0 - (u0 & 3), us = u0 & 3;
  f32x16 dk[G::DT], dv[G::DT];
#pragma unroll
  for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[dt][r] = dv[dt][r] = 0.f;
  float dacc[2 * NT + 1];
#pragma unroll
  for (int j = 0; j <= 2 * NT; ++j) dacc[j] = 0.f;
  if (lists) {   // the slab row's entries: diagonal kb0 + 127 - x, x from the first query on
    meta[0] = kb0;
    meta[1] = qlo * W;
    meta[2] = qlo < qhi ? min(len + 127, (qhi - 1) * W + G::NDIAG) : 0;
  }
  constexpr int STRIP = 16 * G::SLOTS;   // floats of a stream's strips
  float* const mine = strip0 + st * STRIP + ((w * 2 + ((lane >> 4) & 1)) * 2 + half) * G::SLOTS + (lane & 15) + 32 * NT;
  if (dbias && tid < RING) ring[tid] = 0.f;

  // the strips of one iteration into the ring; diagonal R is key - query relative to (kb0, qb). Strip
  // (b = 2 w + kr, half) of stream i holds diagonals 16 b - 4 half + slot - 32 NT - KT i, so R meets 2 NT + 1
  // strips of each half and stream
  float* const slab =
      dbias ? p.part + 4LL * nblk * parts + ((long long)pl.block * parts + piece) * slab_row(p.bias_len) : nullptr;
  const long long slab_head = (long long)nblk * parts * slab_row(p.bias_len);
  const int xend = min((int)slab_row(p.bias_len), len + 127);
  auto fold = [&](int buf, int qb, int h, bool end) {
    const int R = tid + 128 - G::NDIAG;
    if (tid < G::NDIAG) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < ST; ++i)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int x = R + 4 * hf + 32 * NT + KT * i;
#pragma unroll
          for (int db = 0; db <= 2 * NT; ++db) {
            const int b = (x >> 4) - db;
            const bool in = (unsigned)b < 8u;
            const float y = strip0[(buf * ST + i) * STRIP + ((in ? b : 0) * 2 + hf) * G::SLOTS + (x & 15) + 16 * db];
            s += in ? y : 0.f;
          }
        }
      float* const slot = ring + ((kb0 - qb + R) & (RING - 1));
      s += *slot;
      const bool done = end || R > 127 - W;
      *slot = done ? 0.f : s;
      const int x = qb + 127 - R;
      if (done && x < xend) slab[h * slab_head + x] = s;
    }
  };
  auto shed = [&](int buf) {   // the accumulators, to the strips
#pragma unroll
    for (int j = 0; j <= 2 * NT; ++j) {
      mine[buf * ST * STRIP - 16 * j] = dacc[j];
      dacc[j] = 0.f;
    }
  };

  const bool part_block = kb0 + BQ > len;
  for (int it = it0; it < it1; ++it) {
    // (one body and a branch around the masking alone: two bodies in the loop made the compiler copy
    // the accumulators between them)
    const int buf = it & 1, qb = qt * W + st * KT;
    const bool masked = part_block || (CAUSAL && qb < kb0 + BQ - 1);
    char* const Qt = dyn + (st * 2 + buf) * G::BUF;
    char* const Ot = Qt + G::TILE;
    const float* const rb = rows0 + (st * 2 + buf) * 3 * KT + 4 * half;
    wait_all_and_meet();
    if (it + 1 < it1) {
      const bool next_head = qt + 1 == qtn;
      fetch(h0 + g + next_head, next_head ? qt0 : qt + 1, buf ^ 1);
    }
    if (dbias && qt > qt0 && it > it0) fold(buf ^ 1, (qt - 1) * W, h0 + g, false);
    if (live && (ST == 1 || qb < len) && (!CAUSAL || qb + KT - 1 >= k0)) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < G::NS; ++c) {
          mma_row<T>(L.rd_row(Qt, t, c), kf[c], s);
          mma_row<T>(L.rd_row(Ot, t, c), G::VLDS ? L.rd_row(vt, 0, c) : vf[G::VLDS ? 0 : c], dp);
        }
        {
          constexpr int RD = G::VLDS ? 3 : 2, MM = sizeof(T) == 2 ? 2 : 8;
          __builtin_amdgcn_sched_group_barrier(0x100, RD, 0);
#pragma unroll
          for (int c = 0; c + 1 < G::NS; ++c) {
            __builtin_amdgcn_sched_group_barrier(0x100, RD, 0);
            __builtin_amdgcn_sched_group_barrier(0x8, MM, 0);
          }
          __builtin_amdgcn_sched_group_barrier(0x8, MM, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        float pr[16];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const float4 l4 = *reinterpret_cast<const float4*>(rb + 32 * t + 8 * a);
          const float l[4] = {l4.x, l4.y, l4.z, l4.w};
          if constexpr (BIAS) {
            const float4 g4 = *reinterpret_cast<const float4*>(rb + 2 * KT + 32 * t + 8 * a);
            const float4 b4 = *reinterpret_cast<const float4*>(bcopy + buf * 4 * G::SEG + bv_pos(uj + 32 * t + 8 * a, us));
            pr[4 * a] = fmaf(s[4 * a], c1, fmaf(g4.x, b4.x, -l[0]));
            pr[4 * a + 1] = fmaf(s[4 * a + 1], c1, fmaf(g4.y, b4.y, -l[1]));
            pr[4 * a + 2] = fmaf(s[4 * a + 2], c1, fmaf(g4.z, b4.z, -l[2]));
            pr[4 * a + 3] = fmaf(s[4 * a + 3], c1, fmaf(g4.w, b4.w, -l[3]));
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) pr[4 * a + c] = fmaf(s[4 * a + c], c1, -l[c]);
          }
        }
        if (masked) {
          asm volatile("");
          const int first = CAUSAL ? (kj < len ? kj : 1 << 30) : (kj < len ? 0 : 1 << 30);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            pr[r] = qb + 32 * t + 8 * (r >> 2) + 4 * half + (r & 3) >= first ? pr[r] : -INF;
        }
        float ds[16];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const float4 d4 = *reinterpret_cast<const float4*>(rb + KT + 32 * t + 8 * a);
          const float d[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            pr[4 * a + c] = exp2_(pr[4 * a + c]);
            ds[4 * a + c] = pr[4 * a + c] * (dp[4 * a + c] - d[c]);
          }
          if constexpr (BIAS) {
            // (a, c): shift 8 (a & 1) + c, accumulator 2 t + (a >> 1)
            const float4 gg = *reinterpret_cast<const float4*>(rb + 2 * KT + 32 * t + 8 * a);
            float& lo = dacc[2 * t + (a >> 1)];
            float& hi = dacc[2 * t + (a >> 1) + 1];
            if (a & 1) {
              diag_add<8>(gg.x * ds[4 * a], lo, hi);
              diag_add<9>(gg.y * ds[4 * a + 1], lo, hi);
              diag_add<10>(gg.z * ds[4 * a + 2], lo, hi);
              diag_add<11>(gg.w * ds[4 * a + 3], lo, hi);
            } else {
              diag_add<0>(gg.x * ds[4 * a], lo, hi);
              diag_add<1>(gg.y * ds[4 * a + 1], lo, hi);
              diag_add<2>(gg.z * ds[4 * a + 2], lo, hi);
              diag_add<3>(gg.w * ds[4 * a + 3], lo, hi);
            }
            // (here, not sunk to where they are stored: the shifted values would all live until then, and the
            // shifts would not fold into the additions)
            asm volatile("" : "+v"(lo), "+v"(hi));
          }
        }
        mma_col<T, G>(L, Ot, 32 * t, pr, dv, lane);
        mma_col<T, G>(L, Qt, 32 * t, ds, dk, lane);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (dbias) shed(buf);
    if (it + 1 < it1) keep(buf ^ 1);
    if (dbias && (qt + 1 == qtn || it + 1 == it1)) {
      // the head's last tile (of this slice): fold it too, and empty the ring
      __syncthreads();
      fold(buf, qt * W, h0 + g, true);
    }
    if (++qt == qtn) {
      qt = qt0;
      ++g;
    }
  }
  if constexpr (ST > 1) {
    // join: stream 0 leaves with dK, stream 1 with dV, each the sum in stream order. (A slice without a pair comes
    // here with its V copies still on their way, and the join's places lie over V's: they are waited for.)
    wait_all_and_meet();
    float* const put = reinterpret_cast<float*>(dyn) + ((st == 0 ? 4 : 0) + w) * (D / 2) * 64 + lane;
    const float* const get = reinterpret_cast<const float*>(dyn) + ((st == 0 ? 0 : 4) + w) * (D / 2) * 64 + lane;
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) put[(dt * 16 + r) * 64] = st == 0 ? dv[dt][r] : dk[dt][r];
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (st == 0) dk[dt][r] += get[(dt * 16 + r) * 64];
        else dv[dt][r] = get[(dt * 16 + r) * 64] + dv[dt][r];
      }
  }
  const bool out_k = ST == 1 || st == 0, out_v = ST == 1 || st == 1;
  if (kj >= len) return;
  if (sums) {   // this slice's f32 sums; dkv_kernel adds the slices in order
    const long long n = p.rows * p.hkv * D;
    float* const a = sums + pl.g * 2 * n + (krow * p.hkv + pl.kvh) * D + 4 * half;
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (out_k) store4<float>(a + 32 * dt + 8 * i, dk[dt][4 * i], dk[dt][4 * i + 1], dk[dt][4 * i + 2], dk[dt][4 * i + 3]);
        if (out_v) store4<float>(a + n + 32 * dt + 8 * i, dv[dt][4 * i], dv[dt][4 * i + 1], dv[dt][4 * i + 2], dv[dt][4 * i + 3]);
      }
    return;
  }
  T* const dko = (T*)p.dk + krow * p.dk_row + pl.kvh * p.dk_head + 4 * half;
  T* const dvo = (T*)p.dv + krow * p.dv_row + pl.kvh * p.dv_head + 4 * half;
#pragma unroll
  for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      if (out_k)
        store4<T>(dko + 32 * dt + 8 * a, dk[dt][4 * a] * p.scale, dk[dt][4 * a + 1] * p.scale,
                  dk[dt][4 * a + 2] * p.scale, dk[dt][4 * a + 3] * p.scale);
      if (out_v) store4<T>(dvo + 32 * dt + 8 * a, dv[dt][4 * a], dv[dt][4 * a + 1], dv[dt][4 * a + 2], dv[dt][4 * a + 3]);
    }
}

// dk, dv = the slices' f32 sums, added in order: one workgroup per 32 rows and key head, loads of four
// slices at once. Bound by the sums' own bytes: 4 slices of 4096 rows x 4 heads of 128, 67 MB in and 8 MB out, 13.7 us = 5.5 TB/s
// (27 one load at a time).
template <typename T, int D>
__global__ __launch_bounds__(256) void dkv_kernel(const nrse_attn_packed_bwd_params p, int slices,
                                                  const float* __restrict__ sums) {
  constexpr int BR = 32;
  const int nblk = (int)(p.rows / BR) + p.nseq;
  const Place pl = place(nblk, p.hkv, 1);
  if (pl.block >= nblk) return;
  const Block bl = find_block<BR>(p.cu_seqlens, p.seq_lens, p.nseq, (int)p.rows, pl.block);
  if (!bl.any) return;
  const int n4 = min(BR, bl.len - bl.row0) * (D / 4);
  const long long n = p.rows * p.hkv * D;
  for (int i = threadIdx.x; i < 2 * n4; i += 256) {
    const bool second = i >= n4;
    const int j = second ? i - n4 : i;
    const long long row = bl.seq0 + bl.row0 + j / (D / 4);
    const int d = j % (D / 4) * 4;
    const float* a = sums + (second ? n : 0) + (row * p.hkv + pl.kvh) * D + d;
    f32x4 x{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < slices; s += 4) {
      f32x4 y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = *reinterpret_cast<const f32x4*>(a + min(s + k, slices - 1) * 2 * n);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (s + k < slices) x += y[k];
    }
    if (second) store4<T>((T*)p.dv + row * p.dv_row + pl.kvh * p.dv_head + d, x[0], x[1], x[2], x[3]);
    else store4<T>((T*)p.dk + row * p.dk_row + pl.kvh * p.dk_head + d, x[0] * p.scale, x[1] * p.scale, x[2] * p.scale, x[3] * p.scale);
  }
}

// dbias[h, d] (+)= the slab's rows: for each diagonal, the blocks that hold it, in block order within 4
// quarters of the blocks, then the quarters in order. A row's place is uniform, its entry a lane's: eight
// rows' loads at once, from a clamped entry where a row does not hold the diagonal. Bound by those loads' latency:
// 4.8 us for 62 rows of 16 heads (12.5 one row at a time).
__global__ __launch_bounds__(256) void dbias_kernel(const float* __restrict__ part, float* __restrict__ dvec, int nblk,
                                                    int bias_len, int accumulate) {
  __shared__ float red[4][64];
  const int nd = 2 * bias_len - 1, h = blockIdx.y;
  const int e = blockIdx.x * 64 + (threadIdx.x & 63), wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int d = e - (bias_len - 1);
  const int4* meta = (const int4*)part;
  const long long ld = slab_row(bias_len);
  const float* slab = part + 4LL * nblk + (long long)h * nblk * ld;
  const int per = (nblk + 3) / 4, b0 = wv * per, b1 = min(nblk, b0 + per);
  float s = 0.f;
  for (int b = b0; b < b1; b += 8) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = min(b + k, nblk - 1);
      const int4 m = meta[r];
      const int x = m.x + 127 - d;
      const bool in = b + k < b1 && x >= m.y && x < m.z && x < ld;
      const float y = slab[(long long)r * ld + (in ? x : 0)];
      v[k] = in ? y : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) s += v[k];
  }
  red[wv][threadIdx.x & 63] = s;
  __syncthreads();
  if (wv == 0 && e < nd) {
    const int i = threadIdx.x;
    const float v = red[0][i] + red[1][i] + red[2][i] + red[3][i];
    float* o = dvec + (long long)h * nd + e;
    *o = accumulate ? *o + v : v;
  }
}

// ---------------------------------------------------------------------------------- bias tables
// bucket of a relative position: the last of `edges` (ascending, edges[0] = 0) that is <= its distance;
// two-sided (causal = 0): the keys behind the query take the first n buckets, those ahead the next n;
// causal: all n are the past's, and a key ahead counts as distance 0.
NRSE_DEV int bucket_of(const int* edges, int n, int rel, int causal) {
  const int dist = causal ? max(-rel, 0) : abs(rel);
  int lo = 0, hi = n;  // edges[lo] <= dist < edges[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (edges[mid] <= dist) lo = mid;
    else hi = mid;
  }
  return lo + (!causal && rel > 0 ? n : 0);
}

// (edges in LDS where they fit: a binary search through memory is 8 dependent loads; 1197 entries of 16 heads
// 3 to 5 us, the launch and two round trips to memory)
constexpr int EDGES = 2048;
__global__ __launch_bounds__(256) void rel_expand_kernel(const float* __restrict__ E, const int* __restrict__ edges, int n,
                                                         float* __restrict__ vec, int H, int T, int causal) {
  __shared__ int near[EDGES];
  const int* at = edges;
  if (n <= EDGES) {
    for (int i = threadIdx.x; i < n; i += 256) near[i] = edges[i];
    __syncthreads();
    at = near;
  }
  const int nd = 2 * T - 1;
  for (int e = blockIdx.x * 256 + threadIdx.x; e < nd; e += gridDim.x * 256) {
    const float* row = E + (long long)bucket_of(at, n, e - (T - 1), causal) * H;
    for (int h = blockIdx.y; h < H; h += gridDim.y) vec[(long long)h * nd + e] = row[h];
  }
}

// dE[bucket, h] (+)= the sum of dvec[h, d] over the bucket's distances: they are one run of d (two for
// distance 0's bucket of a causal table: the keys ahead count as distance 0). One workgroup per bucket and head: lanes'
// sums in distance order, then a fixed tree. The widest buckets, a whole length, set the time: 4 loads at
// once (2500 distances, 8 heads: 13 us one at a time, 4.7 four).
__global__ __launch_bounds__(256) void rel_collect_kernel(const float* __restrict__ dvec, const int* __restrict__ edges,
                                                          int n, float* __restrict__ dE, int H, int T, int causal,
                                                          int accumulate) {
  __shared__ float red[4];
  const int b = blockIdx.x / H, h = blockIdx.x % H, k = b % n;
  const bool ahead = b >= n;
  // distances [edges[k], edges[k + 1]), the first bucket's from 0 (as expand's search has it), at most T - 1; none at
  // distance 0 ahead of the query. Both ends are clamped before anything is added to them: a border may be any
  // int, 2^31 - 1 among them (a bucket past every length), and then the run is empty.
  const int d0 = k == 0 ? (ahead ? 1 : 0) : min(max(edges[k], ahead ? 1 : 0), T), d1 = min(k + 1 < n ? edges[k + 1] : T, T);
  const int nd = 2 * T - 1;
  const float* row = dvec + (long long)h * nd + (T - 1);  // row[j - i]
  float s = 0.f;
  auto run = [&](int from, int to, int sign) {
    for (int d = from + (int)threadIdx.x; d < to; d += 1024) {
      float v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = row[sign * min(d + 256 * u, T - 1)];
#pragma unroll
      for (int u = 0; u < 4; ++u) s += d + 256 * u < to ? v[u] : 0.f;
    }
  };
  run(d0, d1, ahead ? 1 : -1);
  if (causal && d0 == 0 && d1 > 0) run(1, T, 1);   // the bucket that holds distance 0
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    const float v = red[0] + red[1] + red[2] + red[3];
    float* o = dE + (long long)b * H + h;
    *o = accumulate ? *o + v : v;
  }
}

// ---------------------------------------------------------------------------------- launches
// Streams of the forward and dQ kernels: one where 128-row workgroups fill the chip (256 CUs take 512 at
// once), two where they do not: under a causal mask, where half of them are short, it takes more. Measured,
// forward / backward us in one stream and in two, 16 heads. One long sequence, full: 288 workgroups at head_dim 64
// 43 / 147 and 41 / 141, 416 60 / 223 and 68 / 234, 416 at 128 96 / 423 and 112 / 436; causal: 672 at 128 150 / 498 and
// 138 / 473, 720 at 64 100 / 330 and 95 / 328, 864 at 128 213 / 730 and 217 / 743. Five unequal ones, causal: 672 at 128
// 62 / 191 and 54 / 178. Many short ones of one length are better off in one stream at any of these numbers (16 causal ones
// of 208 rows, 672 at 128: 17 / 62 and 22 / 71), which the number of workgroups does not tell.
int q_streams(long long rows, int nseq, int hq, int causal) {
  const long long n = (rows / BQ + nseq) * hq;
  return n >= (causal ? 700 : 400) ? 1 : 2;
}

template <typename T, int D>
size_t lds_kv(bool bias) {
  using G = KvGeo<T, D>;
  return std::max(bias ? G::END : G::BIAS_AT, G::JOIN);
}

// Slices of a key block's (head, query tile) pairs: with fewer than 512 workgroups the longest of them, a
// causal sequence's first block, decides the time, and a batch with fewer blocks x key heads is split up
// to 8 ways, each slice writing f32 sums that dkv_kernel adds. Not below 4 pairs a slice (of an average
// sequence; 1 in f32, whose pairs take 8 times as long). Measured: causal f32 batch of 104 groups,
// backward 144 us in 1 slice, 110 in 2, 94 in 4; causal bf16 of 152 groups 197 us in 2, 164 in 3, 155 in 4, 163 in 5,
// 176 in 7 (the sums' traffic); 944 groups 94 us in 1, 162 in 2.
int kv_slices(const nrse_attn_packed_bwd_params& p) {
  const long long groups = (p.rows / BQ + p.nseq) * p.hkv, G = p.hq / p.hkv;
  const bool f32 = p.dtype == NRSE_F32;
  const long long pair = f32 && p.head_dim == 128 ? 32 : 64;   // queries of an iteration
  long long n = (512 + groups - 1) / groups;
  n = std::min(n, std::min(8LL, std::max(1LL, G * (p.rows / p.nseq) / pair / (f32 ? 1 : 4))));
  if (p.bias_vec && n > G) n -= n % G;   // whole heads, or equal parts of each
  if (p.bias_vec && n <= G)
    while (G % n) --n;
  return (int)n;
}
int kv_parts(const nrse_attn_packed_bwd_params& p) { return std::max(1, kv_slices(p) / (p.hq / p.hkv)); }

template <typename F>
void with_streams(int st, F f) {
  if (st == 1) f(std::integral_constant<int, 1>{});
  else f(std::integral_constant<int, 2>{});
}

template <typename T, int D, bool BIAS, bool CAUSAL>
void launch_fwd(const nrse_attn_packed_fwd_params& p, hipStream_t st) {
  with_streams(q_streams(p.rows, p.nseq, p.hq, p.causal), [&](auto s) {
    constexpr int ST = decltype(s)::value;
    const long long n = grid_size(p.rows / (BQ / ST) + p.nseq, p.hkv, p.hq / p.hkv);
    hipLaunchKernelGGL((fwd_kernel<T, D, BIAS, CAUSAL, ST>), dim3((unsigned)n), dim3(256), (lds_q_fwd<QGeo<T, D, ST>>(BIAS)), st, p);
  });
}

// the workspace: the bias gradient's table of blocks and slab, then the slices' sums
long long slab_floats(const nrse_attn_packed_bwd_params& p) {
  const long long nblk = (p.rows / BQ + p.nseq) * kv_parts(p);
  return p.bias_vec && p.dbias_vec ? nblk * 4 + p.hq * nblk * slab_row(p.bias_len) : 0;
}

template <typename T, int D, bool BIAS, bool CAUSAL>
void launch_bwd(const nrse_attn_packed_bwd_params& p, hipStream_t st) {
  const long long nblk = p.rows / BQ + p.nseq;
  with_streams(q_streams(p.rows, p.nseq, p.hq, p.causal), [&](auto s) {
    constexpr int ST = decltype(s)::value;
    const long long n = grid_size(p.rows / (BQ / ST) + p.nseq, p.hkv, p.hq / p.hkv);
    hipLaunchKernelGGL((bwd_q_kernel<T, D, BIAS, CAUSAL, ST>), dim3((unsigned)n), dim3(256), (lds_q<QGeo<T, D, ST>>(BIAS)), st, p);
  });
  const int ns = kv_slices(p);
  float* const sums = ns > 1 ? p.part + slab_floats(p) : nullptr;
  hipLaunchKernelGGL((bwd_kv_kernel<T, D, BIAS, CAUSAL>), dim3((unsigned)grid_size(nblk, p.hkv, ns)),
                     dim3(256 * KvGeo<T, D>::ST), (lds_kv<T, D>(BIAS)), st, p, ns, sums);
  if (ns > 1)
    hipLaunchKernelGGL((dkv_kernel<T, D>), dim3((unsigned)grid_size(p.rows / 32 + p.nseq, p.hkv, 1)), dim3(256), 0, st, p, ns,
                       sums);
}

template <typename P, typename F>
void dispatch(const P& p, F f) {
  const bool b = p.bias_vec, c = p.causal;
  auto with_mask = [&](auto t, auto d, auto bias) {
    if (c) f(t, d, bias, std::true_type{});
    else f(t, d, bias, std::false_type{});
  };
  auto with_bias = [&](auto t, auto d) {
    if (b) with_mask(t, d, std::true_type{});
    else with_mask(t, d, std::false_type{});
  };
  using d64 = std::integral_constant<int, 64>;
  using d128 = std::integral_constant<int, 128>;
  if (p.dtype == NRSE_BF16) p.head_dim == 64 ? with_bias(bf16_t{}, d64{}) : with_bias(bf16_t{}, d128{});
  else p.head_dim == 64 ? with_bias(float{}, d64{}) : with_bias(float{}, d128{});
}

// one operand: 16-byte rows, and no row so far on that 64 of them pass 32 bits of offset; of one that is
// written (`rows` of them), no two elements at one address
int check_rows(const char* fn, const char* name, const void* ptr, long long row, long long head, const int dtype, int D,
               int heads, long long rows = 0) {
  const int es = dtype == NRSE_BF16 ? 2 : 4;
  NRSE_REQUIRE(ptr, "%s: %s is null", fn, name);
  NRSE_REQUIRE(((uintptr_t)ptr & 15) == 0 && (row * es) % 16 == 0 && (head * es) % 16 == 0,
               "%s: %s: base and strides (%lld rows, %lld heads) must be 16-byte multiples", fn, name, row, head);
  NRSE_REQUIRE(row >= D && row * es <= (1 << 24), "%s: %s: row stride %lld outside [head_dim, 2^24 bytes]", fn, name, row);
  NRSE_REQUIRE(heads == 1 || head >= D, "%s: %s: head stride %lld below head_dim", fn, name, head);
  NRSE_REQUIRE(rows <= 1 || heads == 1 || row >= (heads - 1) * head + D || head >= (rows - 1) * row + D,
               "%s: %s is written: its rows and heads (strides %lld, %lld) overlap", fn, name, row, head);
  return NRSE_OK;
}

template <typename P>
int check_common(const char* fn, const P* p) {
  NRSE_REQUIRE(p->dtype == NRSE_BF16 || p->dtype == NRSE_F32, "%s: dtype %d (bf16 and f32 only)", fn, p->dtype);
  NRSE_REQUIRE(p->head_dim == 64 || p->head_dim == 128, "%s: head_dim %d (64 and 128 only)", fn, p->head_dim);
  NRSE_REQUIRE(p->hkv > 0 && p->hq > 0 && p->hq % p->hkv == 0, "%s: %d query heads over %d key heads", fn, p->hq, p->hkv);
  NRSE_REQUIRE(p->rows >= 0 && p->rows < (1LL << 31) - 256 && p->nseq >= 0, "%s: rows %lld, sequences %d", fn, p->rows,
               p->nseq);
  NRSE_REQUIRE(p->nseq == 0 || p->cu_seqlens, "%s: cu_seqlens is null", fn);
  NRSE_REQUIRE(!p->bias_vec || (p->bias_len > 0 && p->bias_len < (1 << 29)), "%s: bias_len %d", fn, p->bias_len);
  NRSE_REQUIRE(p->bias_vec || !p->gate, "%s: a gate needs a bias", fn);
  // a grid has fewer than 2^32 threads: 512 of dK/dV's per 128 rows, 256 of dkv_kernel's per 32
  NRSE_REQUIRE(grid_size(p->rows / BQ + p->nseq, p->hkv, p->hq / p->hkv) < (1LL << 23) &&
                   grid_size(p->rows / 32 + p->nseq, p->hkv, 1) < (1LL << 24),
               "%s: too many workgroups", fn);
  return NRSE_OK;
}

// what is written, and every other operand: an output's workgroups end while others still read
using nrse_overlap::Area;
using nrse_overlap::flat;
int check_apart(const char* fn, std::initializer_list<Area> outs, std::initializer_list<Area> ins) {
  for (auto o = outs.begin(); o != outs.end(); ++o) {
    for (auto i = outs.begin(); i != o; ++i)
      NRSE_REQUIRE(!o->at || !i->at || !meet(*o, *i), "%s: the outputs %s and %s share addresses", fn, i->name, o->name);
    for (const Area& i : ins)
      NRSE_REQUIRE(!o->at || !i.at || !meet(*o, i), "%s: the output %s shares addresses with %s", fn, o->name, i.name);
  }
  return NRSE_OK;
}
#define AREA(x, heads)                                                                                   \
  Area {                                                                                                 \
    #x, (uintptr_t)p->x, p->rows, p->x##_row * es, heads, p->x##_head * es, p->head_dim * es             \
  }
#define PER_ROW(x) flat(#x, p->x, 4LL * p->hq * p->rows)
#define BIAS_SIZED(x) flat(#x, p->x, 4LL * p->hq * (2LL * p->bias_len - 1))
#define LENGTHS flat("cu_seqlens", p->cu_seqlens, 4LL * p->nseq + 4), flat("seq_lens", p->seq_lens, 4LL * p->nseq)
#define ROWS(fn, x) \
  if (const int rc = check_rows(fn, #x, p->x, p->x##_row, p->x##_head, p->dtype, p->head_dim, p->hq)) return rc
#define ROWS_KV(fn, x) \
  if (const int rc = check_rows(fn, #x, p->x, p->x##_row, p->x##_head, p->dtype, p->head_dim, p->hkv)) return rc
#define ROWS_OUT(fn, x, heads) \
  if (const int rc = check_rows(fn, #x, p->x, p->x##_row, p->x##_head, p->dtype, p->head_dim, heads, p->rows)) return rc

}  // namespace

extern "C" int nrse_attn_packed_fwd(const nrse_attn_packed_fwd_params* p, void* stream) {
  const char* fn = "nrse_attn_packed_fwd";
  NRSE_CHECK_PARAMS(p, fn);
  if (const int rc = check_common(fn, p)) return rc;
  if (p->rows == 0 || p->nseq == 0) return NRSE_OK;
  ROWS(fn, q);
  ROWS_KV(fn, k);
  ROWS_KV(fn, v);
  ROWS_OUT(fn, out, p->hq);
  const long long es = p->dtype == NRSE_BF16 ? 2 : 4;
  if (const int rc = check_apart(fn, {AREA(out, p->hq), PER_ROW(lse)},
                                 {AREA(q, p->hq), AREA(k, p->hkv), AREA(v, p->hkv), PER_ROW(gate), BIAS_SIZED(bias_vec), LENGTHS}))
    return rc;
  dispatch(*p, [&](auto t, auto d, auto b, auto c) {
    launch_fwd<decltype(t), decltype(d)::value, decltype(b)::value, decltype(c)::value>(*p, (hipStream_t)stream);
  });
  return nrse_check_launch(fn);
}

extern "C" long long nrse_attn_packed_bwd_workspace(const nrse_attn_packed_bwd_params* p) {
  NRSE_CHECK_PARAMS(p, "nrse_attn_packed_bwd_workspace");
  if (const int rc = check_common("nrse_attn_packed_bwd_workspace", p)) return rc;
  if (p->rows == 0 || p->nseq == 0) return 0;
  const int ns = kv_slices(*p);
  return slab_floats(*p) + (ns > 1 ? 2LL * ns * p->rows * p->hkv * p->head_dim : 0);
}

extern "C" int nrse_attn_packed_bwd(const nrse_attn_packed_bwd_params* p, void* stream) {
  const char* fn = "nrse_attn_packed_bwd";
  NRSE_CHECK_PARAMS(p, fn);
  if (const int rc = check_common(fn, p)) return rc;
  NRSE_REQUIRE(p->bias_vec || (!p->dbias_vec && !p->dgate), "%s: gradients of a bias that is not there", fn);
  NRSE_REQUIRE(p->gate || !p->dgate, "%s: dgate without a gate", fn);
  NRSE_REQUIRE(!p->dbias_vec || p->hq < (1 << 16), "%s: the gradient of a bias of %d heads (65535 at most)", fn, p->hq);
  const hipStream_t st = (hipStream_t)stream;
  if (p->rows == 0 || p->nseq == 0) {
    if (p->dbias_vec && !p->accumulate) {
      const long long n = (long long)p->hq * (2LL * p->bias_len - 1);
      return nrse_zero(p->dbias_vec, n, stream);
    }
    return NRSE_OK;
  }
  ROWS(fn, q);
  ROWS_KV(fn, k);
  ROWS_KV(fn, v);
  ROWS(fn, out);
  ROWS(fn, dout);
  ROWS_OUT(fn, dq, p->hq);
  ROWS_OUT(fn, dk, p->hkv);
  ROWS_OUT(fn, dv, p->hkv);
  NRSE_REQUIRE(p->lse && p->delta, "%s: lse and delta are needed", fn);
  const long long floats = nrse_attn_packed_bwd_workspace(p), es = p->dtype == NRSE_BF16 ? 2 : 4;
  NRSE_REQUIRE(p->part || floats == 0, "%s: part, the workspace, is null", fn);
  NRSE_REQUIRE(((uintptr_t)p->part & 15) == 0, "%s: part, the workspace, is not 16-byte aligned", fn);
  if (const int rc = check_apart(fn,
                                 {AREA(dq, p->hq), AREA(dk, p->hkv), AREA(dv, p->hkv), PER_ROW(delta), PER_ROW(dgate),
                                  BIAS_SIZED(dbias_vec), flat("part", p->part, 4 * floats)},
                                 {AREA(q, p->hq), AREA(k, p->hkv), AREA(v, p->hkv), AREA(out, p->hq), AREA(dout, p->hq),
                                  PER_ROW(lse), PER_ROW(gate), BIAS_SIZED(bias_vec), LENGTHS}))
    return rc;
  dispatch(*p, [&](auto t, auto d, auto b, auto c) {
    launch_bwd<decltype(t), decltype(d)::value, decltype(b)::value, decltype(c)::value>(*p, st);
  });
  if (p->dbias_vec) {
    const int nd = 2 * p->bias_len - 1;
    hipLaunchKernelGGL(dbias_kernel, dim3((nd + 63) / 64, p->hq), dim3(256), 0, st, p->part, p->dbias_vec,
                       ((int)(p->rows / BQ) + p->nseq) * kv_parts(*p), p->bias_len, p->accumulate);
  }
  return nrse_check_launch(fn);
}

extern "C" int nrse_rel_bias_expand(const float* E, const int* edges, int n, float* vec, int H, int T, int causal,
                                    void* stream) {
  NRSE_REQUIRE(E && edges && vec && n > 0 && H > 0 && T > 0 && T <= (1 << 29), "nrse_rel_bias_expand: bad args");
  const Area in[] = {flat("E", E, 4LL * H * (causal ? n : 2LL * n)), flat("edges", edges, 4LL * n)},
             out = flat("vec", vec, 4LL * H * (2LL * T - 1));
  NRSE_REQUIRE(!meet(out, in[0]) && !meet(out, in[1]), "nrse_rel_bias_expand: vec shares addresses with E or edges");
  const long long blocks = (2LL * T - 1 + 255) / 256;
  // a head per workgroup row while that fills the chip, all of them in one loop for a long vector
  const unsigned rows = (unsigned)(blocks >= 1024 ? 1 : std::min(H, 65535));
  hipLaunchKernelGGL(rel_expand_kernel, dim3((unsigned)std::min(blocks, 65536LL), rows), dim3(256), 0, (hipStream_t)stream,
                     E, edges, n, vec, H, T, causal);
  return nrse_check_launch("nrse_rel_bias_expand");
}

extern "C" int nrse_rel_bias_collect(const float* dvec, const int* edges, int n, float* dE, int H, int T, int causal,
                                     int accumulate, void* stream) {
  NRSE_REQUIRE(dvec && edges && dE && n > 0 && H > 0 && T > 0 && T <= (1 << 29), "nrse_rel_bias_collect: bad args");
  const long long items = (causal ? n : 2LL * n) * H;
  const Area in[] = {flat("dvec", dvec, 4LL * H * (2LL * T - 1)), flat("edges", edges, 4LL * n)}, out = flat("dE", dE, 4 * items);
  NRSE_REQUIRE(!meet(out, in[0]) && !meet(out, in[1]), "nrse_rel_bias_collect: dE shares addresses with dvec or edges");
  NRSE_REQUIRE(items < (1LL << 24), "nrse_rel_bias_collect: %lld table entries", items);   // (2^32 threads)
  hipLaunchKernelGGL(rel_collect_kernel, dim3((unsigned)items), dim3(256), 0, (hipStream_t)stream, dvec, edges,
                     n, dE, H, T, causal, accumulate);
  return nrse_check_launch("nrse_rel_bias_collect");
}
