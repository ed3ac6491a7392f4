// What the kernels of the text side's attention share: the arguments, which keys a tile has, the bias by buckets, and the
// LDS tiles of 64 rows that feed 32x32x16 MFMAs both along the rows and, transposed by the reads, across them.
#pragma once

#include <math.h>

#include <algorithm>

#include "common.h"

namespace selas {
namespace textattn {

constexpr int kRows = 64;              // rows (keys or queries) per LDS tile
constexpr int kMaxSide = 128;          // buckets per direction
constexpr int kMaxDistance = 512;      // tables and histograms by distance have to fit LDS beside the tiles
constexpr float kLowest = -3.402823466e38f;
constexpr float kEntry = 131072.0f;  // the largest entry of a bias table that counts as it is
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint32_t kPast = 0x80000000u;  // a byte offset past every buffer range here (ranges stay below 2^31): loads read 0

// [B, heads, rows, channels] with unit channel stride; strides in elements.
struct Side {
  const uint16_t *p;
  int64_t sb, sh, sl;
};

// The learned bias: bucket t of a direction begins at distance edge[t], and from `reach` = edge[n - 1] on the bias no
// longer changes. Keys after the query have the buckets from `ahead` on, or bucket 0 where there is one direction only.
struct Bias {
  const void *table;  // [buckets, H], unit column stride; null: no bias
  int64_t row;
  float inv_scale;  // 1 / scale
  int dtype, n, ahead, reach;
  int edge[kMaxSide];  // from n on: beyond every distance
};

struct Args {
  Side q, k, v;
  uint16_t *out;  // [B, Lq, H * dh], unit column stride
  int64_t out_sb, out_sl;
  float *lse;  // [B, H, Lq] or null
  const int32_t *lengths;  // [B] or null
  const uint8_t *mask;     // [B, Lk] or null
  int64_t mask_sb;
  const int32_t *start;  // position of each image's first query, [B], or null: start0 for all
  int start0;
  int B, H, Hk, group, Lq, Lk, dh, causal;
  float c2;  // scale * log2(e)
  Bias bias;
};

// The arguments of a kernel whose first is an Args, read again where they are used: what is needed only after a loop holds no
// scalar registers in it.
__device__ __forceinline__ const Args &args_here() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Args *)p;
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Keys of image b; the position of its first query. Both are uniform (scalar loads: a vector load's wait would also wait
// for the tiles in flight), and bounded so that sums with them stay in 32 bits.
__device__ __forceinline__ int scalar_load(const int32_t *p, int i) {
  return reinterpret_cast<const __attribute__((address_space(4))) int32_t *>(reinterpret_cast<uintptr_t>(p))[uniform(i)];
}
__device__ __forceinline__ int start_of(const Args &a, int b) {
  const int s = a.start ? scalar_load(a.start, b) : a.start0;
  return min(max(s, -(1 << 29)), 1 << 29);
}
// With a causal mask the keys past the last query's position are none: what they hold must not reach a product either.
__device__ __forceinline__ int keys_of(const Args &a, int b) {
  int n = a.lengths ? min(scalar_load(a.lengths, b), a.Lk) : a.Lk;
  if (a.causal) n = min(n, start_of(a, b) + a.Lq);
  return max(n, 0);
}

__device__ __forceinline__ int split(int v, FastDiv by, int d, int &rest) {  // v % d, and rest = v / d
  const int r = static_cast<int>(div31(v, by));
  rest = r;
  return v - r * d;
}

// ------------------------------------------------------------------ element types

template <bool BF>
__device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two values, already in registers of their own, rounded to nearest even into a packed pair.
template <bool BF>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  if constexpr (BF) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 v = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
  }
}

template <bool BF>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack<BF>(v[0], v[1]), pack<BF>(v[2], v[3]), pack<BF>(v[4], v[5]), pack<BF>(v[6], v[7]));
}
template <bool BF>
__device__ __forceinline__ float lo_of(uint32_t w) {
  return BF ? __uint_as_float(w << 16) : f16_bits_to_f32(static_cast<uint16_t>(w));
}
template <bool BF>
__device__ __forceinline__ float hi_of(uint32_t w) {
  return BF ? __uint_as_float(w & 0xffff0000u) : f16_bits_to_f32(static_cast<uint16_t>(w >> 16));
}

// The probabilities of a forward pass are 2^(s - m) with m this far below the maximum: fp16 has room for it, and then
// holds weights down to 2^-21 of the largest at full precision instead of 2^-14.
template <bool BF>
__device__ constexpr float headroom() {
  return BF ? 0.0f : 7.0f;
}

__device__ __forceinline__ float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ------------------------------------------------------------------ the bias by distance

// The table of head `head` as a function of distance d = key - query, divided by the scale, so that it is added to the
// products of queries and keys. Beyond `reach` it is constant, so
// d in [-reach - 8, reach + 8] is all of it: runs of 8 distances starting anywhere are entries of it once their start is
// clamped to [-reach - 8, reach + 1]. Lanes read runs of 4 distances that start anywhere, in one 16-byte read each: copy c
// (of 4) begins c entries later, so that a run starting at i is aligned in copy i % 4. The copies are `bias_pitch` floats
// apart, 64 bytes past a multiple of 256: the 16 lanes of a read then meet 16 different groups of banks.
__host__ __device__ inline int bias_pitch(int reach) { return (2 * reach + 20 + 47) / 64 * 64 + 16; }
__host__ __device__ inline int bias_bytes(int reach) { return 4 * 4 * bias_pitch(reach); }

__device__ __forceinline__ int bucket_of(const Bias &t, int d) {
  const int side = t.ahead ? abs(d) : max(-d, 0);
  int r = t.ahead && d > 0 ? t.ahead - 1 : -1;
  for (int i = 0; i < t.n; i += 8)  // edge[0] = 0; eight at a time, which are one scalar load
#pragma unroll
    for (int j = 0; j < 8; ++j) r += side >= t.edge[i + j];
  return r;
}

__device__ __forceinline__ float bias_at(const Bias &t, int head, int d, float mul) {
  const int64_t i = bucket_of(t, d) * t.row + head;
  const float v = t.dtype == SELAS_F32   ? load_f<SELAS_F32>(t.table, i)
                  : t.dtype == SELAS_F16 ? load_f<SELAS_F16>(t.table, i)
                                         : load_f<SELAS_BF16>(t.table, i);
  // Finite entries count as +-2^17 beyond it. The lowest numbers of fp32 and bf16, divided by the scale, would be -inf and hide
  // the key; from 1e9 on the difference of a score and its rounded maximum would overflow as an exponent; and products of
  // queries and keys would be lost beside the entry (at 2^17 scores keep 2^-7).
  return (fabsf(v) < __builtin_inff() ? fminf(fmaxf(v, -kEntry), kEntry) : v) * mul;
}

// The four copies of a head's table, into LDS, by all threads of the workgroup; reversed: by query - key. Building them once
// per call, by a launch of its own, took 5 us and gained nothing at any batch.
__device__ __forceinline__ void build_bias(float *lds, const Bias &t, int head, int threads, bool reversed) {
  const int pitch = bias_pitch(t.reach);
  for (int i = threadIdx.x; i < 2 * t.reach + 17; i += threads) {
    const int d = i - t.reach - 8;
    const float v = bias_at(t, head, reversed ? -d : d, t.inv_scale);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (i >= c) lds[c * pitch + i - c] = v;
  }
}

// Eight entries from distance d on.
__device__ __forceinline__ void bias_run(const float *lds, int pitch, int reach, int d, float (&v)[8]) {
  const int i = min(max(d, -reach - 8), reach + 1) + reach + 8;
  const float *p = lds + (i & 3) * pitch + (i & ~3);
  const f32x4 x = *reinterpret_cast<const f32x4 *>(p), y = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = x[e];
    v[4 + e] = y[e];
  }
}

// ------------------------------------------------------------------ LDS tiles

// 64 rows of D channels (dh of them given, the rest zeros), in 16-byte chunks. A DMA instruction fills 1 KiB, a group of 4
// (D = 128) or 8 rows; the groups are 16 bytes further apart than that, and within a group a chunk's place in its row is
// XORed with a function of the row. So two kinds of read are free of bank conflicts: 16 rows at one chunk (a row-wise
// operand), and 4 rows at 64 bytes (ds_read_b64_tr_b16, a transposed operand); and since the function is the same in every
// group, a lane needs few addresses: the rest is in the instructions' offsets.
template <int D>
struct Tile {
  static constexpr int kRow = 2 * D;        // bytes
  static constexpr int kChunks = D / 8;     // per row
  static constexpr int kGroupRows = 1024 / kRow, kGroup = 1024 + 16;
  static constexpr int kLoads = kRows / kGroupRows;
  static constexpr int kBytes = kLoads * kGroup;
  __device__ static __forceinline__ int swizzle(int r) {  // of row r of a group
    return D == 128 ? r << 2 : (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1);
  }
  static constexpr int at(int r) { return r / kGroupRows * kGroup; }  // offset of the group that begins with row r

  // A wave's share of the loads: instructions KJ * wave + j, whose lane fills row `row(j)`.
  template <int KJ>
  struct Loader {
    uint32_t voff;
    int wave, lane;
    __device__ __forceinline__ int row(int j) const { return (KJ * wave + j) * kGroupRows + lane / kChunks; }
    __device__ __forceinline__ Loader(int wave_, int lane_, int64_t sl, int dh) : wave(wave_), lane(lane_) {
      const int r = lane / kChunks, chunk = (lane & (kChunks - 1)) ^ swizzle(r);
      voff = 8 * chunk < dh ? static_cast<uint32_t>(r) * static_cast<uint32_t>(2 * sl) + 16 * chunk : kPast;
    }
    // The tile whose first row is at `p`, of which `rows` exist (the others read as zeros, and so do rows whose bit in
    // `bits` is not set where PART is).
    template <bool PART>
    __device__ __forceinline__ void issue(uint8_t *lds, const uint16_t *p, int64_t sl, int dh, int rows, uint64_t bits) const {
      rows = min(rows, kRows);
      const uint32_t bytes = rows > 0 ? 2 * ((rows - 1) * static_cast<uint32_t>(sl) + dh) : 0;
      const __amdgpu_buffer_rsrc_t r = make_rsrc(p, bytes);
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        const int J = KJ * wave + j;
        uint32_t off = voff;
        if constexpr (PART) off = (bits >> row(j)) & 1 ? off : kPast;
        load_lds16(r, lds + J * kGroup, off, static_cast<uint32_t>(J * kGroupRows) * static_cast<uint32_t>(2 * sl));
      }
    }
  };

  // Row-wise operand: lane (c, h) reads channels 16 s + 8 h .. + 8 of row 32 blk + swap23(c) (bits 2 and 3 exchanged).
  struct RowReader {
    uint32_t off[4];
    __device__ __forceinline__ RowReader(int lane) {
      const int c = lane & 31, r = (c & ~12) | ((c & 4) << 1) | ((c & 8) >> 1), r8 = r % kGroupRows;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int chunk = (D == 128 ? 4 * i : 2 * i) + (lane >> 5);
        off[i] = r / kGroupRows * kGroup + r8 * kRow + ((chunk ^ swizzle(r8)) << 4);
      }
    }
    __device__ __forceinline__ uint4 read(const uint8_t *lds, int blk, int s) const {
      return *reinterpret_cast<const uint4 *>(lds + (D == 128 ? off[s >> 1] + 32 * (s & 1) : off[s]) + at(32 * blk));
    }
  };

  // Transposed operand: lane (c, h) receives channel 32 db + c of rows 32 blk + 16 t + 8 h .. + 8.
  struct ColReader {
    uint32_t off[4];
    __device__ __forceinline__ ColReader(int lane) {
      const int h = lane >> 5, r4 = (lane >> 2) & 3, x = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int db = D == 128 ? i : i >> 1, r = 8 * h + r4 + (D == 128 ? 0 : 4 * (i & 1)), r8 = r % kGroupRows;
        off[i] = r / kGroupRows * kGroup + r8 * kRow + (((4 * db + x) ^ swizzle(r8)) << 4) + 8 * (lane & 1);
      }
    }
    __device__ __forceinline__ uint4 read(uint8_t *lds, int db, int blk, int t) const {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      auto half = [&](int u) {
        const uint32_t o = D == 128 ? off[db] + u * at(4) : off[2 * db + u];
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4 *)(lds + o + at(32 * blk + 16 * t)));
      };
      const s16x4 lo = half(0), hi = half(1);
      return __builtin_bit_cast(uint4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
};

// The kernels are built for 64, 96 and 128 channels; 96 are laid out as 128, whose last quarter no instruction reads.
template <int D>
using TileOf = Tile<D == 64 ? 64 : 128>;

// A wave's 32 rows as the B operand, in registers for the whole loop: lane (c, h) holds channels 16 s + 8 h .. + 8 of row c.
// Rows that do not exist and channels from dh on are zeros.
template <int D>
struct Held {
  uint4 f[D / 16];
  __device__ __forceinline__ void load(const uint16_t *p, int64_t sl, int dh, int rows, int lane, bool keep = true) {
    rows = min(rows, 32);
    const uint32_t bytes = rows > 0 ? 2 * ((rows - 1) * static_cast<uint32_t>(sl) + dh) : 0;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(p, bytes);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const int ch = 16 * s + 8 * (lane >> 5);
      const uint32_t off = static_cast<uint32_t>(lane & 31) * static_cast<uint32_t>(2 * sl) + 2 * ch;
      f[s] = load_b128(r, ch < dh && keep ? off : kPast, 0);
    }
  }
};

// ------------------------------------------------------------------ which keys a tile has

// Bit i of a tile's word: key 64 kt + i exists and is not masked. The mask's bytes are loaded a tile ahead of their use.
struct KeyBits {
  const uint8_t *mask;  // of this image, or null
  int keys, lane;
  __device__ __forceinline__ KeyBits(const Args &a, int b, int keys_, int lane_)
      : mask(a.mask ? a.mask + b * a.mask_sb : nullptr), keys(keys_), lane(lane_) {}
  __device__ __forceinline__ int load(int kt) const {
    const int key = kt * kRows + lane;
    return mask && key < keys ? mask[key] : 0;
  }
  __device__ __forceinline__ uint64_t word(int kt, int byte) const {
    if (mask) return __builtin_amdgcn_ballot_w64(byte != 0);
    const int rows = keys - kt * kRows;
    return rows >= kRows ? ~0ull : rows > 0 ? ~0ull >> (kRows - rows) : 0ull;
  }
};

// The low n + 1 bits (none below 0, all from 63 on): the keys at or before position n of a tile.
__device__ __forceinline__ uint64_t up_to(int n) { return n < 0 ? 0ull : n >= 63 ? ~0ull : (2ull << n) - 1; }

// ------------------------------------------------------------------ host side

int cu_count();
// A stride as the kernels take it. That of an axis of one element says nothing and may be anything: one row's becomes a
// head's width, so that the rows after it are past the buffers' ranges as they are elsewhere.
inline int64_t stride_of(int64_t n, int64_t given, int64_t alone) { return n > 1 ? given : alone; }
inline int width_of(int dh) { return dh <= 64 ? 64 : dh <= 96 ? 96 : 128; }
// Fills and checks the arguments; `pointers`: of a call, not only of a question about sizes.
int check_args(const char *what, const selas_text_attention_problem *p, int dtype, bool pointers, Args &a);
// The largest launch of a call, in threads of one dimension: a grid holds fewer than 2^32.
struct Threads {
  int64_t most = 0;
  void add(int64_t blocks, int64_t threads) { most = std::max(most, blocks * threads); }
  int check(const char *what) const {
    if (most < (1ll << 32)) return SELAS_OK;
    return set_error(SELAS_EUNSUPPORTED, "%s: a launch of 2^32 threads or more (%lld)", what, (long long)most);
  }
};
// Which work item a block takes: the XCDs, which blocks reach in turn, take chunks of consecutive items in turn. One chunk
// each, so that most items that read the same rows meet one L2; where images differ in length (`ragged`) the `inner` items
// of one (image, key head, part), which read the same, are a chunk, so that every XCD has short and long images: 16 x 64
// heads of texts of 30 to 512 tokens otherwise took as long as if all had 512. Unless that leaves XCDs unequal numbers.
struct Deal {
  int total, chunk, blocks;
  FastDiv by_chunk;
};
inline Deal deal(int64_t total, int64_t inner, bool ragged) {
  const int64_t units = total / std::max<int64_t>(inner, 1);
  const int64_t chunk = std::max<int64_t>(1, ragged && (units % 8 == 0 || units >= 32) ? inner : cdiv(total, 8));
  return {static_cast<int>(total), static_cast<int>(chunk), static_cast<int>(8 * chunk * cdiv(cdiv(total, chunk), 8)),
          fast_div(static_cast<uint32_t>(chunk))};
}
__device__ __forceinline__ int item_of(const Deal &d) {
  const int i = blockIdx.x >> 3, turn = static_cast<int>(div31(i, d.by_chunk));
  return (8 * turn + (blockIdx.x & 7)) * d.chunk + i - turn * d.chunk;
}

}  // namespace textattn
}  // namespace selas
