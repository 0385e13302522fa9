// Appending to the 8-bit paged cache (kv_int8.h): norm and rotation on the way, a block's codes,
// scales and bounds once it is full, its 16-bit rows until then.
//
// Norm and rotation are kv_rotate.h's. A token that takes its block's last slot completes it: the
// block's rows that are part of this call are turned again from the input, earlier ones come from
// the sequence's open block (or from the codes, where the block had been full and its sequence was
// cut back into it), and the codes, scales and int8 bounds follow from the 16-bit rows. Bounds are
// those of kv_append.hip.
//
// One launch, no workgroup waits for another. Workgroups at the grid's head look at a tile of
// tokens for one head's keys or values and do the blocks completed there: rows in registers, their
// largest magnitude, then codes (values transposed through LDS). In the others a wave moves a
// token's queries, and its key and value rows to the open block. The open block is read (the first
// block that a call completes) and written (the rows behind the last one) in the same call: a run
// of tokens that begins in one block and ends in a later, open one has these rows written by the
// workgroup that reads the open block first, after it has read.
//
// What bounds it, and what was taken for it: 16384 tokens of 32 rows of 256 channels take 172 us
// (103 at the 4.81 TB/s of a large copy), 9001 normed tokens of 48 rows of 128 71 us (43). The
// blocks' part is three quarters of that: 16 bits to codes is 3 instructions a number and a turn
// through LDS for the values, on rows that arrive after a chain of lookups. Rows that stay in
// registers between the maximum and the codes (334 us when they were read twice), magnitudes and
// bounds two numbers an instruction (230 to 212), and eight waves a workgroup where a block has
// more than 128 channels (212 to 189: more rows under way a CU); earlier rows that come from codes
// are taken there, not by way of the open block (189 to 172 where a call's first blocks have such
// rows). Workgroups of both kinds alternating in the grid instead of the blocks' first were slower.
// A decode step is bound by its launch (5 us; 203 tokens of 14 heads of 64 11 us).
#pragma once

#include <type_traits>

#include "kv_int8.h"
#include "kv_rotate.h"

namespace rt {

// A workgroup's threads: a lane holds up to four rows' chunks of a block of 128 slots, 32
// registers.
constexpr int write_threads(int64_t D) { return D > 128 ? 512 : 256; }

struct WriteArgs : TurnArgs {
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // token and head strides, elements
  int64_t T;
  int32_t Hq, Hkv;
  KvTokens tok;
  KvInt8 cache;
  int8_t* bounds;
  float* bound_scales;
  void* q_out;
  int32_t row_parts;     // waves a token's rows are split over
  uint32_t fill_groups;  // workgroups that look for full blocks
  int32_t tile;          // tokens that one of them looks at
};

// A token's page where it is appended, -1 where it is padding.
__device__ inline int32_t write_page(const WriteArgs& a, const KvPlace& p) {
  if (p.last < 0 || (a.rot > 0 && p.pos >= a.table_len)) return -1;
  return kv_page(a.tok, p, p.last);
}
// Whether token `at` of the call is position `pos` of sequence `seq` and not padding.
__device__ inline bool is_token(const WriteArgs& a, int64_t at, int32_t seq, int64_t pos) {
  if (at < 0 || at >= a.T || pos < 0 || a.tok.seq_ids[at] != seq || a.tok.positions[at] != pos) {
    return false;
  }
  return write_page(a, kv_place(a.tok, at)) >= 0;
}
// Whether the block of token t (at p, not padding) stays open in this call.
__device__ inline bool stays_open(const WriteArgs& a, int64_t t, const KvPlace& p, int32_t seq) {
  const int32_t size = 1 << a.tok.shift, more = size - 1 - (p.pos & (size - 1));
  return !is_token(a, t + more, seq, static_cast<int64_t>(p.pos) + more);
}

// Queries to q_out; key and value rows to the open block, where the call's run of their sequence's
// tokens began in it.
template <class E, int D, int MODE, bool NORM>
__device__ inline void move_rows(const WriteArgs& a, int64_t unit) {
  using V8 = typename Kv<E>::V8;
  constexpr int C = D / 16, SLOTS = kWave / C, FLIGHT = 2;
  const int lane = lane_id() % C, place = lane_id() / C;
  const int64_t t = unit / a.row_parts;
  if (t >= a.T || place >= SLOTS) return;
  const KvPlace p = kv_place(a.tok, t);
  const bool valid = write_page(a, p) >= 0;
  const int size = 1 << a.tok.shift, slot = p.pos & (size - 1);
  int rows = a.Hq;
  int32_t seq = 0;
  if (valid) {
    seq = a.tok.seq_ids[t];
    if (stays_open(a, t, p, seq) &&
        !is_token(a, t - slot - 1, seq, static_cast<int64_t>(p.pos) - slot - 1)) {
      rows += 2 * a.Hkv;
    }
  }
  Pair<E, D, MODE, NORM> pair(a, lane);
  if (valid) pair.load(a, p.pos);
  const int step = a.row_parts * SLOTS;
  const E* q = static_cast<const E*>(a.q) + t * a.q_st;
  const E* k = static_cast<const E*>(a.k) + t * a.k_st;
  const E* v = static_cast<const E*>(a.v) + t * a.v_st;
  E* to_q = static_cast<E*>(a.q_out) + t * a.Hq * D;
  const int64_t open = (static_cast<int64_t>(seq) * a.Hkv << a.tok.shift) * D;
  for (int r0 = static_cast<int>(unit % a.row_parts) * SLOTS + place; r0 < rows;
       r0 += FLIGHT * step) {
    V8 x[FLIGHT][2];
    const E* from[FLIGHT];
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
      const int r = r0 + i * step;
      from[i] = r < a.Hq           ? q + r * a.q_sh
                : r < a.Hq + a.Hkv ? k + (r - a.Hq) * a.k_sh
                                   : v + (r - a.Hq - a.Hkv) * a.v_sh;
      x[i][0] = V8{};
      x[i][1] = V8{};
      if (valid && r < rows) {
        x[i][0] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(from[i]) + pair.chunk[0]);
        x[i][1] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(from[i]) + pair.chunk[1]);
      }
    }
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
      const int r = r0 + i * step;
      if (r >= rows) continue;
      if (valid && r < a.Hq + a.Hkv && (NORM || a.rot > 0)) {
        pair.apply(from[i], a, r < a.Hq ? 0 : 1, x[i]);
      }
      const int64_t head = static_cast<int64_t>(D) << a.tok.shift;  // from head to head
      if (r < a.Hq + a.Hkv) {
        E* to = r < a.Hq ? to_q + r * D
                         : static_cast<E*>(a.cache.k_tail) + open + (r - a.Hq) * head + slot * D;
        __builtin_nontemporal_store(x[i][0], reinterpret_cast<V8*>(to) + pair.chunk[0]);
        __builtin_nontemporal_store(x[i][1], reinterpret_cast<V8*>(to) + pair.chunk[1]);
      } else {
        E* to = static_cast<E*>(a.cache.v_tail) + open + (r - a.Hq - a.Hkv) * head + slot;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int e = 0; e < 8; ++e) to[(8 * pair.chunk[j] + e) << a.tok.shift] = x[i][j][e];
        }
      }
    }
  }
}

// The largest of x over the workgroup (`scratch`: a float a wave).
template <int WAVES>
__device__ inline float group_max(float x, float* scratch) {
  for (int i = 1; i < kWave; i <<= 1) x = fmaxf(x, __shfl_xor(x, i));
  __syncthreads();
  if (lane_id() == 0) scratch[threadIdx.x / kWave] = x;
  __syncthreads();
  x = scratch[0];
  for (int w = 1; w < WAVES; ++w) x = fmaxf(x, scratch[w]);
  return x;
}

// The same of a whole number up to 2^16.
template <int WAVES>
__device__ inline int group_max(int x, float* scratch) {
  return static_cast<int>(group_max<WAVES>(static_cast<float>(x), scratch));
}

// One head's keys (VALUES: values) of a tile of tokens.
template <class E, int D, int MODE, bool NORM, bool VALUES>
struct Fill {
  using V8 = typename Kv<E>::V8;
  using Row = Pair<E, D, MODE, NORM && !VALUES>;
  // a row's chunks of 8 channels, two a lane, lie on neighbouring lanes of one wave
  static constexpr int THREADS = write_threads(D), WAVES = THREADS / kWave;
  static constexpr int C = D / 16, WAVE_ROWS = kWave / C, ROWS = WAVES * WAVE_ROWS;
  static constexpr int ALL = (128 + ROWS - 1) / ROWS;  // rows a lane of the largest block
  const WriteArgs& a;
  char* lds;       // the lanes' least and largest keys; the values' codes
  float* scratch;  // a float a wave
  uint64_t* masks;
  int head, row;   // this thread's (row: ROWS where it has none)
  Row pair;

  __device__ Fill(const WriteArgs& args, int h, char* shared, float* waves, uint64_t* m)
      : a(args), lds(shared), scratch(waves), masks(m), head(h), pair(args, lane_id() % C) {
    row = lane_id() / C < WAVE_ROWS
              ? static_cast<int>(threadIdx.x / kWave) * WAVE_ROWS + lane_id() / C
              : ROWS;
    if (!VALUES) pair.load_weights(a, NORM ? 1 : 0);
  }
  __device__ const E* source(int64_t at) const {
    return VALUES ? static_cast<const E*>(a.v) + head * a.v_sh + at * a.v_st
                  : static_cast<const E*>(a.k) + head * a.k_sh + at * a.k_st;
  }
  // This thread's chunks of a row.
  __device__ void read(const E* from, V8 (&x)[2]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[i] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(from) + pair.chunk[i]);
    }
  }
  // The chunks of a token of this call turned.
  __device__ void turn(int64_t at, int32_t pos, V8 (&x)[2]) const {
    if constexpr (!VALUES) {
      if (NORM || a.rot > 0) {
        Row p = pair;
        p.load_turn(a, pos);
        p.apply(source(at), a, 1, x);
      }
    }
  }
  __device__ int64_t block(int64_t of) const { return (of * a.Hkv + head) << a.tok.shift; }
  __device__ void to_open(int32_t seq, int slot, const V8 (&x)[2]) const {
    const int64_t open = block(seq) * D;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (VALUES) {
        E* to = static_cast<E*>(a.cache.v_tail) + open + slot;
#pragma unroll
        for (int e = 0; e < 8; ++e) to[(8 * pair.chunk[i] + e) << a.tok.shift] = x[i][e];
      } else {
        E* to = static_cast<E*>(a.cache.k_tail) + open + slot * D;
        reinterpret_cast<V8*>(to)[pair.chunk[i]] = x[i];
      }
    }
  }
  __device__ float* scale_of(int32_t page) const {
    return (VALUES ? a.cache.v_scales : a.cache.k_scales) +
           (static_cast<int64_t>(page) * a.Hkv + head);
  }

  // A block that had been full and stays open behind slot `from`: its earlier rows to the open
  // block, eight channels of a slot (values: eight slots of a channel) a thread.
  __device__ void reopen(int32_t page, int32_t seq, int from) const {
    const float scale = *scale_of(page);
    const int size = 1 << a.tok.shift, line = VALUES ? size / 8 : D / 8;
    const int8_t* codes = (VALUES ? a.cache.v_codes : a.cache.k_codes) + block(page) * D;
    E* to = static_cast<E*>(VALUES ? a.cache.v_tail : a.cache.k_tail) + block(seq) * D;
    for (int i = threadIdx.x; i < size * D / 8; i += THREADS) {
      const int slot = VALUES ? i % line * 8 : i / line;
      if (slot >= from) continue;
      const V8 x = numbers(codes + 8 * i, scale);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (VALUES && slot + e >= from) break;
        to[8 * i + e] = x[e];
      }
    }
    __syncthreads();  // (everyone has read the scale)
    if (threadIdx.x == 0) *scale_of(page) = 0.0f;
    __syncthreads();
  }

  // Rows as codes: keys to the cache, values to LDS, whence they go to the cache transposed.
  template <bool ODD>
  __device__ void encode(const BlockCode& code, int32_t page, const V8 (&x)[ALL][2],
                         const bool (&mine)[ALL]) const {
    typedef int V2i __attribute__((ext_vector_type(2)));
    char* to = VALUES ? lds : reinterpret_cast<char*>(a.cache.k_codes) + block(page) * D;
#pragma unroll
    for (int i = 0; i < ALL; ++i) {
      if (!mine[i]) continue;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        V2i out;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          out[h] = code.template four<ODD>(
              static_cast<float>(x[i][j][4 * h]), static_cast<float>(x[i][j][4 * h + 1]),
              static_cast<float>(x[i][j][4 * h + 2]), static_cast<float>(x[i][j][4 * h + 3]));
        }
        *reinterpret_cast<V2i*>(to + (row + i * ROWS) * D + 8 * pair.chunk[j]) = out;
      }
    }
  }
  // Eight codes as the 16-bit numbers that they stand for.
  __device__ static V8 numbers(const int8_t* codes, float scale) {
    typedef int V2i __attribute__((ext_vector_type(2)));
    const V2i c = *reinterpret_cast<const V2i*>(codes);
    V8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = static_cast<E>(static_cast<int8_t>(c[e >> 2] >> (8 * (e & 3))) * scale);
    }
    return x;
  }
  // Where the rows before this call's tokens are: the sequence's open block, or the codes of `page`
  // where it had been full (`scale` > 0; the open block then stays as it is).
  struct Earlier {
    int32_t seq, page;
    int count;  // of them
    float scale;
  };
  // Earlier values, eight slots of a channel a thread (they lie transposed): f(slot, channel, eight
  // numbers).
  template <class F>
  __device__ void earlier_values(const Earlier& had, F&& f) const {
    const int line = 1 << (a.tok.shift - 3);
    const V8* from = reinterpret_cast<const V8*>(static_cast<const E*>(a.cache.v_tail) +
                                                 block(had.seq) * D);
    const int8_t* codes = a.cache.v_codes + block(had.page) * D;
    for (int i = threadIdx.x; i < line * D; i += THREADS) {
      if (i % line * 8 >= had.count) continue;
      f(i % line * 8, i / line, had.scale > 0.0f ? numbers(codes + 8 * i, had.scale) : from[i]);
    }
  }
  // The staged codes [slot][channel] to the cache: four channels of 16 slots a thread.
  __device__ void transpose(int32_t page) const {
    const int size = 1 << a.tok.shift;
    int8_t* to = a.cache.v_codes + block(page) * D;
    for (int i = threadIdx.x; i < D / 4 * (size / 16); i += THREADS) {
      const int c = i % (D / 4) * 4, s = i / (D / 4) * 16;
      v4i out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t x[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          x[b] = *reinterpret_cast<const uint32_t*>(lds + (s + 4 * j + b) * D + c);
        }
        // bytes (slot, channel) 4 x 4 the other way round
        const uint32_t p = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u);
        const uint32_t q = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
        const uint32_t r = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
        const uint32_t t = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
        out[0][j] = static_cast<int>(__builtin_amdgcn_perm(q, p, 0x05040100u));
        out[1][j] = static_cast<int>(__builtin_amdgcn_perm(q, p, 0x07060302u));
        out[2][j] = static_cast<int>(__builtin_amdgcn_perm(t, r, 0x05040100u));
        out[3][j] = static_cast<int>(__builtin_amdgcn_perm(t, r, 0x07060302u));
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        *reinterpret_cast<v4i*>(to + ((c + k) << a.tok.shift) + s) = out[k];
      }
    }
  }

  // The largest finite magnitude of a block that has others.
  __device__ float finite_most(const Earlier& had, const V8 (&x)[ALL][2],
                               const bool (&mine)[ALL]) const {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < ALL; ++i) {
      if (!mine[i]) continue;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          most = fmaxf(most, finite_size(static_cast<float>(x[i][j][e])));
        }
      }
    }
    if constexpr (VALUES) {
      earlier_values(had, [&](int slot, int, V8 v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (slot + e < had.count) most = fmaxf(most, finite_size(static_cast<float>(v[e])));
        }
      });
    }
    return most;
  }

  // The block that token t completes. Its rows stay in registers: their largest magnitude first,
  // then the codes.
  __device__ void fill(int64_t t) const {
    const KvPlace p = kv_place(a.tok, t);
    const int32_t page = kv_page(a.tok, p, p.last), seq = a.tok.seq_ids[t];
    const int size = 1 << a.tok.shift;
    // the slots before this call's tokens: a thread a slot
    {
      const int o = threadIdx.x;
      const int64_t from = t - (size - 1 - o);
      const bool here = o < size && from >= 0 && a.tok.positions[from] == p.pos - (size - 1 - o) &&
                        a.tok.seq_ids[from] == seq;
      const uint64_t m = __ballot(here);
      if (lane_id() == 0 && threadIdx.x < 2 * kWave) masks[2 + threadIdx.x / kWave] = m;
    }
    __syncthreads();
    const uint64_t lo = masks[2], hi = masks[3];
    // (t is among them)
    const int earlier = lo ? __builtin_ctzll(lo) : kWave + __builtin_ctzll(hi);
    const Earlier had{seq, page, earlier, earlier > 0 ? *scale_of(page) : 0.0f};
    V8 x[ALL][2];
    bool mine[ALL];
#pragma unroll
    for (int i = 0; i < ALL; ++i) {
      const int o = row + i * ROWS;
      mine[i] = row < ROWS && o < size && (!VALUES || o >= earlier);
      if (mine[i]) {
        read(o < earlier ? static_cast<const E*>(a.cache.k_tail) + (block(seq) + o) * D
                         : source(t - (size - 1 - o)),
             x[i]);
      }
    }
    if (!VALUES && had.scale > 0.0f) {  // (the rows of the open block are not this block's)
#pragma unroll
      for (int i = 0; i < ALL; ++i) {
        const int o = row + i * ROWS;
        if (!mine[i] || o >= earlier) continue;
        const int8_t* codes = a.cache.k_codes + (block(page) + o) * D;
#pragma unroll
        for (int j = 0; j < 2; ++j) x[i][j] = numbers(codes + 8 * pair.chunk[j], had.scale);
      }
    }
    // the largest magnitude, as the 15 bits below the sign
    v2u16 bits{0, 0};
    const auto see = [&](const V8& v) {
      const v4i w = __builtin_bit_cast(v4i, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) bits = max_magnitude(bits, static_cast<uint32_t>(w[i]));
    };
#pragma unroll
    for (int i = 0; i < ALL; ++i) {
      const int o = row + i * ROWS;
      if (!mine[i]) continue;
      if (o >= earlier) turn(t - (size - 1 - o), p.pos - (size - 1 - o), x[i]);
      see(x[i][0]);
      see(x[i][1]);
    }
    if constexpr (VALUES) {
      earlier_values(had, [&](int slot, int, V8 v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (slot + e >= earlier) v[e] = static_cast<E>(0.0f);
        }
        see(v);
      });
    }
    const int top = group_max<WAVES>(bits[0] > bits[1] ? bits[0] : bits[1], scratch);
    const bool odd = top >= kInfinityBits<E>;
    float most = from_bits<E>(top);
    if (odd) most = group_max<WAVES>(finite_most(had, x, mine), scratch);
    most = fmaxf(most, kKvTopFloor);
    const BlockCode code(most, odd);
    if (threadIdx.x == 0) *scale_of(page) = most / 127.0f;
    if (code.odd) {
      encode<true>(code, page, x, mine);
    } else {
      encode<false>(code, page, x, mine);
    }
    if constexpr (VALUES) {
      earlier_values(had, [&](int slot, int d, V8 v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (slot + e >= earlier) break;
          const uint32_t w = code.template word<true>(static_cast<float>(v[e]));
          lds[(slot + e) * D + d] = static_cast<char>(w);
        }
      });
      __syncthreads();
      transpose(page);
    } else {
      if (odd) {
        bounds<true>(page, x, mine);
      } else {
        bounds<false>(page, x, mine);
      }
    }
    // The first block of a run that ends in an open one: that one's rows, which are not moved (the
    // open block has been read now).
    if (!is_token(a, t - size, seq, static_cast<int64_t>(p.pos) - size)) {
      int64_t full = 0;  // blocks behind this one that are completed as well
      for (;;) {
        __syncthreads();
        const int64_t n = size * (full + threadIdx.x + 1);
        const uint64_t no = ~__ballot(is_token(a, t + n, seq, p.pos + n));
        if (lane_id() == 0) scratch[threadIdx.x / kWave] = no ? __builtin_ctzll(no) : kWave;
        __syncthreads();
        int more = 0;
        for (int i = 0; i < WAVES && more == i * kWave; ++i) {
          more += static_cast<int>(scratch[i]);
        }
        full += more;
        if (more < THREADS) break;
      }
      const int64_t first = t + size * full + 1;
      const int32_t pos = static_cast<int32_t>(p.pos + size * full + 1);
      if (row < ROWS) {
        for (int o = row; o < size - 1; o += ROWS) {
          if (!is_token(a, first + o, seq, static_cast<int64_t>(pos) + o)) break;
          V8 x[2];
          read(source(first + o), x);
          turn(first + o, pos + o, x);
          to_open(seq, o, x);
        }
      }
    }
    __syncthreads();
  }

  // The bounds of a block: a lane's least and largest keys (16-bit numbers all) through LDS. ODD:
  // NaN is passed over.
  template <bool ODD>
  __device__ void bounds(int32_t page, const V8 (&x)[ALL][2], const bool (&mine)[ALL]) const {
    E(*lows)[D] = reinterpret_cast<E(*)[D]>(lds);
    E(*highs)[D] = lows + ROWS;
    if (row < ROWS) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        V8 low, high;
        if constexpr (ODD) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float l = INFINITY, h = -INFINITY;
#pragma unroll
            for (int i = 0; i < ALL; ++i) {
              const float f = static_cast<float>(x[i][j][e]);
              l = mine[i] ? fminf(l, f) : l;
              h = mine[i] ? fmaxf(h, f) : h;
            }
            low[e] = static_cast<E>(l);
            high[e] = static_cast<E>(h);
          }
        } else {
          v4i ends[2];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v2i16 l, h;
#pragma unroll
            for (int i = 0; i < ALL; ++i) {
              const v4i w = __builtin_bit_cast(v4i, x[i][j]);
              const v2i16 v = ordered(static_cast<uint32_t>(w[k]));
              if (i == 0) {  // (a lane has its first row, or none)
                l = h = v;
              } else if (mine[i]) {
                l = __builtin_elementwise_min(l, v);
                h = __builtin_elementwise_max(h, v);
              }
            }
            ends[0][k] = __builtin_bit_cast(
                int, ordered(__builtin_bit_cast(uint32_t, l)));
            ends[1][k] = __builtin_bit_cast(
                int, ordered(__builtin_bit_cast(uint32_t, h)));
          }
          low = __builtin_bit_cast(V8, ends[0]);
          high = __builtin_bit_cast(V8, ends[1]);
        }
        *reinterpret_cast<V8*>(&lows[row][8 * pair.chunk[j]]) = low;
        *reinterpret_cast<V8*>(&highs[row][8 * pair.chunk[j]]) = high;
      }
    }
    __syncthreads();
    const int d = threadIdx.x;
    float mid = 0.0f, half = 0.0f;
    if (d < D) {
      const int rows = ROWS < (1 << a.tok.shift) ? ROWS : 1 << a.tok.shift;
      float l = static_cast<float>(lows[0][d]), h = static_cast<float>(highs[0][d]);
#pragma unroll 4
      for (int i = 1; i < rows; ++i) {
        l = fminf(l, static_cast<float>(lows[i][d]));
        h = fmaxf(h, static_cast<float>(highs[i][d]));
      }
      mid = (l + h) * 0.5f;
      half = (h - l) * 0.5f;
    }
    const float top = fmaxf(group_max<WAVES>(fmaxf(fabsf(mid), half), scratch), kKvTopFloor);
    const int64_t at = static_cast<int64_t>(page) * a.Hkv + head;
    if (d < D) {
      a.bounds[at * 2 * D + d] = static_cast<int8_t>(kv_code(mid, top));
      a.bounds[at * 2 * D + D + d] = static_cast<int8_t>(kv_code(half, top));
    }
    if (d == 0) a.bound_scales[at] = top / 127.0f;
  }

  __device__ void run(int64_t t0) {
    const int size = 1 << a.tok.shift;
    if (threadIdx.x < kWave) {  // one token a lane
      const int64_t mine = t0 + lane_id();
      bool full = false, again = false;
      if (lane_id() < a.tile && mine < a.T) {
        const KvPlace p = kv_place(a.tok, mine);
        const int32_t page = write_page(a, p);
        if (page >= 0) {
          const int32_t seq = a.tok.seq_ids[mine];
          const int slot = p.pos & (size - 1);
          full = slot == size - 1;
          // the first token of a block that stays open
          if (!full &&
              (slot == 0 || !is_token(a, mine - 1, seq, static_cast<int64_t>(p.pos) - 1)) &&
              stays_open(a, mine, p, seq)) {
            again = slot > 0 && *scale_of(page) > 0.0f;
            if (!again) *scale_of(page) = 0.0f;
          }
        }
      }
      const uint64_t f = __ballot(full), r = __ballot(again);
      if (lane_id() == 0) {
        masks[0] = f;
        masks[1] = r;
      }
    }
    __syncthreads();
    for (uint64_t left = masks[1]; left != 0; left &= left - 1) {
      const int64_t t = t0 + __builtin_ctzll(left);
      const KvPlace p = kv_place(a.tok, t);
      reopen(kv_page(a.tok, p, p.last), a.tok.seq_ids[t], p.pos & (size - 1));
    }
    for (uint64_t left = masks[0]; left != 0; left &= left - 1) {
      fill(t0 + __builtin_ctzll(left));
    }
  }
};

// Waves a SIMD that the registers leave room for.
constexpr int write_waves(int mode, bool norm) { return mode == kRotHalfOdd ? 2 : norm ? 3 : 4; }

template <class E, int D, int MODE, bool NORM>
__global__ void __launch_bounds__(write_threads(D), write_waves(MODE, NORM))
    kv_append_int8_kernel(WriteArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int WAVES = write_threads(D) / kWave;
  __shared__ float scratch[WAVES];
  __shared__ uint64_t masks[4];  // tokens that complete a block, that open one again; slots
  if (blockIdx.x < a.fill_groups) {
    const int job = static_cast<int>(blockIdx.x % (2 * a.Hkv));
    const int64_t t0 = static_cast<int64_t>(blockIdx.x / (2 * a.Hkv)) * a.tile;
    if (job < a.Hkv) {
      Fill<E, D, MODE, NORM, false>(a, job, lds, scratch, masks).run(t0);
    } else {
      Fill<E, D, MODE, NORM, true>(a, job - a.Hkv, lds, scratch, masks).run(t0);
    }
  } else {
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    move_rows<E, D, MODE, NORM>(
        a, static_cast<int64_t>(blockIdx.x - a.fill_groups) * WAVES + wave);
  }
}

template <class E, int D>
int append_int8_launch(const WriteArgs& a, unsigned grid, unsigned lds, bool interleaved,
                       hipStream_t s) {
  return kv_turn_dispatch(a.rot, interleaved, a.norm[0].weight || a.norm[1].weight,
                          [&](auto mode, auto norm) -> int {
    kv_append_int8_kernel<E, D, decltype(mode)::value, decltype(norm)::value>
        <<<dim3(grid), dim3(write_threads(D)), lds, s>>>(a);
    RT_CHECK_HIP(hipGetLastError());
    return kOk;
  });
}

// The kernels of a type for heads of up to 128 channels, and of more: a file each.
using AppendInt8 = int(int64_t D, const WriteArgs& a, unsigned grid, unsigned lds, bool interleaved,
                       hipStream_t s);
AppendInt8 append_int8_bf16_128, append_int8_bf16_256, append_int8_f16_128, append_int8_f16_256;

}  // namespace rt
