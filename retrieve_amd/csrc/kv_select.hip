// The best blocks of each token and key/value head, by the int8 bounds' score.
//
// A query head's row is quantised as the bounds are (codes c, scale s); block b's score with it is
// (c . mid_b + |c| . half_b) s times the block's scale, an upper bound on what any of its keys can
// score, and the group's score is the largest of its heads'. The sum is an int32 (at most
// 2 * 256 * 127^2 < 2^23, so exact as fp32 too); the two products are rounded once each, in this
// order, and rounding is monotone, so the largest over the heads is taken before the block's scale.
//
// One launch for single tokens over few blocks, else two: scores and cut.
//
// Scores: [blocks x columns] = bounds [c | |c|]^T on the int8 matrix cores, 16 blocks by 16 columns
// an instruction; the columns stay in registers (quantised by the wave that needs them), the bounds
// come from memory in the operand's layout. Decode: a column is a query head of the wave's one
// token, the largest of them found by lane exchange. Prompts: a column is a token, a tile one
// head of 16 tokens, the largest over the heads found within the lane; the tokens of one sequence
// share the pass over its blocks. One key a (token, head, block) is left behind.
//
// Bound: single tokens by the bounds' bytes, 2 D a (block, head) in scattered pieces (64 sequences
// of 16K to 131K tokens in blocks of 64, 8 heads of 128 channels: 51 us, 3.0 TB/s, the longest
// row's chain behind the others), one launch for up to 4096 blocks; a million tokens of one
// sequence take 13 us of scores and 8 of the cut. Prompts by the vector instructions: a column's
// codes (ten instructions a channel) and a block's key (about seven a head): 4099 tokens over 9K
// to 30K take 76 us.
//
// Keep: few blocks by a wave, which bisects over the keys' bits from the highest in which they
// differ until the count is exact. Many by a workgroup: the want-th largest of the lanes' largest
// keys is a bound that at least `want` keys reach and few more; those are ranked against each
// other.
#include <type_traits>

#include "../../include/retrieve_amd.h"
#include "kv_common.h"

namespace rt {

constexpr int kScoreWaves = 4;  // heads of a workgroup: a page's bounds lie side by side
constexpr int kChunk = 64;      // blocks a wave looks up at a time

struct SelectArgs {
  const void* q;
  int64_t q_st, q_sh;
  int64_t T;
  int32_t Hq, Hkv, G;
  const int8_t* bounds;
  const float* scales;
  KvTokens tok;
  int32_t count, sink, recent;
  int32_t want;       // places for blocks chosen by their score (of a cache without pages: none)
  int32_t* out;       // [T, Hkv, count]
  uint32_t* keys;     // [T * Hkv, stride]
  int64_t stride;
  int32_t splits;     // waves that share a wave's tokens' blocks
  int32_t head_groups;
  int32_t above;      // rows of so many candidates or fewer are another launch's (-1: none)
};

// The key of a candidate's score, the group's times the block's scale (0: not a candidate). A score
// that is not a number is the least. (The sum with 0 makes -0, of a block of scale 0, the other
// zero's equal.)
__device__ inline uint32_t score_key(float group, float scale) {
  return key_of_f32(fmaxf(fmaf(group, scale, 0.0f), -INFINITY));
}

// The largest over aligned groups of 16 lanes, in every lane.
__device__ inline float group_max16(float x) {
  auto step = [&](auto ctrl) {
    const int y = __builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf,
                                              true);
    x = fmaxf(x, __int_as_float(y));
  };
  step(std::integral_constant<int, 0xB1>{});   // lane ^ 1
  step(std::integral_constant<int, 0x4E>{});   // lane ^ 2
  step(std::integral_constant<int, 0x141>{});  // the other four of eight
  step(std::integral_constant<int, 0x140>{});  // the other eight of sixteen
  return x;
}

// The largest (or least) over the wave, in every lane.
template <bool MAX>
__device__ inline uint32_t wave_extreme(uint32_t x) {
  auto step = [&](auto ctrl) {
    // lanes without a source keep their own value
    const uint32_t y = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        static_cast<int>(x), static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf, false));
    x = (MAX ? y > x : y < x) ? y : x;
  };
  step(std::integral_constant<int, 0x111>{});  // row_shr 1, 2, 4, 8
  step(std::integral_constant<int, 0x112>{});
  step(std::integral_constant<int, 0x114>{});
  step(std::integral_constant<int, 0x118>{});
  step(std::integral_constant<int, 0x142>{});  // row_bcast 15, 31: lane 63 has them all
  step(std::integral_constant<int, 0x143>{});
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), 63));
}

// 16 channels of a query row as codes (or their sizes): the bytes of one operand step.
template <class V8>
__device__ inline void pack_codes(const V8 (&x)[2], float top, float r, float small, v4i& codes,
                                  v4i& sizes) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t c4 = 0, s4 = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 4 * w + e;
      const float v = kv_code_value(static_cast<float>(x[i >> 3][i & 7]) * small, top, r);
      c4 = __builtin_amdgcn_cvt_pk_u8_f32(v + 128.0f, e, c4);
      s4 = __builtin_amdgcn_cvt_pk_u8_f32(fabsf(v), e, s4);
    }
    codes[w] = static_cast<int>(c4 ^ 0x80808080u);
    sizes[w] = static_cast<int>(s4);
  }
}

// A wave holds NT tiles of 16 columns. GH = 0 (decode): one token, column = query head, 16 NT heads
// a pass. GH > 0 (prompts): column = token, tile n = head n % GH of token group n / GH, GH heads a
// pass (heads past the group's repeat its last).
// Chunks first, first + step, ... of 64 blocks are scored; `put(token, block)` is where the keys of
// four blocks go.
struct ScoreLds {
  __attribute__((aligned(16))) int32_t pages[2][kChunk];
  __attribute__((aligned(16))) float scales[2][kChunk];
};

template <class E, int D, int NT, int GH, int FLIGHT, class Put>
__device__ inline void score_blocks(const SelectArgs& a, int64_t t0, int head, int first, int step,
                                    ScoreLds& lds, Put&& put) {
  using V8 = typename Kv<E>::V8;
  constexpr int KS = D / 32;  // steps of 64 of a row's 2 D bytes
  constexpr int TG = GH > 0 ? NT / GH : 1, HEADS = GH > 0 ? GH : 16 * NT;
  const int lane = lane_id(), col = lane & 15, grp = lane >> 4;
  const int passes = (a.G + HEADS - 1) / HEADS;
  constexpr int LOADS = D % 64 == 0 ? KS / 2 : KS;  // 16 channels of a query row a lane
  auto load_q = [&](int64_t t, int h, V8 (&x)[LOADS][2]) {
    const E* q = static_cast<const E*>(a.q) + t * a.q_st +
                 static_cast<int64_t>(head * a.G + (h < a.G ? h : a.G - 1)) * a.q_sh;
#pragma unroll
    for (int s = 0; s < LOADS; ++s) {
      const int at = 64 * s + 16 * grp, d = at < D ? at : at - D;
      x[s][0] = *reinterpret_cast<const V8*>(q + d);
      x[s][1] = *reinterpret_cast<const V8*>(q + d + 8);
    }
  };

  // the lane's token of each group, and where its candidates end (0: none)
  int64_t token[TG];
  int32_t seq[TG], end[TG];
  bool any = false;
#pragma unroll
  for (int g = 0; g < TG; ++g) {
    token[g] = t0 + (GH > 0 ? 16 * g + col : 0);
    end[g] = 0;
    seq[g] = -1;
    if (token[g] < a.T) {
      const KvPlace p = kv_place(a.tok, token[g]);
      const int32_t e = p.last - a.recent + 1;
      if (p.last >= 0 && e > a.sink) {
        end[g] = e;
        seq[g] = a.tok.seq_ids[token[g]];
      }
    }
    any |= end[g] > 0;
  }
  if (!__any(any)) return;

  for (int pass = 0; pass < passes; ++pass) {
    // columns: bytes [64 s + 16 grp, +16) of [c | |c|]
    v4i cf[NT][KS];
    float scale[NT];
    auto quantise = [&]() {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int g = GH > 0 ? n / GH : 0;
        V8 x[LOADS][2];
        load_q(end[g] > 0 ? token[g] : t0,
               GH > 0 ? pass * GH + n % GH : (pass * NT + n) * 16 + col, x);
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < LOADS; ++s) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            top = fmaxf(top, fabsf(static_cast<float>(x[s][e >> 3][e & 7])));
          }
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        top = fmaxf(top, kKvTopFloor);
        scale[n] = top / 127.0f;
        const float small = top > 0x1p100f ? 0x1p-64f : 1.0f;
        top *= small;
        const float r = 1.0f / top;
        // (an infinite row: by 1 and r = 0 a finite channel is 0 and an infinite one NaN, as
        // divided)
        if (r == 0.0f) top = 1.0f;
#pragma unroll
        for (int s = 0; s < LOADS; ++s) {
          v4i codes, sizes;
          pack_codes(x[s], top, r, small, codes, sizes);
          if constexpr (D % 64 == 0) {
            cf[n][s] = codes;
            cf[n][s + LOADS] = sizes;
          } else {
            const bool second = 64 * s + 16 * grp >= D;
#pragma unroll
            for (int w = 0; w < 4; ++w) cf[n][s][w] = second ? sizes[w] : codes[w];
          }
        }
      }
    };
    bool quantised = false;
    bool todo[TG];
#pragma unroll
    for (int g = 0; g < TG; ++g) todo[g] = end[g] > 0;
    for (;;) {  // the sequences among the tokens
      int32_t of = -1;
#pragma unroll
      for (int g = TG - 1; g >= 0; --g) {
        const uint64_t m = __ballot(todo[g]);
        if (m != 0) of = __builtin_amdgcn_readlane(seq[g], __builtin_ctzll(m));
      }
      if (of < 0) break;
      int32_t last = 0;
      bool mine[TG];
#pragma unroll
      for (int g = 0; g < TG; ++g) {
        mine[g] = todo[g] && seq[g] == of;
        todo[g] = todo[g] && !mine[g];
        if (mine[g] && end[g] > last) last = end[g];
      }
      last = static_cast<int32_t>(wave_extreme<true>(static_cast<uint32_t>(last)));
      const int32_t* row = a.tok.page_table + static_cast<int64_t>(of) * a.tok.max_pages;

      auto look_up = [&](int64_t chunk) {
        const int64_t b = chunk * kChunk + lane;
        if (b >= last) return -1;
        const int32_t p = row[b];
        return p >= 0 && p < a.tok.P ? p : -1;
      };
      auto scale_of = [&](int32_t page) {
        return page >= 0 ? a.scales[static_cast<int64_t>(page) * a.Hkv + head] : 0.0f;
      };
      v4i bf[FLIGHT][KS];
      auto load_tile = [&](int buf, int tile) {
        const int32_t p = lds.pages[buf][16 * tile + col];
        const int8_t* from = a.bounds +
                             (static_cast<int64_t>(p < 0 ? 0 : p) * a.Hkv + head) * (2 * D) +
                             16 * grp;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          bf[tile % FLIGHT][s] = *reinterpret_cast<const v4i*>(from + 64 * s);
        }
      };

      int64_t chunk = a.sink / kChunk + first;
      const int64_t stop = cdiv(last, kChunk);
      if (chunk >= stop) continue;
      int buf = 0;
      int32_t page = look_up(chunk), page_next = look_up(chunk + step);
      lds.pages[0][lane] = page;
      asm volatile("" ::: "memory");  // (read by other lanes of this wave)
#pragma unroll
      for (int i = 0; i < FLIGHT; ++i) load_tile(0, i);
      lds.scales[0][lane] = scale_of(page);
      if (!quantised) quantise();
      quantised = true;
      for (; chunk < stop; chunk += step, buf ^= 1) {
        const bool more = chunk + step < stop;
        float next_scale = 0.0f;
        if (more) {
          lds.pages[buf ^ 1][lane] = page_next;
          next_scale = scale_of(page_next);
          page_next = look_up(chunk + 2 * static_cast<int64_t>(step));
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v4i acc[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[n] = v4i{0, 0, 0, 0};
#pragma unroll
          for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              acc[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[i % FLIGHT][s], cf[n][s],
                                                             acc[n], 0, 0, 0);
            }
          }
          settle(acc);
          float best[TG][4];
#pragma unroll
          for (int g = 0; g < TG; ++g) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              best[g][r] = static_cast<float>(acc[g * (NT / TG)][r]) * scale[g * (NT / TG)];
#pragma unroll
              for (int n = 1; n < NT / TG; ++n) {
                best[g][r] = fmaxf(best[g][r], static_cast<float>(acc[g * (NT / TG) + n][r]) *
                                                   scale[g * (NT / TG) + n]);
              }
              if (GH == 0) best[g][r] = group_max16(best[g][r]);
            }
          }
          if (i + FLIGHT < 4) {
            load_tile(buf, i + FLIGHT);
          } else if (more) {
            load_tile(buf ^ 1, (i + FLIGHT) % 4);
          }
          const v4i pg = *reinterpret_cast<const v4i*>(&lds.pages[buf][16 * i + 4 * grp]);
          const v4f bs = *reinterpret_cast<const v4f*>(&lds.scales[buf][16 * i + 4 * grp]);
          const int64_t b = chunk * kChunk + 16 * i + 4 * grp;
#pragma unroll
          for (int g = 0; g < TG; ++g) {
            if (!mine[g] || (GH == 0 && col != 0)) continue;
            auto* to = put(token[g], b);
            if (pass > 0) {
              const v4i old = *to;
#pragma unroll
              for (int r = 0; r < 4; ++r) best[g][r] = fmaxf(best[g][r], __int_as_float(old[r]));
            }
            v4i key;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              key[r] = pass + 1 < passes ? __float_as_int(best[g][r])
                       : pg[r] < 0       ? 0
                                         : static_cast<int>(score_key(best[g][r], bs[r]));
            }
            *to = key;
          }
        }
        if (more) lds.scales[buf ^ 1][lane] = next_scale;
        asm volatile("" ::: "memory");
      }
    }
  }
}

// Waves a SIMD, by the registers that the columns take. Four heads of 128 channels are worth three
// with half the tiles in flight (prompts of 4099 tokens: 78 us scores and cut, 84 with two waves
// and four tiles); fewer channels were not measured with three and keep two, wide ones with four
// tiles fit once.
template <int D, int NT, int GH>
constexpr int kScoreOccupancy = D == 128 && GH == 4 ? 3 : D > 128 && NT == 4 ? 1 : 2;

template <class E, int D, int NT, int GH>
__global__ void __launch_bounds__(kScoreWaves* kWave, (kScoreOccupancy<D, NT, GH>))
    kv_score_kernel(SelectArgs a) {
  __shared__ ScoreLds lds[kScoreWaves];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int head = static_cast<int>(blockIdx.x % a.head_groups) * kScoreWaves + wave;
  if (head >= a.Hkv) return;
  const int split = static_cast<int>(blockIdx.x / a.head_groups % a.splits);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x / a.head_groups / a.splits) *
                     (GH > 0 ? 16 * (NT / (GH > 0 ? GH : 1)) : 1);
  // tiles of bounds in flight
  constexpr int FLIGHT = D * NT > 512 || D > 128 || kScoreOccupancy<D, NT, GH> == 3 ? 2 : 4;
  score_blocks<E, D, NT, GH, FLIGHT>(a, t0, head, split, a.splits, lds[wave],
                                     [&](int64_t token, int64_t b) {
                                       return reinterpret_cast<v4i*>(
                                           a.keys + (token * a.Hkv + head) * a.stride + b);
                                     });
}

// --- keep ---------------------------------------------------------------------------------------

// A row's blocks: `lead` forced ones, n candidates, `tail` forced ones; `want` places for
// candidates.
struct Span {
  int32_t* out;
  int32_t lead, n, end, tail;
  uint32_t want;
  __device__ Span(const SelectArgs& a, int64_t row) {
    const KvPlace p = kv_place(a.tok, row / a.Hkv);
    const int32_t blocks = p.last + 1;
    out = a.out + row * a.count;
    lead = a.sink < blocks ? a.sink : blocks;
    end = blocks - a.recent > lead ? blocks - a.recent : lead;
    n = end - lead;
    tail = blocks - end;
    want = static_cast<uint32_t>(a.want);
  }
  // The forced blocks around `kept` candidates, and -1 behind them.
  __device__ void rest(const SelectArgs& a, uint32_t kept, int thread, int threads) const {
    for (int32_t i = thread; i < lead; i += threads) out[i] = i;
    const int32_t from = lead + static_cast<int32_t>(kept);
    for (int32_t i = thread; from + i < a.count; i += threads) {
      out[from + i] = i < tail ? end + i : -1;
    }
  }
};

// A row's candidates as a workgroup of WAVES waves holds them: even shares of neighbours, up to R
// keys a lane. R = 0: any number, read again where they are needed.
template <int WAVES, int R>
struct Row {
  uint32_t k[R > 0 ? R : 1];
  const uint32_t* keys;
  int32_t first, n;  // this wave's first candidate (from the row's first) and how many
  __device__ void load(const uint32_t* row, int32_t candidates, int wave) {
    const int32_t each = (candidates + 64 * WAVES - 1) / (64 * WAVES) * 64;  // at most 64 R
    first = wave * each;
    n = candidates - first < each ? candidates - first : each;
    keys = row + first;
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int32_t at = 64 * i + lane_id();
        k[i] = at < n ? keys[at] : 0u;
      }
    }
  }
  template <class F>
  __device__ void each(F&& f) const {  // f(key, candidate in the row), 64 neighbours at a time
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (64 * i < n) f(k[i], first + 64 * i + lane_id());
      }
    } else {
      for (int32_t i = 0; i < n; i += 64) {
        f(i + lane_id() < n ? keys[i + lane_id()] : 0u, first + i + lane_id());
      }
    }
  }
};

// The largest cut that at least `want` of a wave's keys reach (1 where fewer are above 0), and how
// many do. `count(probe)`: how many reach a key, the same in every lane.
template <class F>
__device__ inline uint32_t bisect(uint32_t most, uint32_t least, uint32_t total, uint32_t want,
                                  F&& count, uint32_t& reach) {
  reach = total;
  if (total <= want) return 1u;
  const uint32_t differ = most ^ least;
  if (differ == 0) return most;
  int bit = 31 - __builtin_clz(differ);
  uint32_t cut = most & ~((2u << bit) - 1u);
  for (; bit >= 0 && reach != want; --bit) {
    const uint32_t probe = cut | (1u << bit);
    const uint32_t n = count(probe);
    if (n >= want) {
      cut = probe;
      reach = n;
    }
  }
  return cut;
}

// The kept of up to N keys a lane, in order (index(i): the candidate of key i): how many.
template <int N, class F>
__device__ inline uint32_t keep_in_order(const Span& p, const uint32_t (&k)[N], int32_t n,
                                         F&& index) {
  const int lane = lane_id();
  const uint64_t below = (uint64_t{1} << lane) - 1;
  uint32_t most = 0u, least = ~0u, total = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (64 * i < n) {
      total += static_cast<uint32_t>(__popcll(__ballot(k[i] != 0)));
      most = k[i] > most ? k[i] : most;
      least = k[i] != 0 && k[i] < least ? k[i] : least;
    }
  }
  uint32_t reach;
  const uint32_t cut = bisect(
      wave_extreme<true>(most), wave_extreme<false>(least), total, p.want,
      [&](uint32_t probe) {
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (64 * i < n) c += static_cast<uint32_t>(__popcll(__ballot(k[i] >= probe)));
        }
        return c;
      },
      reach);
  // more keys than places reach the cut: the lowest blocks of the cut's own key
  uint32_t ties = ~0u;
  if (reach > p.want) {
    ties = p.want;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (64 * i < n) ties -= static_cast<uint32_t>(__popcll(__ballot(k[i] > cut)));
    }
  }
  uint32_t kept = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (64 * i >= n) continue;
    const uint64_t same = __ballot(k[i] == cut);
    const bool keep =
        k[i] > cut || (k[i] == cut && static_cast<uint32_t>(__popcll(same & below)) < ties);
    const uint64_t m = __ballot(keep);
    if (keep) p.out[p.lead + kept + __popcll(m & below)] = p.lead + index(i);
    kept += static_cast<uint32_t>(__popcll(m));
    const uint32_t seen = static_cast<uint32_t>(__popcll(same));
    ties = ties > seen ? ties - seen : 0;
  }
  return kept;
}

// A wave a row, R keys a lane. Where few are wanted of many: the want-th largest of the lanes'
// largest keys bounds the cut; the keys that reach it, one a lane if they are 64 or fewer, hold the
// kept.
template <int R>
__device__ inline void keep_few(const SelectArgs& a, const Span& p, const uint32_t* keys,
                                uint32_t* near, int32_t* near_at) {
  const int lane = lane_id();
  uint32_t k[R];
#pragma unroll
  for (int i = 0; i < R; ++i) k[i] = 64 * i + lane < p.n ? keys[64 * i + lane] : 0u;
  uint32_t kept = 0;
  bool done = p.want == 0;
  if (R > 1 && !done && p.n > 2 * kWave && p.want <= 40) {
    uint32_t top = k[0], reach;
#pragma unroll
    for (int i = 1; i < R; ++i) top = k[i] > top ? k[i] : top;
    const uint32_t floor = bisect(
        wave_extreme<true>(top), wave_extreme<false>(top != 0 ? top : ~0u),
        static_cast<uint32_t>(__popcll(__ballot(top != 0))), p.want,
        [&](uint32_t probe) { return static_cast<uint32_t>(__popcll(__ballot(top >= probe))); },
        reach);
    int n = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (64 * i < p.n) {
        const uint64_t m = __ballot(k[i] >= floor);
        const int at = n + __popcll(m & ((uint64_t{1} << lane) - 1));
        if (k[i] >= floor && at < kWave) {
          near[at] = k[i];
          near_at[at] = 64 * i + lane;
        }
        n += __popcll(m);
      }
    }
    asm volatile("" ::: "memory");  // (read by other lanes of this wave)
    if (n <= kWave) {
      const uint32_t one[1] = {lane < n ? near[lane] : 0u};
      const int32_t at = lane < n ? near_at[lane] : 0;
      kept = keep_in_order(p, one, kWave, [&](int) { return at; });
      done = true;
    }
  }
  if (!done) kept = keep_in_order(p, k, p.n, [&](int i) { return 64 * i + lane; });
  p.rest(a, kept, lane, kWave);
}

template <int R>
__global__ void __launch_bounds__(4 * kWave) kv_keep_few_kernel(SelectArgs a) {
  __shared__ uint32_t near[4][kWave];
  __shared__ int32_t near_at[4][kWave];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  if (row >= a.T * a.Hkv) return;
  const Span p(a, row);
  if (p.n > R * kWave) return;  // (kv_keep_many_kernel's)
  keep_few<R>(a, p, a.keys + row * a.stride + p.lead, near[wave], near_at[wave]);
}

// A workgroup of WAVES waves a row, R keys a lane (0: read again where they are needed).
constexpr int kRankMost = 2048;  // keys that are ranked against each other

template <int WAVES>
struct KeepLds {
  __attribute__((aligned(16))) uint32_t tops[WAVES * kWave];
  uint64_t near[kRankMost];  // key << 32 | ~candidate: the order of (key desc, block asc)
  int32_t winners[1024];
  uint32_t cut, listed, sums[WAVES];
};

template <int WAVES, int R>
__device__ inline void keep_many(const SelectArgs& a, const Span& p, const uint32_t* keys,
                                 KeepLds<WAVES>& lds) {
  constexpr int LANES = WAVES * kWave;
  auto& tops = lds.tops;
  auto& near = lds.near;
  auto& winners = lds.winners;
  auto& sums = lds.sums;
  auto& listed = lds.listed;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = lane_id();
  Row<WAVES, R> r;
  r.load(keys, p.n, wave);
  uint32_t top = 0u;
  r.each([&](uint32_t k, int32_t) { top = k > top ? k : top; });
  tops[threadIdx.x] = top;
  if (threadIdx.x == 0) listed = 0u;
  __syncthreads();
  if (wave == 0) {
    // Groups of lanes, some more than places: the want-th largest of their largest keys.
    auto cut_of = [&](auto groups, auto load) {
      constexpr int N = decltype(groups)::value;
      uint32_t g[N], most = 0u, least = ~0u, total = 0u, reach;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        g[i] = load(i);
        total += static_cast<uint32_t>(__popcll(__ballot(g[i] != 0)));
        most = g[i] > most ? g[i] : most;
        least = g[i] != 0 && g[i] < least ? g[i] : least;
      }
      return bisect(
          wave_extreme<true>(most), wave_extreme<false>(least), total, p.want,
          [&](uint32_t probe) {
            uint32_t n = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
              n += static_cast<uint32_t>(__popcll(__ballot(g[i] >= probe)));
            }
            return n;
          },
          reach);
    };
    uint32_t cut = ~0u;
    if (p.want == 0) {
    } else if (WAVES == 16 && p.want <= 96) {
      cut = cut_of(std::integral_constant<int, WAVES / 4>{}, [&](int i) {
        const v4i x = *reinterpret_cast<const v4i*>(&tops[4 * (64 * i + lane)]);
        const uint32_t u = static_cast<uint32_t>(x[0]), v = static_cast<uint32_t>(x[1]);
        const uint32_t y = static_cast<uint32_t>(x[2]), z = static_cast<uint32_t>(x[3]);
        const uint32_t f = u > v ? u : v, t = y > z ? y : z;
        return f > t ? f : t;
      });
    } else {
      cut = cut_of(std::integral_constant<int, WAVES>{},
                   [&](int i) { return tops[64 * i + lane]; });
    }
    if (lane == 0) lds.cut = cut;
  }
  __syncthreads();
  const uint32_t floor = lds.cut;
  if (p.want > 0) {
    r.each([&](uint32_t k, int32_t at) {
      const uint64_t m = __ballot(k >= floor);
      if (m == 0) return;
      uint32_t first = 0;
      if (lane == 0) first = atomicAdd(&listed, static_cast<uint32_t>(__popcll(m)));
      first = __builtin_amdgcn_readfirstlane(first) + __popcll(m & ((uint64_t{1} << lane) - 1));
      if (k >= floor && first < kRankMost) {
        near[first] = static_cast<uint64_t>(k) << 32 | (0xffffffffu - static_cast<uint32_t>(at));
      }
    });
  }
  __syncthreads();
  const uint32_t n = listed;
  uint32_t kept = n < p.want ? n : p.want;
  if (n <= kRankMost) {
    for (uint32_t i = threadIdx.x; i < n; i += LANES) {
      const uint64_t x = near[i];
      uint32_t rank = 0;
#pragma unroll 8
      for (uint32_t j = 0; j < n; ++j) rank += near[j] > x ? 1u : 0u;
      if (rank < p.want) {
        winners[rank] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(x));
      }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kept; i += LANES) {
      const int32_t x = winners[i];
      int32_t at = 0;
#pragma unroll 8
      for (uint32_t j = 0; j < kept; ++j) at += winners[j] < x ? 1 : 0;
      p.out[p.lead + at] = p.lead + x;
    }
  } else {
    // (keys that mostly tie) the cut over all of them, then the kept in order, ties from the lowest
    auto count = [&](auto pred) {
      uint32_t c = 0;
      r.each([&](uint32_t k, int32_t) { c += static_cast<uint32_t>(__popcll(__ballot(pred(k)))); });
      __syncthreads();
      if (lane == 0) sums[wave] = c;
      __syncthreads();
      c = 0;
      for (int w = 0; w < WAVES; ++w) c += sums[w];
      return c;
    };
    uint32_t cut = 0u;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t probe = cut | (1u << bit);
      if (count([&](uint32_t k) { return k >= probe; }) >= p.want) cut = probe;
    }
    const uint32_t above = count([&](uint32_t k) { return k > cut; });
    uint32_t mine_above = 0, mine_same = 0;
    r.each([&](uint32_t k, int32_t) {
      mine_above += static_cast<uint32_t>(__popcll(__ballot(k > cut)));
      mine_same += static_cast<uint32_t>(__popcll(__ballot(k == cut)));
    });
    __syncthreads();
    if (lane == 0) {
      tops[wave] = mine_above;
      tops[WAVES + wave] = mine_same;
    }
    __syncthreads();
    uint32_t ties = p.want - above, place = 0, same_before = 0;
    for (int w = 0; w < wave; ++w) {
      const uint32_t left = ties > same_before ? ties - same_before : 0;
      place += tops[w] + (tops[WAVES + w] < left ? tops[WAVES + w] : left);
      same_before += tops[WAVES + w];
    }
    ties = ties > same_before ? ties - same_before : 0;
    const uint64_t below = (uint64_t{1} << lane) - 1;
    r.each([&](uint32_t k, int32_t at) {
      const uint64_t same = __ballot(k == cut);
      const bool keep =
          k > cut || (k == cut && static_cast<uint32_t>(__popcll(same & below)) < ties);
      const uint64_t m = __ballot(keep);
      if (keep) p.out[p.lead + place + __popcll(m & below)] = p.lead + at;
      place += static_cast<uint32_t>(__popcll(m));
      const uint32_t seen = static_cast<uint32_t>(__popcll(same));
      ties = ties > seen ? ties - seen : 0;
    });
  }
  p.rest(a, kept, static_cast<int>(threadIdx.x), LANES);
}

template <int WAVES, int R>
__global__ void __launch_bounds__(WAVES* kWave) kv_keep_many_kernel(SelectArgs a) {
  __shared__ KeepLds<WAVES> lds;
  const int64_t row = blockIdx.x;
  const Span p(a, row);
  if (p.n <= a.above) return;
  keep_many<WAVES, R>(a, p, a.keys + row * a.stride + p.lead, lds);
}

// Both in one launch, a workgroup a (token, key/value head): decode over page tables of up to
// kFusedMost blocks. The keys stay in LDS. Workgroups go to the eight XCDs in turn: each takes rows
// side by side, as the heads of a token share lines of the page table and of the scales (64
// sequences, 8 heads: 57 us with the heads spread, 53 with this step, 51 now).
constexpr int kFusedWaves = 8;
constexpr int kFusedMost = 4096;

template <class E, int D, int NT>
__global__ void __launch_bounds__(kFusedWaves* kWave, D <= 128 && NT == 1 ? 4 : 2)
    kv_select_kernel(SelectArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t keys[kFusedMost];
  __shared__ ScoreLds score_lds[kFusedWaves];
  __shared__ KeepLds<kFusedWaves> keep_lds;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const unsigned share = gridDim.x / 8;
  const int64_t row = static_cast<int64_t>(blockIdx.x % 8) * share + blockIdx.x / 8;
  if (row >= a.T * a.Hkv) return;
  if (a.want > 0) {
    score_blocks<E, D, NT, 0, 2>(
        a, row / a.Hkv, static_cast<int>(row % a.Hkv), wave, kFusedWaves, score_lds[wave],
        [&](int64_t, int64_t b) { return reinterpret_cast<v4i*>(&keys[b]); });
  }
  __syncthreads();
  const Span p(a, row);
  if (p.n <= 8 * kWave) {
    if (wave == 0) keep_few<8>(a, p, keys + p.lead, keep_lds.tops, keep_lds.winners);
  } else {
    keep_many<kFusedWaves, kFusedMost / (kFusedWaves * kWave)>(a, p, keys + p.lead, keep_lds);
  }
}

// Whether tokens mostly share their sequences (`seqs` of them at most) and there are rows and keys
// enough (their scores are then taken several tokens a wave), and whether a call is one launch: few
// enough places for 512 lanes to bound well, and two chunks a wave or rows enough to fill the GPU
// (one row of 1258 blocks: 13 us in two launches, 16 in one). Rows for little more than a workgroup
// a CU take less as single tokens do (32 tokens of 8 heads of 128 over 470 blocks: 15 us for 21,
// 128 tokens 32 for 22; 4 heads of 256: 64 tokens 19 for 41; 6 of 256 over 403: 93 tokens 36 for
// 26; over 2032 blocks, two launches where rows are few, 8 tokens of 4 heads of 256 18 for 36, 16
// of 8 heads of 128 27 for 19).
inline bool select_prompt(int64_t T, int64_t Hkv, int64_t seqs, int64_t max_pages) {
  if (seqs <= 0 || T < 4 * seqs) return false;
  if (T > 320 / Hkv) return true;
  return max_pages > 2 * kFusedWaves * kChunk && T * Hkv * max_pages > 1 << 17;
}
inline bool select_fused(int64_t T, int64_t Hkv, int64_t seqs, int64_t max_pages, int64_t want) {
  return !select_prompt(T, Hkv, seqs, max_pages) && want <= 256 &&
         max_pages <= (T * Hkv >= 128 ? kFusedMost : 2 * kFusedWaves * kChunk);
}

constexpr int64_t kKeepRows = 2048;  // rows whose short ones are cut in a launch of their own

// gh = 0: a token a wave, its heads across `tiles` tiles. gh > 0: tokens across the lanes, gh heads
// a pass.
struct SelectPlan {
  int64_t stride;
  int32_t tiles, gh, per_wave, splits, head_groups;
};

inline SelectPlan select_plan(bool prompt, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                              int64_t max_pages, int64_t sink) {
  SelectPlan p;
  const int64_t G = Hq / Hkv;
  p.stride = align_up(static_cast<size_t>(max_pages), kChunk);
  p.head_groups = static_cast<int32_t>(cdiv(Hkv, kScoreWaves));
  // (a wave with tokens of several sequences passes over each one's blocks)
  if (prompt) {
    // heads whose columns fit in registers beside the bounds
    const int64_t most = D <= 128 ? 8 : 4;
    const int64_t gh = next_pow2(G);
    p.gh = static_cast<int32_t>(gh < most ? gh : most);
    p.tiles = p.gh < 4 ? 4 : p.gh;
    p.per_wave = 16 * p.tiles / p.gh;
  } else {
    p.gh = 0;
    p.tiles = G <= 16 ? 1 : G <= 32 || D > 128 ? 2 : 4;
    p.per_wave = 1;
  }
  const int64_t waves = cdiv(T, p.per_wave) * Hkv;
  const int64_t chunks = cdiv(max_pages > sink ? max_pages - sink : 1, kChunk);
  const int64_t want = cdiv(4096, waves > 0 ? waves : 1);
  p.splits = static_cast<int32_t>(want < chunks ? want : chunks);
  return p;
}

// In two launches a call's tokens are taken in slabs whose keys fit in kSlabBytes (of 64s of
// tokens, whole waves of either form, where that many fit), one after the other over the same
// workspace, so it grows neither with a prompt's length nor, but for a token's own rows, with the
// page table. A slab has to fill the GPU: 4099 tokens of 8 heads behind 313 blocks of a table of
// 16384 columns take 602 us in slabs of 128 MiB, 403 of 256, 269 of 512 and 168 in one of 2.1 GiB;
// 8192 tokens in a table of 2048 columns 303, 232, and 202 in the one of 512.
constexpr int64_t kSlabBytes = int64_t{512} << 20;
inline int64_t select_slab(int64_t T, int64_t Hkv, int64_t max_pages) {
  const size_t row = align_up(static_cast<size_t>(max_pages > 0 ? max_pages : 1), kChunk);
  int64_t n = kSlabBytes / static_cast<int64_t>(Hkv * row * sizeof(uint32_t));
  if (n >= 64) n &= ~int64_t{63};
  if (n < 1) n = 1;
  return n < T ? n : T;
}

// The launches of a slab: scores, then the cut.
inline int select_slab_blocks(SelectArgs a, const SelectPlan& plan, int dtype, int64_t D,
                              int64_t max_pages, hipStream_t s) {
  const int64_t grid = cdiv(a.T, plan.per_wave) * plan.splits * plan.head_groups;
  RT_CHECK_ARG(grid <= INT32_MAX, "too many tokens");
  if (max_pages > a.sink && a.want > 0) {  // else no block is chosen by its score
    const int st = kv_dispatch(dtype, D, [&](auto e, auto d) -> int {
      using E = decltype(e);
      constexpr int DD = decltype(d)::value;
      const dim3 g(static_cast<unsigned>(grid)), b(kScoreWaves * kWave);
      constexpr int W = DD <= 128 ? 4 : 2;  // the widest decode form
      if (plan.gh == 0) {
        if (plan.tiles == 1) {
          kv_score_kernel<E, DD, 1, 0><<<g, b, 0, s>>>(a);
        } else if (plan.tiles == 2) {
          kv_score_kernel<E, DD, 2, 0><<<g, b, 0, s>>>(a);
        } else {
          kv_score_kernel<E, DD, W, 0><<<g, b, 0, s>>>(a);
        }
      } else if (plan.gh == 1) {
        kv_score_kernel<E, DD, 4, 1><<<g, b, 0, s>>>(a);
      } else if (plan.gh == 2) {
        kv_score_kernel<E, DD, 4, 2><<<g, b, 0, s>>>(a);
      } else if (plan.gh == 4) {
        kv_score_kernel<E, DD, 4, 4><<<g, b, 0, s>>>(a);
      } else if constexpr (DD <= 128) {
        kv_score_kernel<E, DD, 8, 8><<<g, b, 0, s>>>(a);
      }
      RT_CHECK_HIP(hipGetLastError());
      return kOk;
    });
    if (st != kOk) return st;
  }
  // A wave a row while its keys fit in 16 registers a lane; then four waves, unless more places are
  // wanted than their lanes bound well; then sixteen. Of many rows each is cut by its own number of
  // candidates, not by the table's width: the short ones a wave a row in a launch before (4099
  // tokens of 8 heads behind 313 blocks of a table of 16384 columns: 168 for 616 us). With fewer
  // rows that launch costs what it saves (1024 rows behind 313 blocks of 2048 columns: 28 us for
  // 23.5).
  const int64_t rows = a.T * a.Hkv;
  const dim3 one(static_cast<unsigned>(rows)), four(static_cast<unsigned>(cdiv(rows, 4)));
  const bool few = max_pages <= 64 * 16;
  a.above = -1;
  if (max_pages <= 64 * 4) {
    kv_keep_few_kernel<4><<<four, 4 * kWave, 0, s>>>(a);
  } else if (few || rows >= kKeepRows) {
    kv_keep_few_kernel<16><<<four, 4 * kWave, 0, s>>>(a);
    a.above = 64 * 16;
  }
  if (few) {
  } else if (max_pages <= 4 * 64 * 16 && a.count - a.sink - a.recent <= 128) {
    kv_keep_many_kernel<4, 16><<<one, 4 * kWave, 0, s>>>(a);
  } else if (max_pages <= 16 * 64 * 16) {
    kv_keep_many_kernel<16, 16><<<one, 16 * kWave, 0, s>>>(a);
  } else {
    kv_keep_many_kernel<16, 0><<<one, 16 * kWave, 0, s>>>(a);
  }
  RT_CHECK_HIP(hipGetLastError());
  return kOk;
}

}  // namespace rt

using namespace rt;

extern "C" size_t rt_kv_select_workspace(int64_t T, int64_t Hkv, int64_t sequences,
                                         int64_t max_pages, int64_t count, int64_t sink,
                                         int64_t recent) {
  if (T < 1 || Hkv < 1 || max_pages < 1) return 0;
  if (select_fused(T, Hkv, sequences, max_pages, count - sink - recent)) return 0;
  return static_cast<size_t>(select_slab(T, Hkv, max_pages)) * Hkv *
         align_up(static_cast<size_t>(max_pages), kChunk) * sizeof(uint32_t);
}

extern "C" int rt_kv_select(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t T,
                            int64_t Hq, int64_t Hkv, int64_t D, int dtype, const int8_t* bounds,
                            const float* bound_scales, int64_t P, int64_t page,
                            const int32_t* positions, const int32_t* seq_ids,
                            const int32_t* page_table, int64_t B, int64_t max_pages, int64_t count,
                            int64_t sink, int64_t recent, int32_t* out, void* workspace,
                            size_t workspace_bytes, rt_stream_t stream) {
  return rt_kv_select_of(q, q_token_stride, q_head_stride, T, Hq, Hkv, D, dtype, bounds,
                         bound_scales, P, page, positions, seq_ids, page_table, B, max_pages, count,
                         sink, recent, B, out, workspace, workspace_bytes, stream);
}

extern "C" int rt_kv_select_of(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                               int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int dtype,
                               const int8_t* bounds, const float* bound_scales, int64_t P,
                               int64_t page, const int32_t* positions, const int32_t* seq_ids,
                               const int32_t* page_table, int64_t B, int64_t max_pages,
                               int64_t count, int64_t sink, int64_t recent, int64_t sequences,
                               int32_t* out, void* workspace, size_t workspace_bytes,
                               rt_stream_t stream) {
  if (const int st = kv_check(T, Hq, Hkv, D, dtype, B, max_pages, P, page)) return st;
  RT_CHECK_ARG(count >= 1 && count <= 1024, "count must be in [1, 1024], got %lld",
               static_cast<long long>(count));
  RT_CHECK_ARG(sink >= 0 && recent >= 1 && sink + recent <= count,
               "sink >= 0 and recent >= 1 must fit in count");
  if (T == 0) return kOk;
  RT_CHECK_ARG(q && positions && seq_ids && out, "null pointer");
  RT_CHECK_ARG(B * max_pages == 0 || page_table, "null page table");
  RT_CHECK_ARG(P == 0 || (bounds && bound_scales), "null bounds");
  RT_CHECK_ARG(kv_rows_aligned(q, q_token_stride, q_head_stride) && kv_rows_aligned(bounds, 0, 0),
               "rows must start on 16 bytes");
  RT_CHECK_ARG(T * Hkv <= INT32_MAX - 8, "too many tokens");
  RT_CHECK_ARG(sequences >= 0, "sequences must not be negative, got %lld",
               static_cast<long long>(sequences));
  const size_t need = rt_kv_select_workspace(T, Hkv, sequences, max_pages, count, sink, recent);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) {
    set_error("workspace too small: %zu < %zu", workspace_bytes, need);
    return kWorkspaceTooSmall;
  }
  SelectArgs a{};
  a.q = q, a.q_st = q_token_stride, a.q_sh = q_head_stride, a.T = T;
  a.Hq = static_cast<int32_t>(Hq), a.Hkv = static_cast<int32_t>(Hkv), a.G = a.Hq / a.Hkv;
  a.bounds = bounds, a.scales = bound_scales;
  a.tok = {positions, seq_ids, page_table, static_cast<int32_t>(B),
           static_cast<int32_t>(max_pages), static_cast<int32_t>(P), kv_shift(page)};
  a.count = static_cast<int32_t>(count), a.sink = static_cast<int32_t>(sink);
  a.recent = static_cast<int32_t>(recent), a.out = out, a.keys = static_cast<uint32_t*>(workspace);
  // (blocks without a page read page 0's bounds, so there has to be one)
  a.want = P > 0 ? static_cast<int32_t>(count - sink - recent) : 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (select_fused(T, Hkv, sequences, max_pages, count - sink - recent)) {
    return kv_dispatch(dtype, D, [&](auto e, auto d) -> int {
      using E = decltype(e);
      constexpr int DD = decltype(d)::value;
      const dim3 g(static_cast<unsigned>(cdiv(T * Hkv, 8) * 8)), b(kFusedWaves * kWave);
      if (a.G <= 16) {
        kv_select_kernel<E, DD, 1><<<g, b, 0, s>>>(a);
      } else {
        kv_select_kernel<E, DD, 2><<<g, b, 0, s>>>(a);
      }
      RT_CHECK_HIP(hipGetLastError());
      return kOk;
    });
  }
  const bool prompt = select_prompt(T, Hkv, sequences, max_pages);
  const int64_t slab = select_slab(T, Hkv, max_pages);
  for (int64_t t0 = 0; t0 < T; t0 += slab) {
    SelectArgs part = a;
    part.T = T - t0 < slab ? T - t0 : slab;
    part.q = static_cast<const uint16_t*>(q) + t0 * q_token_stride;  // (16 bits an element)
    part.tok.positions += t0, part.tok.seq_ids += t0;
    part.out += t0 * Hkv * count;
    const SelectPlan plan = select_plan(prompt, part.T, Hq, Hkv, D, max_pages, sink);
    part.stride = plan.stride, part.splits = plan.splits, part.head_groups = plan.head_groups;
    if (const int st = select_slab_blocks(part, plan, dtype, D, max_pages, s)) return st;
  }
  return kOk;
}
