// The best blocks of each token and key/value head, by the int8 bounds' score.
//
// A query head's row is quantised as the bounds are (codes c, scale s); block b's score with it is
// (c . mid_b + |c| . half_b) s times the block's scale, an upper bound on what any of its keys can
// score, and the group's score is the largest of its heads'. The sum is an int32 (at most
// 2 * 256 * 127^2 < 2^23, so exact as fp32 too); the two products are rounded once each, in this
// order, and rounding is monotone, so the largest over the heads is taken before the block's scale.
//
// Two launches. Scores: [blocks x columns] = bounds [c | |c|]^T on the int8 matrix cores, 16 blocks
// by 16 columns an instruction, a column being one query head of one token; the columns stay in
// registers (quantised there by the wave that needs them), the bounds come from memory in the
// operand's layout with a chunk of 64 blocks in flight; the largest of a token's neighbouring
// columns by lane exchange, then one key a (token, head, block). Keep: the cut by bisection over the
// keys' bits, from the highest bit in which they differ until the count is exact, then the kept
// blocks in order.
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
  int32_t* out;       // [T, Hkv, count]
  uint32_t* keys;     // [T * Hkv, stride]
  int64_t stride;
  int32_t cols;       // columns of a token in a tile of 16: a power of two
  int32_t per_wave;   // tokens a wave holds
  int32_t splits;     // waves that share a token tile's blocks
  int32_t head_groups;
};

// The key of a candidate's score (0: not a candidate). A score that is not a number is the least.
__device__ inline uint32_t score_key(float s) {
  return key_of_f32(s == s ? s : -INFINITY);
}

// The largest over aligned groups of `n` lanes (a power of two up to 16), in every lane.
__device__ inline float group_max(float x, int n) {
  auto step = [&](auto ctrl) {
    const int y = __builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf,
                                              true);
    x = fmaxf(x, __int_as_float(y));
  };
  if (n > 1) step(std::integral_constant<int, 0xB1>{});   // lane ^ 1
  if (n > 2) step(std::integral_constant<int, 0x4E>{});   // lane ^ 2
  if (n > 4) step(std::integral_constant<int, 0x141>{});  // the other four of eight
  if (n > 8) step(std::integral_constant<int, 0x140>{});  // the other eight of sixteen
  return x;
}

// A wave holds NT tiles of 16 columns: `per_wave` tokens of `cols` columns each (heads past the
// group's repeat its last), or one token of 16 NT heads, its further heads in later passes. The
// tokens of one sequence share a pass over its blocks.
template <class E, int D, int NT>
__global__ void __launch_bounds__(kScoreWaves* kWave, D == 256 && NT == 2 ? 1 : 2)
    kv_score_kernel(SelectArgs a) {
  using V8 = typename Kv<E>::V8;
  constexpr int KS = D / 32;  // steps of 64 of a row's 2 D bytes
  __shared__ __attribute__((aligned(16))) int32_t pages[kScoreWaves][2][kChunk];
  __shared__ __attribute__((aligned(16))) float block_scales[kScoreWaves][2][kChunk];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = lane_id(), col = lane & 15, grp = lane >> 4;
  const int head = static_cast<int>(blockIdx.x % a.head_groups) * kScoreWaves + wave;
  if (head >= a.Hkv) return;
  const int split = static_cast<int>(blockIdx.x / a.head_groups % a.splits);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x / a.head_groups / a.splits) * a.per_wave;
  const bool wide = a.G > 16;
  const int passes = wide ? (a.G + 16 * NT - 1) / (16 * NT) : 1;

  // the lane's token in each tile, and where its candidates end (0: none)
  int64_t token[NT];
  int32_t seq[NT], end[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int i = wide ? 0 : (n * 16 + col) / a.cols;
    token[n] = t0 + i;
    end[n] = 0;
    seq[n] = -1;
    if (i < a.per_wave && token[n] < a.T) {
      const KvPlace p = kv_place(a.tok, token[n]);
      const int32_t e = p.last - a.recent + 1;
      if (p.last >= 0 && e > a.sink) {
        end[n] = e;
        seq[n] = a.tok.seq_ids[token[n]];
      }
    }
  }
  bool any = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) any |= end[n] > 0;
  if (!__any(any)) return;

  for (int pass = 0; pass < passes; ++pass) {
    // columns: bytes [64 s + 16 grp, +16) of [c | |c|]
    v4i cf[NT][KS];
    float scale[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      int g = wide ? (pass * NT + n) * 16 + col : col & (a.cols - 1);
      if (g >= a.G) g = a.G - 1;
      const int64_t t = end[n] > 0 ? token[n] : t0;
      const E* q = static_cast<const E*>(a.q) + t * a.q_st +
                   static_cast<int64_t>(head * a.G + g) * a.q_sh;
      constexpr int LOADS = D % 64 == 0 ? KS / 2 : KS;
      V8 x[LOADS][2];
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < LOADS; ++s) {
        const int at = 64 * s + 16 * grp, d = at < D ? at : at - D;
        x[s][0] = *reinterpret_cast<const V8*>(q + d);
        x[s][1] = *reinterpret_cast<const V8*>(q + d + 8);
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(static_cast<float>(x[s][e >> 3][e & 7])));
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      top = fmaxf(top, kKvTopFloor);
      scale[n] = top / 127.0f;
#pragma unroll
      for (int s = 0; s < LOADS; ++s) {
        const bool size = 64 * s + 16 * grp >= D;
        v4i codes, sizes;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t c4 = 0, s4 = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 4 * w + e;
            const int c = kv_code(static_cast<float>(x[s][i >> 3][i & 7]), top);
            c4 |= static_cast<uint32_t>(c & 255) << (8 * e);
            s4 |= static_cast<uint32_t>(c < 0 ? -c : c) << (8 * e);
          }
          codes[w] = static_cast<int>(c4);
          sizes[w] = static_cast<int>(s4);
        }
        if constexpr (D % 64 == 0) {
          cf[n][s] = codes;
          cf[n][s + LOADS] = sizes;
        } else {
          cf[n][s] = size ? sizes : codes;
        }
      }
    }

    bool todo[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) todo[n] = end[n] > 0;
    for (;;) {  // the sequences among the tokens
      int32_t of = -1;
#pragma unroll
      for (int n = NT - 1; n >= 0; --n) {
        const uint64_t m = __ballot(todo[n]);
        if (m != 0) {
          const int l = __builtin_ctzll(m);
          of = __builtin_amdgcn_readlane(seq[n], l);
        }
      }
      if (of < 0) break;
      int32_t last = 0;
      bool mine[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mine[n] = todo[n] && seq[n] == of;
        todo[n] = todo[n] && !mine[n];
        if (mine[n] && end[n] > last) last = end[n];
      }
      for (int i = 1; i < kWave; i <<= 1) {
        const int32_t o = __shfl_xor(last, i);
        last = o > last ? o : last;
      }
      last = __builtin_amdgcn_readfirstlane(last);
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
      v4i bf[4][KS];
      auto load_tile = [&](int buf, int tile) {
        const int32_t p = pages[wave][buf][16 * tile + col];
        const int8_t* from = a.bounds +
                             (static_cast<int64_t>(p < 0 ? 0 : p) * a.Hkv + head) * (2 * D) +
                             16 * grp;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          bf[tile][s] = p < 0 ? v4i{0, 0, 0, 0} : *reinterpret_cast<const v4i*>(from + 64 * s);
        }
      };

      int64_t chunk = a.sink / kChunk + split;
      const int64_t stop = cdiv(last, kChunk);
      if (chunk >= stop) continue;
      int buf = 0;
      int32_t page = look_up(chunk), page_next = look_up(chunk + a.splits);
      pages[wave][0][lane] = page;
      block_scales[wave][0][lane] = scale_of(page);
      asm volatile("" ::: "memory");  // (read by other lanes of this wave)
#pragma unroll
      for (int i = 0; i < 4; ++i) load_tile(0, i);
      for (; chunk < stop; chunk += a.splits, buf ^= 1) {
        const bool more = chunk + a.splits < stop;
        float next_scale = 0.0f;
        if (more) {
          pages[wave][buf ^ 1][lane] = page_next;
          next_scale = scale_of(page_next);
          page_next = look_up(chunk + 2 * static_cast<int64_t>(a.splits));
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v4i acc[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[n] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              acc[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[i][s], cf[n][s], acc[n], 0, 0, 0);
            }
          }
          if (more) load_tile(buf ^ 1, i);
          const v4i pg = *reinterpret_cast<const v4i*>(&pages[wave][buf][16 * i + 4 * grp]);
          const v4f bs = *reinterpret_cast<const v4f*>(&block_scales[wave][buf][16 * i + 4 * grp]);
          const int64_t b = chunk * kChunk + 16 * i + 4 * grp;
          float best[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) best[n][r] = static_cast<float>(acc[n][r]) * scale[n];
          }
          if (wide) {
#pragma unroll
            for (int n = 1; n < NT; ++n) {
#pragma unroll
              for (int r = 0; r < 4; ++r) best[0][r] = fmaxf(best[0][r], best[n][r]);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (wide && n > 0) break;
#pragma unroll
            for (int r = 0; r < 4; ++r) best[n][r] = group_max(best[n][r], wide ? 16 : a.cols);
            if (!mine[n] || (wide ? col != 0 : (col & (a.cols - 1)) != 0)) continue;
            v4i* to = reinterpret_cast<v4i*>(a.keys + (token[n] * a.Hkv + head) * a.stride + b);
            if (pass > 0) {
              const v4i old = *to;
#pragma unroll
              for (int r = 0; r < 4; ++r) best[n][r] = fmaxf(best[n][r], __int_as_float(old[r]));
            }
            v4i key;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              key[r] = pass + 1 < passes ? __float_as_int(best[n][r])
                       : pg[r] < 0       ? 0
                                         : static_cast<int>(score_key(best[n][r] * bs[r]));
            }
            *to = key;
          }
        }
        if (more) block_scales[wave][buf ^ 1][lane] = next_scale;
        asm volatile("" ::: "memory");
      }
    }
  }
}

// --- keep ---------------------------------------------------------------------------------------

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

// Candidates of a row as a wave or a workgroup of WAVES waves holds them: R keys a lane, in block
// order (a wave has 64 R neighbours). R = 0: any number, read again where they are needed.
template <int WAVES, int R>
struct Row {
  uint32_t k[R > 0 ? R : 1];
  const uint32_t* keys;
  int32_t first, n;  // this wave's first candidate (from the row's first) and how many
  __device__ void load(const uint32_t* row, int32_t candidates, int wave) {
    const int32_t each = R > 0 ? 64 * R : (candidates + 64 * WAVES - 1) / (64 * WAVES) * 64;
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
      for (int i = 0; i < R; ++i) f(k[i], first + 64 * i + lane_id());
    } else {
      for (int32_t i = 0; i < n; i += 64) {
        f(i + lane_id() < n ? keys[i + lane_id()] : 0u, first + i + lane_id());
      }
    }
  }
};

template <int WAVES, int R>
__global__ void __launch_bounds__(WAVES == 1 ? 4 * kWave : WAVES * kWave)
    kv_keep_kernel(SelectArgs a) {
  __shared__ uint32_t sums[WAVES > 1 ? 40 : 1];
  __shared__ uint32_t part[2][WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int64_t row = WAVES == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + wave : blockIdx.x;
  const int lane = lane_id(), me = WAVES == 1 ? 0 : wave;
  const uint64_t below = (uint64_t{1} << lane) - 1;
  if (row >= a.T * a.Hkv) return;  // (whole waves, and none where a workgroup has one row)
  const KvPlace p = kv_place(a.tok, row / a.Hkv);
  int32_t* out = a.out + row * a.count;
  const int32_t blocks = p.last + 1;
  const int32_t lead = a.sink < blocks ? a.sink : blocks;
  const int32_t end = blocks - a.recent > lead ? blocks - a.recent : lead;
  const int32_t tail = blocks - end;  // of the last `recent`
  const uint32_t want = a.count - a.sink - a.recent;
  Row<WAVES, R> r;
  r.load(a.keys + row * a.stride + lead, end - lead, me);

  if (WAVES > 1) {
    for (int i = threadIdx.x; i < 40; i += WAVES * kWave) sums[i] = 0;
  }
  // candidates and their extreme keys
  uint32_t least = ~0u, most = 0u, total = 0u;
  r.each([&](uint32_t k, int32_t) {
    total += static_cast<uint32_t>(__popcll(__ballot(k != 0)));
    most = k > most ? k : most;
    least = k != 0 && k < least ? k : least;
  });
  most = wave_extreme<true>(most);
  least = wave_extreme<false>(least);
  if (WAVES > 1) {
    __shared__ uint32_t ends[2][WAVES];
    if (lane == 0) {
      ends[0][wave] = most;
      ends[1][wave] = least;
      part[0][wave] = total;
    }
    __syncthreads();
    total = 0;
    for (int w = 0; w < WAVES; ++w) {
      most = ends[0][w] > most ? ends[0][w] : most;
      least = ends[1][w] < least ? ends[1][w] : least;
      total += part[0][w];
    }
  }
  // the largest cut that at least `want` keys reach
  uint32_t cut = 1u, reach = total;
  if (total > want && want > 0) {
    const uint32_t differ = most ^ least;
    int bit = differ != 0 ? 31 - __builtin_clz(differ) : -1;
    cut = bit >= 0 ? most & ~((2u << bit) - 1u) : most;
    int step = 0;
    for (; bit >= 0 && reach != want; --bit, ++step) {
      const uint32_t probe = cut | (1u << bit);
      uint32_t n = 0;
      r.each([&](uint32_t k, int32_t) {
        n += static_cast<uint32_t>(__popcll(__ballot(k >= probe)));
      });
      if (WAVES > 1) {
        if (lane == 0) atomicAdd(&sums[step], n);
        __syncthreads();
        n = sums[step];
      }
      if (n >= want) {
        cut = probe;
        reach = n;
      }
    }
  } else if (want == 0) {
    cut = ~0u;
    reach = 0;
  }
  // more keys than places reach the cut: the lowest blocks of the cut's own key
  uint32_t ties = ~0u;
  uint32_t above = 0, equal = 0;  // this wave's
  const bool tied = reach > want;
  if (want == 0) {
    ties = 0;
  } else if (tied || WAVES > 1) {
    r.each([&](uint32_t k, int32_t) {
      above += static_cast<uint32_t>(__popcll(__ballot(k > cut)));
      equal += static_cast<uint32_t>(__popcll(__ballot(k == cut)));
    });
  }
  uint32_t place = 0;  // kept before this wave's first
  if (WAVES > 1) {
    __syncthreads();  // (every wave has read `part`)
    if (lane == 0) {
      part[0][wave] = above;
      part[1][wave] = equal;
    }
    __syncthreads();
    uint32_t all = 0, ties_before = 0;
    for (int w = 0; w < WAVES; ++w) all += part[0][w];
    if (want > 0) ties = want - all;
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) {
        const uint32_t left = ties > ties_before ? ties - ties_before : 0;
        place += part[0][w] + (part[1][w] < left ? part[1][w] : left);
        ties_before += part[1][w];
      }
    }
    ties = ties > ties_before ? ties - ties_before : 0;
  } else if (tied) {
    ties = want - above;
  }
  r.each([&](uint32_t k, int32_t at) {
    const uint64_t same = __ballot(k == cut);
    const bool keep = k > cut || (k == cut && static_cast<uint32_t>(__popcll(same & below)) < ties);
    const uint64_t kept = __ballot(keep);
    if (keep) out[lead + place + __popcll(kept & below)] = lead + at;
    place += static_cast<uint32_t>(__popcll(kept));
    const uint32_t seen = static_cast<uint32_t>(__popcll(same));
    ties = ties > seen ? ties - seen : 0;
  });
  // the forced blocks and the padding, by the last wave, which knows how many were kept
  if (me == WAVES - 1) {
    for (int32_t i = lane; i < lead; i += kWave) out[i] = i;
    for (int32_t i = lane; i < a.count - lead - static_cast<int32_t>(place); i += kWave) {
      out[lead + place + i] = i < tail ? end + i : -1;
    }
  }
}

struct SelectPlan {
  int64_t stride;
  int32_t tiles, cols, per_wave, splits, head_groups;
};

inline SelectPlan select_plan(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t B,
                              int64_t max_pages, int64_t sink) {
  SelectPlan p;
  const int64_t G = Hq / Hkv;
  p.stride = align_up(static_cast<size_t>(max_pages), kChunk);
  p.cols = static_cast<int32_t>(next_pow2(G < 16 ? G : 16));
  p.head_groups = static_cast<int32_t>(cdiv(Hkv, kScoreWaves));
  const int32_t most = D <= 128 ? 4 : 2;  // tiles whose columns fit in registers beside a chunk
  if (G > 16) {
    p.tiles = G <= 32 ? 2 : most;
    p.per_wave = 1;
  } else {
    // A wave's tokens should mostly be of one sequence: each sequence among them is a pass of all
    // its tiles over that sequence's blocks.
    const int64_t same = B > 0 ? T / B : 0, tile = 16 / p.cols;
    p.tiles = same >= 2 * most * tile ? most : 1;
    p.per_wave = static_cast<int32_t>(same >= 2 ? p.tiles * tile : 1);
  }
  const int64_t waves = cdiv(T, p.per_wave) * Hkv;
  const int64_t chunks = cdiv(max_pages > sink ? max_pages - sink : 1, kChunk);
  const int64_t want = cdiv(4096, waves > 0 ? waves : 1);
  p.splits = static_cast<int32_t>(want < chunks ? want : chunks);
  return p;
}

}  // namespace rt

using namespace rt;

extern "C" size_t rt_kv_select_workspace(int64_t T, int64_t Hkv, int64_t max_pages) {
  if (T < 1 || Hkv < 1 || max_pages < 1) return 0;
  return static_cast<size_t>(T) * Hkv * align_up(static_cast<size_t>(max_pages), kChunk) *
         sizeof(uint32_t);
}

extern "C" int rt_kv_select(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t T,
                            int64_t Hq, int64_t Hkv, int64_t D, int dtype, const int8_t* bounds,
                            const float* bound_scales, int64_t P, int64_t page,
                            const int32_t* positions, const int32_t* seq_ids,
                            const int32_t* page_table, int64_t B, int64_t max_pages, int64_t count,
                            int64_t sink, int64_t recent, int32_t* out, void* workspace,
                            size_t workspace_bytes, rt_stream_t stream) {
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
  RT_CHECK_ARG(T * Hkv <= INT32_MAX, "too many tokens");
  const size_t need = rt_kv_select_workspace(T, Hkv, max_pages);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) {
    set_error("workspace too small: %zu < %zu", workspace_bytes, need);
    return kWorkspaceTooSmall;
  }
  const SelectPlan plan = select_plan(T, Hq, Hkv, D, B, max_pages, sink);
  SelectArgs a{};
  a.q = q, a.q_st = q_token_stride, a.q_sh = q_head_stride, a.T = T;
  a.Hq = static_cast<int32_t>(Hq), a.Hkv = static_cast<int32_t>(Hkv), a.G = a.Hq / a.Hkv;
  a.bounds = bounds, a.scales = bound_scales;
  a.tok = {positions, seq_ids, page_table, static_cast<int32_t>(B),
           static_cast<int32_t>(max_pages), static_cast<int32_t>(P), kv_shift(page)};
  a.count = static_cast<int32_t>(count), a.sink = static_cast<int32_t>(sink);
  a.recent = static_cast<int32_t>(recent), a.out = out, a.keys = static_cast<uint32_t*>(workspace);
  a.stride = plan.stride, a.cols = plan.cols, a.per_wave = plan.per_wave;
  a.splits = plan.splits, a.head_groups = plan.head_groups;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t grid = cdiv(T, plan.per_wave) * plan.splits * plan.head_groups;
  RT_CHECK_ARG(grid <= INT32_MAX, "too many tokens");
  if (max_pages > sink && count > sink + recent) {  // else no block is chosen by its score
    const int st = kv_dispatch(dtype, D, [&](auto e, auto d) -> int {
      using E = decltype(e);
      constexpr int DD = decltype(d)::value;
      const dim3 g(static_cast<unsigned>(grid)), b(kScoreWaves * kWave);
      if (plan.tiles == 1) {
        kv_score_kernel<E, DD, 1><<<g, b, 0, s>>>(a);
      } else if (plan.tiles == 2) {
        kv_score_kernel<E, DD, 2><<<g, b, 0, s>>>(a);
      } else if constexpr (DD <= 128) {
        kv_score_kernel<E, DD, 4><<<g, b, 0, s>>>(a);
      }
      RT_CHECK_HIP(hipGetLastError());
      return kOk;
    });
    if (st != kOk) return st;
  }
  // One wave a row while its keys fit in a few registers a lane, else a workgroup of 16 waves.
  const int64_t rows = T * Hkv;
  const dim3 one(static_cast<unsigned>(rows)), four(static_cast<unsigned>(cdiv(rows, 4)));
  if (max_pages <= 64 * 4) {
    kv_keep_kernel<1, 4><<<four, 4 * kWave, 0, s>>>(a);
  } else if (max_pages <= 64 * 16) {
    kv_keep_kernel<1, 16><<<four, 4 * kWave, 0, s>>>(a);
  } else if (max_pages <= 64 * 16 * 4) {
    kv_keep_kernel<16, 4><<<one, 16 * kWave, 0, s>>>(a);
  } else if (max_pages <= 64 * 16 * 16) {
    kv_keep_kernel<16, 16><<<one, 16 * kWave, 0, s>>>(a);
  } else {
    kv_keep_kernel<16, 0><<<one, 16 * kWave, 0, s>>>(a);
  }
  RT_CHECK_HIP(hipGetLastError());
  return kOk;
}
