// Softmax attention of each token over chosen blocks of the 8-bit paged cache (kv_int8.h).
//
// out = sum_j w_j v_j / sum_j w_j with w_j = exp(x_j), x_j = scale q . k_j over the listed blocks'
// keys at positions up to the token's; keys and values of full blocks are codes times one scale a
// block and head, those of the token's own open block 16-bit numbers.
//
// Codes meet the matrix cores as fp16, which holds them exactly (1024 + 128 + code by a byte
// permutation, less 1152). bf16 queries do as well: a row is scaled by a power of two so that its
// largest magnitude is in [2^14, 2^15), where fp16 holds every 8-bit significand down to 2^-17, so
// what is lost is below 2^-39 of the row's largest. The block's scale of keys multiplies the scores;
// that of values, s_v, goes into the exponent: with t = x log2 e + log2 s_v and m the running maximum
// of t, p = 2^(t - m) is the weight that the second product wants (codes stand for s_v each), and
// p / s_v what the sum of weights wants. So neither product is rescaled from block to block, and p is
// rounded to fp16 (2^-11, held 2^7 times as large as the maximum: it reaches 2^15, and its step
// below 2^-14 is 2^-31 of the largest weight) whatever the type.
//
// A wave holds up to 16 query heads of one key/value head and takes 64 keys a step, four subtiles of
// 16 slots, lane group g (lanes 16 g to 16 g + 15) having subtile g:
//   S^T [keys x heads] = K Q^T     four products of 16 keys: row m of product j is slot 4 j + m % 4 of
//                                  subtile m / 4, so that lane group g gets slots 4 j .. 4 j + 3 of its
//                                  own subtile: 16 neighbouring slots over the four products;
//   O^T [channels x heads] += V^T P^T   the weights are where the first product left them, and the
//                                  operand V^T is 16 bytes of a channel, straight from memory (values
//                                  lie transposed). Nothing passes through LDS.
// A lane's column is one head in both products: maxima, sums and rescaling stay in the lane.
#include <cmath>
#include <type_traits>

#include "../../include/retrieve_amd.h"
#include "kv_attend.h"
#include "kv_int8.h"

namespace rt {

struct AttendInt8Args : AttendBase {
  KvInt8 cache;
};

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef int v2i __attribute__((ext_vector_type(2)));

__device__ inline v4f mma16(v8h a, v8h b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline v4f mma16(Kv<__bf16>::V8 a, Kv<__bf16>::V8 b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Eight codes (two words) as fp16.
__device__ inline v8h codes_to_half(int lo, int hi) {
  union {
    uint32_t u[4];
    v2h h[4];
    v8h v;
  } x;
  const uint32_t a = static_cast<uint32_t>(lo) ^ 0x80808080u;
  const uint32_t b = static_cast<uint32_t>(hi) ^ 0x80808080u;
  x.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
  x.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
  x.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
  x.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
  const v2h bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
#pragma unroll
  for (int i = 0; i < 4; ++i) x.h[i] -= bias;
  return x.v;
}

template <bool STREAM, class V>
__device__ inline V load_once(const V* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  return *p;
}

// A wave's accumulators (channel 16 i + 4 (lane / 16) + r of column lane % 16), the columns' maxima
// of t (less kLift) and this lane's share of their sums; its queries and the step in flight.
template <class E, int D>
struct Int8Wave {
  using V8 = typename Kv<E>::V8;
  static constexpr int DT = D / 16, KS = D / 32;  // channel tiles, steps of 32 channels
  static constexpr int KL = D / 64;               // 16-byte loads of a key a lane
  static constexpr bool HALF = D % 64 != 0;       // and one of 8 bytes
  static constexpr float kLift = 7.0f;            // maximum - m
  v4f acc[DT];
  float m, l;
  v8h qf[KS];
  float factor;  // what a score is multiplied by besides its block's scale
  v4i kf[4][KL];
  v2i kh[HALF ? 4 : 1];
  v4i vf[DT];

  __device__ void clear() {
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
    m = -3.402823466e38f;
    l = 0.0f;
  }
  // The channel of a lane group's eight in step s of the first product.
  __device__ static int channel(int s, int grp) {
    return s < 2 * KL ? 64 * (s >> 1) + 16 * grp + 8 * (s & 1) : 64 * KL + 8 * grp;
  }
  // This lane's column is query head `head` of token t (zeros where it is not `real`).
  __device__ void load_q(const AttendInt8Args& a, int64_t t, int64_t head, bool real) {
    const int grp = lane_id() >> 4;
    const E* q = static_cast<const E*>(a.q) + (real ? t * a.q_st + head * a.q_sh : 0);
    V8 x[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      x[s] = *reinterpret_cast<const V8*>(q + channel(s, grp));
      if (!real) x[s] = V8{};
      if (a.minus) x[s] = -x[s];
    }
    factor = a.scale;
    if constexpr (std::is_same<E, _Float16>::value) {
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[s] = x[s];
    } else {
      float most = 0.0f, odd = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = static_cast<float>(x[s][e]);
          most = fmaxf(most, fabsf(f));
          odd = fmaf(f, 0.0f, odd);  // (not a number beside an infinity or a NaN)
        }
      }
#pragma unroll
      for (int i = 16; i < kWave; i <<= 1) {
        most = fmaxf(most, __shfl_xor(most, i));
        odd += __shfl_xor(odd, i);
      }
      const int up = most > 0.0f && most < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
      factor = ldexpf(factor, -up);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          qf[s][e] = static_cast<_Float16>(ldexpf(static_cast<float>(x[s][e]), up) + odd);
        }
      }
    }
  }

  // What a lane knows of its subtile (16 slots) of the 64 that are looked up at a time.
  struct Subtiles {
    const int32_t* list;
    KvPlace place;
    int32_t head, part, parts;
    int32_t page, at;  // physical page; first slot * 32 + keys (0: none)
    float ks, vs;
    uint64_t full, open;  // subtiles with keys: in codes, in the open block

    // Chunk `chunk` of this wave's units of 64 keys (units part, part + parts, ...). False: past
    // the list's end.
    __device__ bool fetch(const AttendInt8Args& a, int chunk) {
      const int64_t first = (part + static_cast<int64_t>(parts) * 16 * chunk) * 64;
      if (first >= static_cast<int64_t>(a.count) << a.tok.shift) return false;
      const int64_t unit = part + static_cast<int64_t>(parts) * (16 * chunk + (lane_id() >> 2));
      const int64_t key = unit * 64 + 16 * (lane_id() & 3);
      const int64_t entry = key >> a.tok.shift;
      page = 0;
      at = 0;
      ks = vs = 1.0f;
      bool is_open = false;
      if (entry < a.count) {
        const int32_t block = list[entry];
        if (block >= 0 && block <= place.last) {
          const int32_t p = kv_page(a.tok, place, block);
          const int32_t slot = static_cast<int32_t>(key) & ((1 << a.tok.shift) - 1);
          const int32_t n = place.pos - (block << a.tok.shift) - slot + 1;
          if (p >= 0 && n > 0) {
            const int64_t row = static_cast<int64_t>(p) * a.Hkv + head;
            const float k = a.cache.k_scales[row], v = a.cache.v_scales[row];
            is_open = !(k > 0.0f);
            // (a block before the token's own that has no codes was never filled)
            if (!is_open || block == place.last) {
              page = p;
              at = slot * 32 + (n < 16 ? n : 16);
              if (!is_open) ks = k, vs = v;
            }
          }
        }
      }
      full = __ballot(at != 0 && !is_open);
      open = __ballot(at != 0 && is_open);
      return true;
    }
  };
  // A step's four subtiles, as this lane needs them: the one whose keys it loads, the one whose
  // values it loads and whose scores it has.
  struct Step {
    int64_t k_row, v_at;  // first row of keys; first slot of channel 0, bytes
    int32_t n;            // keys of the lane's own subtile
    float ks, vs;
    bool whole;  // of all subtiles every key counts
  };
  // The step of quad i of the subtiles; those outside `mask` have no keys.
  __device__ Step step_of(const AttendInt8Args& a, const Subtiles& s, int i, uint64_t mask) const {
    const int k_from = 4 * i + ((lane_id() & 15) >> 2), own = 4 * i + (lane_id() >> 4);
    Step x;
    const int32_t kp = __shfl(s.page, k_from), ka = __shfl(s.at, k_from);
    const int32_t vp = __shfl(s.page, own), va = __shfl(s.at, own);
    x.k_row = ((static_cast<int64_t>(kp) * a.Hkv + s.head) << a.tok.shift) + (ka >> 5);
    x.v_at = ((static_cast<int64_t>(vp) * a.Hkv + s.head) * D << a.tok.shift) + (va >> 5);
    x.n = (mask >> own) & 1 ? va & 31 : 0;
    x.ks = __shfl(s.ks, own);
    x.vs = __shfl(s.vs, own);
    x.whole = __ballot(x.n != 16) == 0;
    return x;
  }
  template <bool STREAM>
  __device__ void load_k(const AttendInt8Args& a, const Step& s) {
    const int grp = lane_id() >> 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int8_t* row = a.cache.k_codes + (s.k_row + 4 * j + (lane_id() & 3)) * D;
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        kf[j][i] = load_once<STREAM>(reinterpret_cast<const v4i*>(row + 64 * i + 16 * grp));
      }
      if constexpr (HALF) {
        kh[j] = load_once<STREAM>(reinterpret_cast<const v2i*>(row + 64 * KL + 8 * grp));
      }
    }
  }
  template <bool STREAM>
  __device__ void load_v(const AttendInt8Args& a, const Step& s) {
    const int8_t* at = a.cache.v_codes + s.v_at;
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      vf[i] = load_once<STREAM>(
          reinterpret_cast<const v4i*>(at + ((16 * i + (lane_id() & 15)) << a.tok.shift)));
    }
  }
  // The weights of a step's scores (slot 4 j + r of this lane's subtile): the maximum raised, the
  // sum extended. f multiplies the scores, vs is the scale of the subtile's values.
  template <class P>
  __device__ void weigh(v4f (&sc)[4], float f, float vs, int n, bool whole, P (&p)[2]) {
    settle(sc);
    if (!whole) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[j][r] = 4 * j + r < n ? sc[j][r] : -INFINITY;
      }
    }
    f = fmaxf(f, 1.17549435e-38f);  // (a score of -inf stays that)
    const float lift = __builtin_amdgcn_logf(vs);
    float top[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      top[j] = fmaxf(fmaxf(sc[j][0], sc[j][1]), fmaxf(sc[j][2], sc[j][3]));
    }
    const float high = fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), f, lift);
    if (__any(high - m > 8.0f + kLift)) {
      float next = fmaxf(high, __shfl_xor(high, 16));
      next = fmaxf(next, __shfl_xor(next, 32));
      next = fmaxf(next - kLift, m);
      const float keep = __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= keep;
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[i] *= keep;
    }
    const float less = lift - m;
    float sum[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float e[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        e[r] = __builtin_amdgcn_exp2f(fmaf(sc[j][r], f, less));
        p[j / 2][4 * (j % 2) + r] =
            static_cast<std::remove_reference_t<decltype(p[0][0])>>(e[r]);
      }
      sum[j] = (e[0] + e[1]) + (e[2] + e[3]);
    }
    l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), 1.0f / vs, l);
  }
  // One step on what load_k and load_v brought; `fetch_k` and `fetch_v` start the next one's loads
  // as soon as the registers are free.
  template <class FK, class FV>
  __device__ void step(const Step& s, FK&& fetch_k, FV&& fetch_v) {
    v4f sc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sc[j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        sc[j] = mma16(codes_to_half(kf[j][i][0], kf[j][i][1]), qf[2 * i], sc[j]);
        sc[j] = mma16(codes_to_half(kf[j][i][2], kf[j][i][3]), qf[2 * i + 1], sc[j]);
      }
      if constexpr (HALF) sc[j] = mma16(codes_to_half(kh[j][0], kh[j][1]), qf[2 * KL], sc[j]);
    }
    fetch_k();
    v8h p[2];
    weigh(sc, s.ks * factor, s.vs, s.n, s.whole, p);
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      acc[i] = mma16(codes_to_half(vf[i][0], vf[i][1]), p[0], acc[i]);
      acc[i] = mma16(codes_to_half(vf[i][2], vf[i][3]), p[1], acc[i]);
    }
    fetch_v();
  }
  // One step over the open block of token t's sequence: 16-bit rows, in their own type. (Once a list
  // at most, so its queries are read again.)
  __device__ void open_step(const AttendInt8Args& a, int64_t t, int head, int64_t hq, bool real,
                            int first, int n) {
    const int grp = lane_id() >> 4, col = lane_id() & 15;
    const int64_t open =
        ((static_cast<int64_t>(a.tok.seq_ids[t]) * a.Hkv + head) << a.tok.shift) * D;
    const E* q = static_cast<const E*>(a.q) + (real ? t * a.q_st + hq * a.q_sh : 0) + 8 * grp;
    v4f sc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) sc[j] = v4f{0.f, 0.f, 0.f, 0.f};
    const int k_slot = __shfl(first, 16 * (col >> 2));  // (first slot of the keys' subtile)
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      V8 x = *reinterpret_cast<const V8*>(q + 32 * s);
      if (!real) x = V8{};
      if (a.minus) x = -x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const E* k = static_cast<const E*>(a.cache.k_tail) + open +
                     (k_slot + 4 * j + (col & 3)) * D + 32 * s + 8 * grp;
        sc[j] = mma16(*reinterpret_cast<const V8*>(k), x, sc[j]);
      }
    }
    V8 p[2];
    weigh(sc, a.scale, 1.0f, n, false, p);
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      const V8* v = reinterpret_cast<const V8*>(static_cast<const E*>(a.cache.v_tail) + open +
                                                ((16 * i + col) << a.tok.shift) + first);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        V8 x = v[h];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (8 * h + e >= n) x[e] = static_cast<E>(0.0f);  // (slots that hold anything)
        }
        acc[i] = mma16(x, p[h], acc[i]);
      }
    }
  }
  __device__ void join_sums() {
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
  }

  // One token's heads (tile `tile` of the group) over part of its list.
  template <bool STREAM>
  __device__ void run(const AttendInt8Args& a, int64_t t, int head, int tile, int part, int parts) {
    clear();
    Subtiles s;
    s.place = kv_place(a.tok, t);
    if (s.place.last < 0) return;
    s.list = a.blocks + (t * a.Hkv + head) * a.count;
    s.head = head;
    s.part = part;
    s.parts = parts;
    const int g = tile * 16 + (lane_id() & 15);
    const int64_t hq = head * a.G + g;
    load_q(a, t, hq, g < a.G);
    for (int chunk = 0; s.fetch(a, chunk); ++chunk) {
      uint64_t left = s.full;
      Step then;
      bool more = left != 0;
      auto next = [&] {
        const int i = __builtin_ctzll(left) >> 2;
        left &= ~(uint64_t{15} << (4 * i));
        then = step_of(a, s, i, s.full);
      };
      if (more) {
        next();
        load_k<STREAM>(a, then);
        load_v<STREAM>(a, then);
      }
      while (more) {
        const Step now = then;
        more = left != 0;
        if (more) next();
        step(now, [&] { if (more) load_k<STREAM>(a, then); },
             [&] { if (more) load_v<STREAM>(a, then); });
      }
      for (uint64_t open = s.open; open != 0;) {
        const int i = __builtin_ctzll(open) >> 2, own = 4 * i + (lane_id() >> 4);
        const int32_t at = __shfl(s.at, own);
        const bool here = (open >> own) & 1;
        open &= ~(uint64_t{15} << (4 * i));
        open_step(a, t, head, hq, g < a.G, here ? at >> 5 : 0, here ? at & 31 : 0);
      }
    }
    join_sums();
  }
};

// This lane's column, query head `head` of token t, to the outputs.
template <class E, int D>
__device__ inline void emit(const AttendInt8Args& a, const Int8Wave<E, D>& w, int64_t t, int head) {
  typedef E V4 __attribute__((ext_vector_type(4)));
  const int grp = lane_id() >> 4;
  const int64_t row = t * a.Hq + head;
  const float inv = inverse_sum(w.l);
  E* out = static_cast<E*>(a.out) + row * D + 4 * grp;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    V4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = static_cast<E>(w.acc[i][r] * inv);
    *reinterpret_cast<V4*>(out + 16 * i) = x;
  }
  if (grp == 0) a.lse[row] = log_sum(w.m, w.l);
}

// Many rows: a wave a row, four neighbouring tokens of one head a workgroup.
template <class E, int D>
__global__ void __launch_bounds__(kAttendWaves* kWave, D <= 128 ? 2 : 1)
    kv_attend_int8_rows_kernel(AttendInt8Args a) {
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int heads = a.Hkv * a.tiles;
  const int64_t t = static_cast<int64_t>(blockIdx.x / heads) * kAttendWaves + wave;
  if (t >= a.T) return;
  const int head = blockIdx.x % heads / a.tiles, tile = blockIdx.x % heads % a.tiles;
  Int8Wave<E, D> w;
  w.template run<false>(a, t, head, tile, 0, 1);
  const int g = tile * 16 + (lane_id() & 15);
  if (g < a.G) emit(a, w, t, head * a.G + g);
}

// Few rows: the workgroup's waves (and `parts` workgroups) share a row's list.
template <class E, int D>
__global__ void __launch_bounds__(kAttendWaves* kWave, D <= 128 ? 2 : 1)
    kv_attend_int8_split_kernel(AttendInt8Args a) {
  __shared__ __attribute__((aligned(16))) char lds[kAttendWaves][64 * D];
  __shared__ float ml[kAttendWaves][16][2];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int part = blockIdx.x % a.parts;
  const int64_t row = blockIdx.x / a.parts;  // (token, key/value head, tile)
  const int tile = static_cast<int>(row % a.tiles);
  const int head = static_cast<int>(row / a.tiles % a.Hkv);
  const int64_t t = row / a.tiles / a.Hkv;
  Int8Wave<E, D> w;
  // (neighbours of one sequence choose mostly the same blocks: these stay in L2)
  const int32_t seq = a.tok.seq_ids[t];
  const bool beside = (t > 0 && a.tok.seq_ids[t - 1] == seq) ||
                      (t + 1 < a.T && a.tok.seq_ids[t + 1] == seq);
  const int first = part * kAttendWaves + wave, parts = a.parts * kAttendWaves;
  if (beside) {
    w.template run<false>(a, t, head, tile, first, parts);
  } else {
    w.template run<true>(a, t, head, tile, first, parts);
  }
  join_waves<E, D>(a, w.acc, w.m, w.l, t, head, tile, row, part, lds, ml);
}

// How a call of `seqs` sequences at most is spread: `parts` workgroups a row; 0: a wave a row.
struct AttendInt8Plan {
  int64_t rows;
  int32_t tiles, parts;
};

inline AttendInt8Plan attend_int8_plan(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t seqs,
                                       int64_t page, int64_t count) {
  AttendInt8Plan p;
  p.tiles = static_cast<int32_t>(cdiv(Hq / Hkv, 16));
  p.rows = T * Hkv * p.tiles;
  p.parts = 0;
  if (T > seqs && p.rows >= 4096) return p;
  // Workgroups of four waves for two on every CU, each wave with a unit of 64 keys at least.
  const int64_t most = cdiv(count * page, 64 * kAttendWaves);
  const int64_t want = cdiv(512, p.rows > 0 ? p.rows : 1);
  p.parts = static_cast<int32_t>(want < most ? want : most);
  if (p.parts < 1) p.parts = 1;
  return p;
}

}  // namespace rt

using namespace rt;

extern "C" size_t rt_kv_attention_int8_workspace(int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                                 int64_t page, int64_t count) {
  if (Hkv < 1 || T < 1) return 0;
  const AttendInt8Plan p = attend_int8_plan(T, Hq, Hkv, D, 0, page, count);
  return p.parts > 1 ? static_cast<size_t>(p.rows) * p.parts * 16 * (D + 2) * sizeof(float) : 0;
}

extern "C" int rt_kv_attention_int8(
    const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t T, int64_t Hq,
    int64_t Hkv, int64_t D, int dtype, const int8_t* k_codes, const int8_t* v_codes,
    const float* k_scales, const float* v_scales, const void* k_tail, const void* v_tail, int64_t P,
    int64_t page, const int32_t* blocks, int64_t count, const int32_t* positions,
    const int32_t* seq_ids, const int32_t* page_table, int64_t B, int64_t max_pages, float scale,
    int64_t sequences, void* out, float* lse, void* workspace, size_t workspace_bytes,
    rt_stream_t stream) {
  if (const int st = kv_check(T, Hq, Hkv, D, dtype, B, max_pages, P, page)) return st;
  RT_CHECK_ARG(count >= 0 && count <= (1 << 20), "count must be in [0, 2^20], got %lld",
               static_cast<long long>(count));
  if (T == 0) return kOk;
  RT_CHECK_ARG(q && positions && seq_ids && out && lse && (count == 0 || blocks), "null pointer");
  RT_CHECK_ARG(B * max_pages == 0 || page_table, "null page table");
  const KvInt8 cache{const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes),
                     const_cast<float*>(k_scales), const_cast<float*>(v_scales),
                     const_cast<void*>(k_tail), const_cast<void*>(v_tail)};
  if (const int st = kv_check_int8(cache, B, P)) return st;
  RT_CHECK_ARG(kv_rows_aligned(q, q_token_stride, q_head_stride) && kv_rows_aligned(out, 0, 0),
               "rows must start on 16 bytes");
  RT_CHECK_ARG(T * Hq <= INT32_MAX, "too many tokens");
  RT_CHECK_ARG(std::isfinite(scale * kLog2e), "the scale must be finite, got %g",
               static_cast<double>(scale));
  RT_CHECK_ARG(sequences >= 0, "sequences must not be negative, got %lld",
               static_cast<long long>(sequences));
  const size_t need = rt_kv_attention_int8_workspace(T, Hq, Hkv, D, page, count);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) {
    set_error("workspace too small: %zu < %zu", workspace_bytes, need);
    return kWorkspaceTooSmall;
  }
  const AttendInt8Plan plan = attend_int8_plan(T, Hq, Hkv, D, sequences, page, count);
  AttendInt8Args a{};
  a.q = q, a.q_st = q_token_stride, a.q_sh = q_head_stride, a.T = T;
  a.Hq = static_cast<int32_t>(Hq), a.Hkv = static_cast<int32_t>(Hkv);
  a.G = a.Hq / a.Hkv, a.tiles = plan.tiles;
  a.cache = cache, a.blocks = blocks;
  a.count = static_cast<int32_t>(count);
  a.tok = {positions, seq_ids, page_table, static_cast<int32_t>(B),
           static_cast<int32_t>(max_pages), static_cast<int32_t>(P), kv_shift(page)};
  // (a scale of 0 becomes the least number: the scores are 0 all the same, and -inf stays -inf)
  a.scale = fmaxf(fabsf(scale * kLog2e), 1.17549435e-38f), a.minus = scale < 0.0f;
  a.out = out, a.lse = lse, a.parts = plan.parts;
  a.part_out = static_cast<float*>(workspace);
  a.part_ml = a.part_out + (plan.parts > 1 ? plan.rows * plan.parts * 16 * D : 0);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return kv_dispatch(dtype, D, [&](auto e, auto d) -> int {
    using E = decltype(e);
    constexpr int DD = decltype(d)::value;
    const dim3 threads(kAttendWaves * kWave);
    if (plan.parts == 0) {
      const int64_t grid = cdiv(T, kAttendWaves) * Hkv * plan.tiles;
      kv_attend_int8_rows_kernel<E, DD><<<dim3(static_cast<unsigned>(grid)), threads, 0, s>>>(a);
    } else {
      const int64_t grid = plan.rows * plan.parts;
      kv_attend_int8_split_kernel<E, DD><<<dim3(static_cast<unsigned>(grid)), threads, 0, s>>>(a);
      if (plan.parts > 1) {
        kv_join_kernel<E, DD><<<dim3(static_cast<unsigned>(T * Hq)), dim3(DD / 4), 0, s>>>(a);
      }
    }
    RT_CHECK_HIP(hipGetLastError());
    return kOk;
  });
}
