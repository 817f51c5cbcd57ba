// Attention of a few query rows over a run of cached keys, on the matrix cores, straight from memory: the body that
// the decode attention over the 8-bit cache (kvq8.hip) and the attention under a shared prefix (prefix.hip) have in common.
//
//   x_j = (q . k_j) / sqrt(hd) + bias_j,   p_j = 2^(x_j log2 e - m),   out = sum p_j v_j / sum p_j
//
// One pass with a running maximum m and denominator per row (fp32).  A wave takes 32 keys at a time and up to 16 * RT
// rows; the four waves of a workgroup take every fourth run of 32 and merge at the end through LDS.
//
// Operands come from memory in the shape the matrix instruction wants, without a trip through LDS:
//   S^T = K . Q^T    lane (key = l & 15, kq = l >> 4) holds 8 channels of its key: pieces of a cache row
//   O^T = V^T . P^T  the operand wants 8 *keys* of one channel per lane.  A lane loads, for its 8 keys, the VC = hd / 16
//                    channels (l & 15) * VC ..; channel tile j of the product then takes element j of each of the 8 rows
//                    (a permuted numbering of the output channels, undone when the result is written).
//   The 8 keys of lane group kq are 4 kq .. + 3 and 16 + 4 kq .. + 3 of the 32: where the accumulators of S^T already
//   sit, so the probabilities go from accumulators to the second product inside the lane.
#pragma once
#include <type_traits>

#include "common.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef f32x4 f32x4_a4 __attribute__((aligned(4)));

constexpr float kRowsMaskThreshold = -1e30f;  // bias entries at or below: the key is masked
constexpr float kRowsLazyMax = 8.f;           // log2 units the running maximum may lag behind (probabilities stay below 2^8)
constexpr float kLog2e = 1.4426950408889634f;
// fp16 weights count from 2^7 down, not from 1: with the maximum's lag still inside the range, and what falls below its
// smallest number (2^-24) is 2^-31 of the sum.  Sums and results carry the same factor.
template <int PV> constexpr float kWeightTop = PV == O355_F16 ? 7.f : 0.f;

// eight consecutive elements along k of a matrix operand, and the 16 x 16 x 32 product of two such fragments
template <int DT> struct Frag8;
template <> struct Frag8<O355_BF16> {
  typedef bf16x8 T;
  static __device__ __forceinline__ T ld(const void* p) { return *reinterpret_cast<const bf16x8*>(p); }
  static __device__ __forceinline__ T pack(const float (&f)[8]) {
    const u32x4 w = {pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
    return __builtin_bit_cast(bf16x8, w);
  }
  static __device__ __forceinline__ float rest(float f) { return f - round_bf16(f); }
  static __device__ __forceinline__ f32x4 mma(T a, T b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Frag8<O355_F16> {
  typedef f16x8 T;
  static __device__ __forceinline__ T ld(const void* p) { return *reinterpret_cast<const f16x8*>(p); }
  static __device__ __forceinline__ T pack(const float (&f)[8]) {
    const u32x4 w = {pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]), pack_f16x2(f[6], f[7])};
    return __builtin_bit_cast(f16x8, w);
  }
  static __device__ __forceinline__ float rest(float f) { return f - (float)(_Float16)f; }
  static __device__ __forceinline__ f32x4 mma(T a, T b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Frag8<O355_F32> {  // eight 16 x 16 x 4 products: full fp32
  struct T { float f[8]; };
  static __device__ __forceinline__ T ld(const void* p) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
    return T{{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
  }
  static __device__ __forceinline__ T pack(const float (&f)[8]) { return T{{f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]}}; }
  static __device__ __forceinline__ f32x4 mma(const T& a, const T& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.f[i], b.f[i], c, 0, 0, 0);
    return c;
  }
};

// N words from 4 N-byte aligned memory (N = 1, 2, 4, 8)
template <int N>
__device__ __forceinline__ void ld_words(const void* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    w[0] = v[0], w[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4 v = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[4 * i + e] = v[e];
    }
  }
}

// ---- the 32 keys of one step as they come from memory -------------------------------------------------------
// K / V in the activation type.  kb, vb: the step's first row; row[i]: the lane's rows within the step (already
// clamped to the last key): row_k[2] for the two key tiles, row_v[8] for its 8 keys.
template <int DT, int HD>
struct RawKeys {
  static constexpr bool SCALED = false;
  // The weights of a 16-bit type: their rounding to the type, and what it left through a second product.  16 bits of a weight
  // (fp16: 22) leave the result's own rounding as the only one that counts, as where the weights stay in fp32
  // (32 sequences, 32 heads, under 4001 keys 34.3 us with and without; 64 under 2048 27.0 against 26.5 with weights of 8 bits).
  static constexpr bool REST = DT != O355_F32;
  static constexpr int PV = DT;  // type of the second product
  static constexpr int ES = DT == O355_F32 ? 4 : 2, STEPS = HD / 32, VC = HD / 16, VW = VC * ES / 4;
  typename Frag8<DT>::T k[2][STEPS];
  uint32_t v[8][VW];
  static __device__ __forceinline__ int q_elem(int s, int kq) { return 32 * s + 8 * kq; }
  __device__ __forceinline__ void load_k(const unsigned char* kb, const int (&row_k)[2], int kq) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int s = 0; s < STEPS; ++s) k[kt][s] = Frag8<DT>::ld(kb + (uint32_t)(row_k[kt] * (HD * ES) + (32 * s + 8 * kq) * ES));
  }
  __device__ __forceinline__ void load_v(const unsigned char* vb, const int (&row_v)[8], int col) {
#pragma unroll
    for (int e = 0; e < 8; ++e) ld_words<VW>(vb + (uint32_t)(row_v[e] * (HD * ES) + col * (VC * ES)), v[e]);
  }
  __device__ __forceinline__ typename Frag8<DT>::T kfrag(int kt, int s) const { return k[kt][s]; }
  __device__ __forceinline__ typename Frag8<DT>::T vfrag(int j) const {
    if constexpr (DT == O355_F32) {
      typename Frag8<DT>::T r;
#pragma unroll
      for (int e = 0; e < 8; ++e) r.f[e] = __uint_as_float(v[e][j]);
      return r;
    } else {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i)  // half j & 1 of word j / 2 of two neighbouring keys
        w[i] = __builtin_amdgcn_perm(v[2 * i + 1][j >> 1], v[2 * i][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
      return __builtin_bit_cast(typename Frag8<DT>::T, w);
    }
  }
  __device__ __forceinline__ void keep(int e, uint32_t ones) {  // ones 0: key e of the lane weighs nothing, whatever its values hold
#pragma unroll
    for (int i = 0; i < VW; ++i) v[e][i] &= ones;
  }
};

// K / V as 8-bit codes.  A 16-byte load holds two steps' worth of a key: its channels 64 i + 16 kq .. + 15.
template <int DT, int HD>
struct Q8Keys {
  static constexpr bool SCALED = true;
  // The value codes are multiplied with p * scale in bf16 for both 16-bit types: p * scale has no bound that would keep it
  // inside fp16's range.  REST: what the rounding to bf16 left goes through a second product, which keeps 16 bits of every
  // weight; fp16 results need them.  fp32 activations stay in fp32.
  static constexpr bool REST = DT != O355_F32;
  static constexpr int PV = DT == O355_F32 ? O355_F32 : O355_BF16;
  static constexpr int STEPS = HD / 32, VC = HD / 16, KW = HD / 16;  // KW: words of a key per lane
  uint32_t k[2][KW];
  u32x2 v[8];  // VC codes: 8, 4 or 2 of the bytes
  static __device__ __forceinline__ int q_elem(int s, int kq) { return HD == 32 ? 8 * kq : 64 * (s >> 1) + 16 * kq + 8 * (s & 1); }
  __device__ __forceinline__ void load_k(const unsigned char* kb, const int (&row_k)[2], int kq) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      if constexpr (HD == 32) {
        ld_words<2>(kb + (uint32_t)(row_k[kt] * HD + 8 * kq), k[kt]);
      } else {
#pragma unroll
        for (int i = 0; i < HD / 64; ++i) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(kb + (uint32_t)(row_k[kt] * HD + 64 * i + 16 * kq));
#pragma unroll
          for (int e = 0; e < 4; ++e) k[kt][4 * i + e] = w[e];
        }
      }
    }
  }
  __device__ __forceinline__ void load_v(const unsigned char* vb, const int (&row_v)[8], int col) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned char* p = vb + (uint32_t)(row_v[e] * HD + col * VC);
      if constexpr (VC == 8) v[e] = *reinterpret_cast<const u32x2*>(p);
      else if constexpr (VC == 4) v[e] = u32x2{*reinterpret_cast<const uint32_t*>(p), 0u};
      else v[e] = u32x2{(uint32_t)*reinterpret_cast<const uint16_t*>(p), 0u};
    }
  }
  static __device__ __forceinline__ float code(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }
  __device__ __forceinline__ typename Frag8<DT>::T kfrag(int kt, int s) const {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = code(k[kt][2 * s + (e >> 2)], e & 3);
    return Frag8<DT>::pack(f);  // integers up to 127: exact in every type
  }
  __device__ __forceinline__ typename Frag8<PV>::T vfrag(int j) const {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = code(v[e][j >> 2], j & 3);
    return Frag8<PV>::pack(f);
  }
};

// ---- rows x keys -> (m, l, o) -----------------------------------------------------------
struct RowsIn {
  const unsigned char* q;  // the activation rows [token][H][HD]
  int tok0;                // row r belongs to token tok0 + r / G, head head0 + r % G
  int G, H, head0;
  int r0, nrows;           // rows r0 .. nrows - 1 are this workgroup's (at most 16 * RT of them are taken)
  const unsigned char *k, *v;   // this kv head's keys and values, row 0
  const float *ks, *vs;         // scales of the 8-bit form
  const float* bias;            // per key, or NULL
  int keys;                     // keys in all (rows past them are not read)
  int past;                     // causal: row r sees keys <= past + r / G; -1: all keys
};

// run `i` of `n` of `steps` steps
struct Run {
  int lo, hi;
};
__device__ __forceinline__ Run run_of(uint32_t steps, uint32_t i, uint32_t n) {
  const uint32_t each = steps / n, rest = steps - each * n, lo = i * each + min(i, rest);
  return {(int)lo, (int)(lo + each + (i < rest ? 1 : 0))};
}

template <int HD>
struct RowsLds {
  static constexpr int PITCH = HD + 4;
  float m[4][64], l[4][64];
  float o[4][16][PITCH];
};

template <int HD, int RT>
struct RowsAcc {  // O^T: lane (row = l & 15, kq) holds channels (4 kq + r) * VC + j of its row in o[.][j][r]
  f32x4 o[RT][HD / 16];
  float m[RT], l[RT];  // l: this lane's share (its 8 of every 32 keys)
};

// One wave: its rows over the runs of 32 keys step_lo, step_lo + stride, ... < step_hi.
// What a row's masked keys count: KEEP_MASKED: a masked key keeps the type's lowest value as its score (so a row of nothing
// but masked keys averages them, as the decode attention does); otherwise it weighs nothing.
template <int DT, int HD, int RT, bool KEEP_MASKED, class Keys>
__device__ __forceinline__ void walk_keys(const RowsIn& in, int step_lo, int step_hi, int stride, RowsAcc<HD, RT>& acc) {
  typedef Frag8<DT> FQ;
  typedef Frag8<Keys::PV> FP;
  constexpr int STEPS = HD / 32, VC = HD / 16, ES = DT == O355_F32 ? 4 : 2;
  constexpr int KROW = Keys::SCALED ? HD : HD * ES;  // bytes of a key row
  // fp32 heads of 128 under two row tiles: K and V of a step are 64 registers each beside 128 of q and o.  They take turns in
  // the same 64 (V is asked for behind the first product, K behind the second), so that two waves fit a SIMD
  // (41 sequences x 17 tokens of 32 / 16 heads behind 517 keys 136 -> 105 us; 64 x 1 of 8 heads behind 4001 39 -> 32).
  constexpr bool TURNS = DT == O355_F32 && HD == 128 && RT == 2;
  const float* const bias = in.bias;
  const int lane = threadIdx.x & 63, col = lane & 15, kq = lane >> 4;
  const float c2 = kLog2e / sqrtf((float)HD);  // scores in the log2 domain
  // the masked keys' score in the log2 domain; where it would pass fp32's range the type's own lowest is below all others too
  const float lowest = DT == O355_F16 ? Act<DT>::lowest() * kLog2e : Act<DT>::lowest();
  auto& o = acc.o;
  auto& m = acc.m;
  auto& l = acc.l;

  typename FQ::T qf[RT][STEPS];
  int sees[RT];  // last key visible to the row
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = min(in.r0 + 16 * rt + col, in.nrows - 1);
    const int t = r / in.G;
    sees[rt] = in.past < 0 ? in.keys - 1 : min(in.past + t, in.keys - 1);
    const unsigned char* src = in.q + (((int64_t)(in.tok0 + t) * in.H + in.head0 + (r - t * in.G)) * HD) * ES;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) qf[rt][s] = FQ::ld(src + Keys::q_elem(s, kq) * ES);
    m[rt] = -INFINITY, l[rt] = 0.f;
#pragma unroll
    for (int j = 0; j < VC; ++j) o[rt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (step_lo >= step_hi) return;
  const int all_see = in.past < 0 ? in.keys - 1 : in.past + in.r0 / in.G;  // the last key that every row sees

  // The loads of the next 32 keys go out as soon as the registers of the present ones are free: K after the first product, V
  // after the second, so that one of them is on its way at any time without a second set of registers.  No load sits in a
  // branch: behind a join the compiler would have to wait for all loads in flight instead of the older half.
  // Per-key numbers (scales, bias): the four lanes of a quad load those of the lane group's four keys of a tile, one each,
  // and get the others' by quad broadcast when they are used.
  Keys kv;
  float sk[2], sv[2], bs[2], next_sk[2], next_sv[2], next_bs[2];
  auto request_k = [&](int step) {
    const int k0 = step * 32, left = in.keys - 1 - k0;  // left >= 0: the last row of the step that exists
    int row_k[2] = {col, 16 + col}, row_s[2] = {4 * kq + (col & 3), 16 + 4 * kq + (col & 3)};
    if (left < 31) {
#pragma unroll
      for (int i = 0; i < 2; ++i) row_k[i] = min(row_k[i], left), row_s[i] = min(row_s[i], left);
    }
    kv.load_k(in.k + (int64_t)k0 * KROW, row_k, kq);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (Keys::SCALED) next_sk[h] = in.ks[k0 + row_s[h]], next_sv[h] = in.vs[k0 + row_s[h]];
      next_bs[h] = bias ? bias[k0 + row_s[h]] : 0.f;
    }
  };
  auto request_v = [&](int step) {
    const int k0 = step * 32, left = in.keys - 1 - k0;
    int row_v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) row_v[e] = 4 * kq + (e & 3) + 16 * (e >> 2);
    if (left < 31) {
#pragma unroll
      for (int e = 0; e < 8; ++e) row_v[e] = min(row_v[e], left);
    }
    kv.load_v(in.v + (int64_t)k0 * KROW, row_v, col);
  };
  auto of_quad = [](const float (&f)[2], int e) {  // lane e & 3 of the quad
    return (e & 3) == 0 ? dpp_lane<0x00>(f[e >> 2]) : (e & 3) == 1 ? dpp_lane<0x55>(f[e >> 2]) : (e & 3) == 2 ? dpp_lane<0xAA>(f[e >> 2]) : dpp_lane<0xFF>(f[e >> 2]);
  };
  auto multiply = [&](int step, auto more) {
    constexpr bool MORE = decltype(more)::value;
    const int k0 = step * 32;
#pragma unroll
    for (int h = 0; h < 2; ++h) sk[h] = next_sk[h], sv[h] = next_sv[h], bs[h] = next_bs[h];
    // ---- S^T = K . Q^T
    f32x4 s[RT][2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        const auto kf = kv.kfrag(kt, st);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][kt] = FQ::mma(kf, qf[rt][st], st == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[rt][kt]);
      }
    if constexpr (TURNS) request_v(step);
    else if constexpr (MORE) request_k(step + stride);
    if constexpr (Keys::SCALED) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float k = of_quad(sk, e);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][e >> 2][e & 3] *= k;
      }
    }
    // scores into the log2 domain: at once where a bias is added or keys are hidden, else inside the exponent
    const bool hides = k0 + 31 > all_see, plain = !bias && !hides;
    if (!plain) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float b1 = of_quad(bs, e), b2 = b1 * kLog2e;
        const bool masked = b1 <= kRowsMaskThreshold;
        if constexpr (!KEEP_MASKED) kv.keep(e, masked ? 0u : ~0u);
        const int key = k0 + 4 * kq + (e & 3) + 16 * (e >> 2);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float v = __builtin_fmaf(s[rt][e >> 2][e & 3], c2, b2);
          v = masked ? (KEEP_MASKED ? lowest : -INFINITY) : v;
          s[rt][e >> 2][e & 3] = key > sees[rt] ? -INFINITY : v;
        }
      }
    }
    const float cs = plain ? c2 : 1.f;
    // ---- running maximum, probabilities
    typename FP::T pf[RT], pl[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float tmax = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) tmax = fmaxf(tmax, s[rt][e >> 2][e & 3]);
      tmax *= cs;  // cs > 0: the maximum commutes with the scaling
      // The reference maximum moves only when some row's new maximum is more than kRowsLazyMax above it.
      if (__builtin_amdgcn_ballot_w64(tmax > m[rt] + kRowsLazyMax) != 0) {
        tmax = combine_xor32(combine_xor16(tmax, MaxOp{}), MaxOp{});
        const float mn = tmax > m[rt] + kRowsLazyMax ? tmax : m[rt];
        const float alpha = mn == m[rt] ? 1.f : __builtin_amdgcn_exp2f(m[rt] - mn);
        l[rt] *= alpha;
#pragma unroll
        for (int j = 0; j < VC; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[rt][j][r] = alpha == 0.f ? 0.f : o[rt][j][r] * alpha;  // see merge_waves
        m[rt] = mn;
      }
      const float mref = (m[rt] == -INFINITY ? 0.f : m[rt]) - kWeightTop<Keys::PV>;  // 0: a row that has seen no key yet
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][e >> 2][e & 3], cs, -mref));
        l[rt] += p[e];
        if constexpr (Keys::SCALED) {  // the scale of a key that weighs nothing may be NaN
          const float v = of_quad(sv, e);
          p[e] = p[e] == 0.f ? 0.f : p[e] * v;
        }
      }
      pf[rt] = FP::pack(p);
      if constexpr (Keys::REST) {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = FP::rest(p[e]);
        pl[rt] = FP::pack(p);
      }
    }
    // ---- O^T += V^T . P^T
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      const auto vf = kv.vfrag(j);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        o[rt][j] = FP::mma(vf, pf[rt], o[rt][j]);
        if constexpr (Keys::REST) o[rt][j] = FP::mma(vf, pl[rt], o[rt][j]);
      }
    }
    if constexpr (MORE && TURNS) request_k(step + stride);
    else if constexpr (MORE) request_v(step + stride);
  };
  request_k(step_lo);
  if constexpr (!TURNS) request_v(step_lo);
  int step = step_lo;
  for (; step + stride < step_hi; step += stride) multiply(step, std::true_type{});
  multiply(step, std::false_type{});
}

// The results of a workgroup's four waves, which took every fourth run of 32 keys, as one.
// emit(row, channel, VC values of o, m, l): called by 16 threads per row, once for every row of the workgroup.
template <int HD, int RT, class Emit>
__device__ __forceinline__ void merge_waves(const RowsIn& in, RowsAcc<HD, RT>& acc, RowsLds<HD>& lds, Emit emit) {
  constexpr int VC = HD / 16;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, kq = lane >> 4;
  auto& o = acc.o;
  auto& m = acc.m;
  auto& l = acc.l;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] = combine_xor32(combine_xor16(l[rt], AddOp{}), AddOp{});
    if (kq == 0) lds.m[wave][16 * rt + col] = m[rt], lds.l[wave][16 * rt + col] = l[rt];
  }
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, lds.m[w][16 * rt + col]);
    // What a wave gathered under a maximum that turns out to weigh nothing is left out, not multiplied by zero: it may be the
    // mean of masked keys' values, which are not looked at once the row has a key that is not masked.
    const float alpha = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[rt] - mm);
    if (in.r0 + 16 * rt + col < in.nrows) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VC; ++j) lds.o[wave][col][(4 * kq + r) * VC + j] = alpha == 0.f ? 0.f : o[rt][j][r] * alpha;
    }
    __syncthreads();
    const int rr = tid >> 4, c = (tid & 15) * VC, row = in.r0 + 16 * rt + rr;
    if (row < in.nrows) {
      float ov[VC], mrow = -INFINITY, lrow = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) mrow = fmaxf(mrow, lds.m[w][16 * rt + rr]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float mw = lds.m[w][16 * rt + rr], lw = lds.l[w][16 * rt + rr];
        lrow += mw == -INFINITY ? lw : lw * __builtin_amdgcn_exp2f(mw - mrow);  // lw is 0 there, or NaN from a NaN score
      }
#pragma unroll
      for (int j = 0; j < VC; ++j) ov[j] = (lds.o[0][rr][c + j] + lds.o[1][rr][c + j]) + (lds.o[2][rr][c + j] + lds.o[3][rr][c + j]);
      emit(row, c, ov, mrow, lrow);
    }
    if (rt + 1 < RT) __syncthreads();
  }
}

// VC consecutive values of an output row
template <int DT, int VC>
__device__ __forceinline__ void st_row(void* out, int64_t elem, const float (&f)[VC]) {
  if constexpr (DT == O355_F32) {
#pragma unroll
    for (int i = 0; i < VC; i += 2) *reinterpret_cast<u32x2*>((float*)out + elem + i) = u32x2{__float_as_uint(f[i]), __float_as_uint(f[i + 1])};
  } else {
#pragma unroll
    for (int i = 0; i < VC; i += 2)
      *reinterpret_cast<uint32_t*>((uint16_t*)out + elem + i) = DT == O355_BF16 ? pack_bf16x2(f[i], f[i + 1]) : pack_f16x2(f[i], f[i + 1]);
  }
}

// Partial results of rows whose keys several workgroups share: o unnormalised [part][rows][HD], then (m, l) [part][rows].
__host__ __device__ __forceinline__ int64_t rows_parts_floats(int64_t rows, int hd, int parts) { return rows * parts * (hd + 2); }

// A wave per row: its four groups of 16 lanes take every fourth part, lane c the VC channels c * VC ...
template <int DT, int HD>
__global__ __launch_bounds__(256) void rows_combine_kernel(const float* __restrict__ ws, void* __restrict__ out, int64_t rows, int parts) {
  constexpr int VC = HD / 16;
  const int lane = threadIdx.x & 63, grp = lane >> 4, c = (lane & 15) * VC;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const f32x2* ml = reinterpret_cast<const f32x2*>(ws + rows * parts * HD);
  float mm = -INFINITY;
  for (int i = lane; i < parts; i += 64) mm = fmaxf(mm, ml[i * rows + row][0]);
  mm = wave_max(mm);
  float l = 0.f, o[VC];
#pragma unroll
  for (int j = 0; j < VC; ++j) o[j] = 0.f;
#pragma unroll 4
  for (int i = grp; i < parts; i += 4) {
    const f32x2 p = ml[i * rows + row];
    const float* src = ws + (i * rows + row) * HD + c;
    float v[VC];
#pragma unroll
    for (int j = 0; j < VC; ++j) v[j] = src[j];
    const float w = p[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(p[0] - mm);
    l += p[0] == -INFINITY ? p[1] : p[1] * w;  // no key seen: 0, or NaN from a NaN score
#pragma unroll
    for (int j = 0; j < VC; ++j) o[j] += w == 0.f ? 0.f : w * v[j];
  }
  l = combine_xor32(combine_xor16(l, AddOp{}), AddOp{});
#pragma unroll
  for (int j = 0; j < VC; ++j) o[j] = combine_xor32(combine_xor16(o[j], AddOp{}), AddOp{}) / l;
  if (grp == 0) st_row<DT, VC>(out, row * HD + c, o);
}

}  // namespace
