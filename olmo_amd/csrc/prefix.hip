// Attention of a batch whose sequences share one prefix (a system prompt, a document asked about many times).
//
// The prefix's keys and values exist once, [Hkv, Pmax, hd]; every sequence has its own cache [B, Hkv, Lmax, hd] for what
// follows.  Row (b, t) sees all P prefix keys and its own keys 0 .. past + t:
//   out = (sum_prefix p v + sum_own p v) / (sum_prefix p + sum_own p),   p = exp(q . k / sqrt(hd) + bias)
// The prefix part is the same keys for every sequence: all B * T * (H / Hkv) rows of a kv head go through the matrix
// product together, so the prefix is read once per 16 * RT rows instead of once per sequence.
#include "attn_rows.h"

namespace {

struct PrefixPlan {
  int rtp, rto;          // 16-row tiles per workgroup, prefix part and own part
  int tiles_p, tiles_o;  // row tiles per kv head (prefix) and per sequence and kv head (own)
  int splits_p, splits_o;
  int most;                // both for any fewer own or prefix keys, counted or not (what a workspace has to hold)
  int64_t wgs_p, wgs_o;    // workgroups per kv head
  int64_t own_waves;       // waves of the own part per kv head
};

// counted: n_keys_max is the count of own keys, not a bound that a captured step was given.
PrefixPlan prefix_plan(int B, int T, int H, int Hkv, int P, int n_keys_max, bool counted) {
  PrefixPlan p;
  const int64_t G = H / Hkv, rows_o = T * G, rows_p = B * rows_o;
  // (four tiles need the registers of a whole SIMD: 64 sequences of 32 heads under 2048 keys took 66 us against 39 with two when
  // both were built, 256 sequences 175 against 114)
  p.rtp = rows_p <= 16 ? 1 : 2;
  p.rto = rows_o <= 16 ? 1 : p.rtp;
  p.tiles_p = (int)((rows_p + 16 * p.rtp - 1) / (16 * p.rtp));
  p.tiles_o = (int)((rows_o + 16 * p.rto - 1) / (16 * p.rto));
  auto at_most = [](int64_t want, int64_t most) { return (int)(want < 1 ? 1 : want > most ? most : want); };
  // Rounds of two workgroups per CU (512, or 2048 waves of own keys), shared between own keys and prefix in proportion to
  // their keys, so that every wave has about as many: at least two steps of own keys each, a step per wave of the prefix's.
  // Whole rounds matter more than the share: 32 heads, 8 sequences of 4000 own keys behind 1000 take 97 us with 448 + 64
  // workgroups, 119 with 256 + 256, 129 with 256 + 32; 16 of 2000 behind 500 97 with 384 + 128, 126 with 256 + 128, 111 with
  // 512 + 128; 4 under 16384 52 with 480 + 32, 59 with 512 + 32; 32 of 100 under 4001 29.5 with 256 + 256, 33 with 512 + 512.
  // So own keys round down, and the prefix gets a round of its own only if what is left falls short of its share.
  // Where the count of own keys is only bounded, they get half a round: by proportion, 8 sequences of 50 keys out of 3000
  // behind 1000 take 18 us instead of 12 (of 1900 51 instead of 61), 16 of 50 out of 2048, 8 kv heads, behind 2000 22 instead of 17.
  const int64_t units_o = (int64_t)B * Hkv * p.tiles_o, units_p = (int64_t)Hkv * p.tiles_p;
  const int64_t work_o = units_o * n_keys_max, work_p = units_p * P, steps_o = (n_keys_max + 63ll) / 64, steps_p = (P + 127ll) / 128;
  const double share_p = counted ? (double)work_p / (double)(work_o + work_p) : 0.5;
  p.splits_o = at_most((int64_t)(2048 * (1 - share_p)) / units_o, steps_o);
  const int64_t own = ((int64_t)B * p.tiles_o * p.splits_o + 3) / 4 * Hkv, room = 512 - own % 512;
  p.splits_p = at_most((room < at_most((int64_t)(512 * share_p), 192) ? room + 512 : room) / units_p, steps_p);
  p.most = at_most(2048 / units_o, steps_o) + at_most((192 + 511) / units_p, steps_p);
  p.wgs_p = (int64_t)p.tiles_p * p.splits_p;
  p.own_waves = (int64_t)B * p.tiles_o * p.splits_o;
  p.wgs_o = (p.own_waves + 3) / 4;
  return p;
}

// Two waves per SIMD in every instance: with the registers of one the compiler keeps accumulators and operands in AGPRs, and its
// scheduler has then let scores overwrite value words that a product had still to read (fp32).
template <int DT, int HD, int RTP, int RTO>
__global__ __launch_bounds__(256, 2) void attn_shared_prefix_kernel(
    const void* __restrict__ q, const void* __restrict__ kp, const void* __restrict__ vp, const void* __restrict__ kc,
    const void* __restrict__ vc, const float* __restrict__ key_bias, float* __restrict__ ws, int B, int T, int G, int Hkv, int P,
    int64_t Pmax, int64_t Lmax, int past_len, const int32_t* __restrict__ past_dev, int n_keys_max, int bias_stride, PrefixPlan plan) {
  constexpr int ES = DT == O355_F32 ? 4 : 2, VC = HD / 16;
  __shared__ RowsLds<HD> lds;
  const int H = Hkv * G;
  const int64_t rows = (int64_t)B * T * H;
  const int parts = plan.splits_p + plan.splits_o;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, kq = lane >> 4;
  RowsIn in;
  in.q = (const unsigned char*)q, in.G = G, in.H = H, in.ks = in.vs = nullptr;
  int part;
  auto emit = [&](int r, int c, auto& o, float m, float l) {
    const int t = r / G;
    const int64_t at = (int64_t)(in.tok0 + t) * H + in.head0 + (r - t * G);
    st_row<O355_F32, VC>(ws, (part * rows + at) * HD + c, o);
    if (c == 0) {
      float* ml = ws + rows * parts * HD + (part * rows + at) * 2;
      ml[0] = m, ml[1] = l;
    }
  };
  const int hk = blockIdx.y;
  uint32_t i = blockIdx.x;
  if (i < (uint32_t)plan.wgs_p) {
    // The row tiles that read the same keys: eight workgroups apart, so on the same die, one after the other, as long as there
    // are eight runs to go round (16 sequences, 40 / 8 heads, prefix 8000, 2000 own keys 41.8 -> 37.3 us; 17 of 12 / 4 heads,
    // 8266, 608 20.1 -> 18.8; with fewer runs as it was).
    const uint32_t splits = plan.splits_p, tiles = plan.tiles_p, whole = splits & ~7u;
    uint32_t tile;
    if (i < whole * tiles) {
      const uint32_t group = i / (8 * tiles), r = i - group * 8 * tiles;
      tile = r >> 3, part = (int)(group * 8 + (r & 7));
    } else {
      const uint32_t r = i - whole * tiles, left = splits - whole;
      tile = r / left, part = (int)(whole + r - tile * left);
    }
    in.tok0 = 0, in.head0 = hk * G;
    in.r0 = tile * 16 * RTP, in.nrows = B * T * G;
    in.k = (const unsigned char*)kp + hk * Pmax * HD * ES, in.v = (const unsigned char*)vp + hk * Pmax * HD * ES;
    in.bias = nullptr, in.keys = P, in.past = -1;
    const Run run = run_of((uint32_t)(P + 31) / 32, part, plan.splits_p);
    RowsAcc<HD, RTP> acc;
    walk_keys<DT, HD, RTP, false, RawKeys<DT, HD>>(in, run.lo + wave, run.hi, 4, acc);
    merge_waves<HD, RTP>(in, acc, lds, emit);
    return;
  }
  i = (i - (uint32_t)plan.wgs_p) * 4 + wave;  // the own keys: a wave of its own for every run of keys of a row tile
  if (i >= (uint32_t)plan.own_waves) return;
  const uint32_t i1 = i / (uint32_t)plan.splits_o, split = i - i1 * plan.splits_o;
  const uint32_t b = i1 / (uint32_t)plan.tiles_o, tile = i1 - b * plan.tiles_o;
  const int64_t bh = (int64_t)b * Hkv + hk;
  const int past = past_dev ? max(0, min(*past_dev, n_keys_max - 1)) : past_len;
  part = plan.splits_p + split;
  in.tok0 = b * T, in.head0 = hk * G;
  in.r0 = tile * 16 * RTO, in.nrows = T * G;
  const int last = past + min(in.r0 + 16 * RTO - 1, T * G - 1) / G;  // the last key that a row of this tile sees
  in.k = (const unsigned char*)kc + bh * Lmax * HD * ES, in.v = (const unsigned char*)vc + bh * Lmax * HD * ES;
  in.bias = key_bias ? key_bias + (int64_t)b * bias_stride : nullptr;
  in.keys = last + 1, in.past = past;
  const Run run = run_of((uint32_t)(last + 32) / 32, split, plan.splits_o);
  RowsAcc<HD, RTO> acc;
  walk_keys<DT, HD, RTO, false, RawKeys<DT, HD>>(in, run.lo, run.hi, 1, acc);
#pragma unroll
  for (int rt = 0; rt < RTO; ++rt) {
    const float l = combine_xor32(combine_xor16(acc.l[rt], AddOp{}), AddOp{});
    const int r = in.r0 + 16 * rt + col, t = r / G;
    if (r >= in.nrows) continue;
    const int64_t at = part * rows + (int64_t)(in.tok0 + t) * H + in.head0 + (r - t * G);
#pragma unroll
    for (int j4 = 0; j4 < 4; ++j4) {
      float f[VC];
#pragma unroll
      for (int j = 0; j < VC; ++j) f[j] = acc.o[rt][j][j4];
      st_row<O355_F32, VC>(ws, at * HD + (4 * kq + j4) * VC, f);
    }
    if (kq == 0) *reinterpret_cast<f32x2*>(ws + rows * parts * HD + at * 2) = f32x2{acc.m[rt], l};
  }
}

// ---- many new tokens per sequence: one pass over prefix and own keys --------------------------------------------------
// A workgroup takes 128 rows (token, head of the group) of one sequence and kv head, 32 to a wave, through the prefix and then
// through the sequence's own keys with the same running maximum: nothing is left to merge (unless there are
// so few workgroups that several share the keys).  64 keys at a time lie in LDS,
// two tiles of them: the next one travels memory -> LDS directly while the present one is multiplied, one barrier per tile.
//   K: [key tile 4][hd step][64 lanes][8]: fragments of S^T = K . Q^T, each one conflict-free ds_read_b128
//   V: [key 64][hd], the 32-byte units of a row XOR-swizzled by the key, read with the transposing load: lane r of a group of 16
//      supplies the address of four channels of key 4 kq + r / 4, lane j receives its channel of keys 4 kq .. + 3
// Bound by the matrix and exponent units: see the measurements at the plan below.
template <int HD>
struct ChainLds {
  static constexpr int KT = 64, TILE = KT * HD * 2, BYTES = 4 * TILE + 2 * KT * 4;  // K x 2, V x 2, bias x 2
};

// One wave's requests for a K / V tile: HD / 32 instructions of 1 KiB per operand.  (The body is for the device pass alone: the
// host pass does not know the memory -> LDS builtin, drops the templates that reach it, and leaves the kernel without a
// launch stub.)
template <int S>
__device__ __forceinline__ void chain_request_tile(__amdgpu_buffer_rsrc_t rk, __amdgpu_buffer_rsrc_t rv, unsigned char* kdst,
                                                   unsigned char* vdst, const int (&k_row)[S], const int (&k_in)[S], const int (&v_row)[S],
                                                   const int (&v_in)[S], int left) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int ROW = 64 * S;  // bytes of a key row
#pragma unroll
  for (int i = 0; i < S; ++i) {  // rows past the last key may hold anything: the last one is read in their place
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_ptr_t)(kdst + (i << 10)), 16, min(k_row[i], left) * ROW + k_in[i], 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_ptr_t)(vdst + (i << 10)), 16, min(v_row[i], left) * ROW + v_in[i], 0, 0, 0);
  }
#endif
}

template <int DT, int HD>
__global__ __launch_bounds__(256, 2) void attn_prefix_chain_kernel(const uint16_t* __restrict__ q, const uint16_t* __restrict__ kp,
                                                                   const uint16_t* __restrict__ vp, const uint16_t* __restrict__ kc,
                                                                   const uint16_t* __restrict__ vc, const float* __restrict__ key_bias,
                                                                   uint16_t* __restrict__ out, float* __restrict__ ws, int T, int G, int Hkv, int P,
                                                                   int64_t Pmax, int64_t Lmax, int past, int bias_stride, int parts) {
  typedef Frag8<DT> F;
  constexpr int KT = 64, STEPS = HD / 32, HT = HD / 16, QT = 2, TILE = ChainLds<HD>::TILE, CPR = HD / 8, VROW = HD * 2;
  constexpr bool REST = DT == O355_F16;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* const lds_k = smem;
  unsigned char* const lds_v = smem + 2 * TILE;
  float* const lds_bias = reinterpret_cast<float*>(smem + 4 * TILE);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, kq = lane >> 4;
  const int hk = blockIdx.x, b = blockIdx.z;
  const uint32_t of_end = gridDim.y - 1 - blockIdx.y;  // the blocks with the most keys first
  const int block = (int)(of_end / (uint32_t)parts), part = (int)(of_end - (uint32_t)block * parts);
  const int H = Hkv * G, nrows = T * G, r0 = block * 128 + wave * 32;
  const int64_t bh = (int64_t)b * Hkv + hk;
  const float c2 = kLog2e / sqrtf((float)HD);

  typename F::T qf[QT][STEPS];
  int sees[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = min(r0 + 16 * qt + col, nrows - 1), t = r / G;
    sees[qt] = past + t;
    const uint16_t* src = q + (((int64_t)b * T + t) * H + hk * G + (r - t * G)) * HD;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) qf[qt][s] = F::ld(src + 32 * s + 8 * kq);
  }
  f32x4 o[QT][HT];
  float m[QT], l[QT];  // l: this lane's share (16 of 64 keys)
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m[qt] = -INFINITY, l[qt] = 0.f;
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) o[qt][ht] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int own_keys = past + min(block * 128 + 127, nrows - 1) / G + 1;  // what the workgroup's rows see of the own keys
  const int all_see = past + min(r0, nrows - 1) / G;                      // the last own key that every row of this wave sees
  const int wave_last = past + min(r0 + 31, nrows - 1) / G;               // ... that any does
  const int tiles_p = (P + KT - 1) / KT, all_tiles = tiles_p + (own_keys + KT - 1) / KT;
  // this workgroup's run of tiles
  const int each = all_tiles / parts, rest = all_tiles - each * parts;
  const int first_tile = part * each + min(part, rest), tiles = first_tile + each + (part < rest ? 1 : 0);

  const unsigned char* const head_k[2] = {(const unsigned char*)(kp + hk * Pmax * HD), (const unsigned char*)(kc + bh * Lmax * HD)};
  const unsigned char* const head_v[2] = {(const unsigned char*)(vp + hk * Pmax * HD), (const unsigned char*)(vc + bh * Lmax * HD)};
  auto v_swz = [](int key) { return HD == 128 ? (key & 7) : ((key >> 1) & 3); };
  int k_row[STEPS], k_in[STEPS], v_row[STEPS], v_in[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    k_row[i] = 16 * wave + col;
    k_in[i] = (4 * i + kq) * 16;
    const int slot = (wave * STEPS + i) * 64 + lane, row = slot / CPR, pos = slot % CPR;
    v_row[i] = row;
    v_in[i] = ((((pos >> 1) ^ v_swz(row)) << 1) | (pos & 1)) * 16;
  }
  const float* const bias_row = key_bias ? key_bias + (int64_t)b * bias_stride : nullptr;
  float rbias = 0.f;
  auto fetch = [&](int tile, int buf) {
    const int own = tile >= tiles_p, k0 = (own ? tile - tiles_p : tile) * KT, left = (own ? own_keys : P) - 1 - k0;
    const __amdgpu_buffer_rsrc_t rk = make_rsrc(head_k[own] + (int64_t)k0 * VROW, min(left + 1, KT) * VROW);
    const __amdgpu_buffer_rsrc_t rv = make_rsrc(head_v[own] + (int64_t)k0 * VROW, min(left + 1, KT) * VROW);
    chain_request_tile(rk, rv, lds_k + buf * TILE + wave * (STEPS << 10), lds_v + buf * TILE + wave * (STEPS << 10), k_row, k_in,
                              v_row, v_in, left);
    if (tid < KT) rbias = own && bias_row ? bias_row[k0 + min(tid, left)] : 0.f;
  };
  auto publish = [&](int buf) {  // own requests landed, then everybody's
    if (tid < KT) lds_bias[buf * KT + tid] = rbias;
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, true));
    __builtin_amdgcn_s_barrier();
  };
  int v_rd[HT];  // this lane's row of the transposing loads
#pragma unroll
  for (int ht = 0; ht < HT; ++ht) v_rd[ht] = (4 * kq + (col >> 2)) * VROW + ((ht ^ v_swz(4 * kq + (col >> 2))) << 5) + 8 * (col & 3);

  if (first_tile < tiles) {  // the first rows of a long prompt see fewer tiles than there are parts: such a part has no tile to ask for
    fetch(first_tile, 0);
    publish(0);
  }
  int buf = 0;
  for (int tile = first_tile; tile < tiles; ++tile, buf ^= 1) {
    if (tile + 1 < tiles) fetch(tile + 1, buf ^ 1);  // read during the tile before, and everybody is past that tile's barrier
    const bool own = tile >= tiles_p;
    const int k0 = (own ? tile - tiles_p : tile) * KT;
    if (!own || k0 <= wave_last) {  // else no row of this wave sees the tile (the barriers stay uniform)
      const u32x4* kt_ = reinterpret_cast<const u32x4*>(lds_k + buf * TILE);
      const unsigned char* vt_ = lds_v + buf * TILE;
      const float* bias_ = lds_bias + buf * KT;
      // ---- S^T = K . Q^T: all fragments asked for before the first product
      f32x4 s[QT][4];
      u32x4 kf[4 * STEPS];
#pragma unroll
      for (int i = 0; i < 4 * STEPS; ++i) kf[i] = kt_[i * 64 + lane];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int st = 0; st < STEPS; ++st)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
            s[qt][kt] = F::mma(__builtin_bit_cast(typename F::T, kf[kt * STEPS + st]), qf[qt][st], st == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[qt][kt]);
      // ---- softmax, in the log2 domain: only tiles that hide keys or carry a bias look at their keys one by one
      const bool biased = own && bias_row, hides = own ? k0 + KT - 1 > all_see : k0 + KT > P;
      const float cs = biased || hides ? 1.f : c2;
      uint32_t keep[2][4];  // which of a lane's keys count, a half word each
      if (biased || hides) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = kt * 16 + 4 * kq + r;
            const float bias = bias_[key];
            const bool masked = bias <= kRowsMaskThreshold;
            const uint32_t half = masked ? 0u : 0xffffu;
            if ((r & 1) == 0) keep[kt >> 1][2 * (kt & 1) + (r >> 1)] = half;
            else keep[kt >> 1][2 * (kt & 1) + (r >> 1)] |= half << 16;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
              const float v = __builtin_fmaf(s[qt][kt][r], c2, bias * kLog2e);
              const bool out_of_sight = k0 + key > (own ? sees[qt] : P - 1);
              s[qt][kt][r] = masked || out_of_sight ? -INFINITY : v;
            }
          }
      }
      // fp16 weights keep 22 bits, as in attn_rows.h (olmo355_attn_prefill has them in fp32; 8 x 250 tokens, 32 heads, prefix 2048
      // 110 us, 82 with weights of 11 bits); bf16 weights are rounded once (8 bits), as olmo355_attn_prefill has them
      typename F::T pf[QT][2], pl[QT][2];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        float tmax = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) tmax = fmaxf(tmax, s[qt][kt][r]);
        tmax *= cs;
        if (__builtin_amdgcn_ballot_w64(tmax > m[qt] + kRowsLazyMax) != 0) {
          tmax = combine_xor32(combine_xor16(tmax, MaxOp{}), MaxOp{});
          const float mn = tmax > m[qt] + kRowsLazyMax ? tmax : m[qt];
          const float alpha = mn == m[qt] ? 1.f : __builtin_amdgcn_exp2f(m[qt] - mn);
          l[qt] *= alpha;
#pragma unroll
          for (int ht = 0; ht < HT; ++ht)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[qt][ht][r] *= alpha;
          m[qt] = mn;
        }
        const float mref = (m[qt] == -INFINITY ? 0.f : m[qt]) - kWeightTop<DT>;  // 0: a row that has seen no key yet
        float p[4][4], psum = 0.f;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[qt][kt][r], cs, -mref));
            psum += p[kt][r];
          }
        l[qt] += psum;
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          float f[8] = {p[2 * s2][0], p[2 * s2][1], p[2 * s2][2], p[2 * s2][3], p[2 * s2 + 1][0], p[2 * s2 + 1][1], p[2 * s2 + 1][2], p[2 * s2 + 1][3]};
          pf[qt][s2] = F::pack(f);
          if constexpr (REST) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = F::rest(f[i]);
            pl[qt][s2] = F::pack(f);
          }
        }
      }
      // ---- O^T += V^T . P^T
      u32x4 vf[HT][2];
#pragma unroll
      for (int ht = 0; ht < HT; ++ht)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          typedef short s16x4 __attribute__((ext_vector_type(4)));
          typedef s16x4 __attribute__((address_space(3))) * tr_ptr;
          typedef short s16x8 __attribute__((ext_vector_type(8)));
          const unsigned char* vp_ = vt_ + v_rd[ht] + (32 * s2) * VROW;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)vp_);
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(vp_ + 16 * VROW));
          vf[ht][s2] = __builtin_bit_cast(u32x4, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
        }
      __builtin_amdgcn_sched_barrier(0);
      if (biased) {  // a masked key weighs nothing, whatever its values hold
#pragma unroll
        for (int ht = 0; ht < HT; ++ht)
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int i = 0; i < 4; ++i) vf[ht][s2][i] &= keep[s2][i];
      }
#pragma unroll
      for (int ht = 0; ht < HT; ++ht)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            o[qt][ht] = F::mma(__builtin_bit_cast(typename F::T, vf[ht][s2]), pf[qt][s2], o[qt][ht]);
            if constexpr (REST) o[qt][ht] = F::mma(__builtin_bit_cast(typename F::T, vf[ht][s2]), pl[qt][s2], o[qt][ht]);
          }
    }
    publish(buf ^ 1);  // the next tile is in LDS and this one has been read by everybody
  }
  // ---- a lane holds channels 16 ht + 4 kq .. + 3 of its query column: out[row][hd], or this run's partial result
  const int64_t rows = (int64_t)gridDim.z * T * H;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float lsum = combine_xor32(combine_xor16(l[qt], AddOp{}), AddOp{});
    const int r = r0 + 16 * qt + col;
    if (r >= nrows) continue;
    const int t = r / G;
    const int64_t at = ((int64_t)b * T + t) * H + hk * G + (r - t * G);
    if (parts == 1) {
      const float inv = 1.f / lsum;
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
        const float f[4] = {o[qt][ht][0] * inv, o[qt][ht][1] * inv, o[qt][ht][2] * inv, o[qt][ht][3] * inv};
        st_row<DT, 4>(out, at * HD + 4 * kq + 16 * ht, f);
      }
    } else {
      float* dst = ws + (part * rows + at) * HD + 4 * kq;
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) *reinterpret_cast<f32x4*>(dst + 16 * ht) = o[qt][ht];
      if (kq == 0) *reinterpret_cast<f32x2*>(ws + rows * parts * HD + (part * rows + at) * 2) = f32x2{m[qt], lsum};
    }
  }
}

// Which form a call takes: the one-pass form where a sequence has rows to fill a good part of a workgroup's 128; the split
// form (any type, head size and count of rows) elsewhere.  Measured, 32 heads of 128, prefix 2048, us split / one pass, bf16:
// 8 x 16 tokens 31 / 47, 32 x 16 81 / 150, 8 x 32 62 / 48, 16 x 32 77 / 77, 8 x 64 76 / 53, 16 x 100 behind 100 keys 66 / 19.
// fp16, whose one-pass form has a second product: 16 x 32 78 / 108, 16 x 48 95 / 110, 4 x 56 35 / 41, 8 x 64 76 / 69,
// 16 x 64 121 / 110, 16 x 100 behind 100 keys 66 / 22.
// Parts: with fewer workgroups than two per CU the keys are shared too, at least four tiles of 64 to a workgroup
// (eight: 1 x 64 tokens 23.3 us against 19.7, 2 x 40 tokens behind 517 keys 20.2 against 16.6).
int prefix_chain_parts(int B, int T, int H, int Hkv, int hd, int P, int n_keys_max, int dtype) {
  const int64_t rows = (int64_t)T * (H / Hkv), blocks = (rows + 127) / 128, wgs = blocks * B * Hkv;
  if (dtype == O355_F32 || hd == 32 || T == 1 || rows < (dtype == O355_F16 ? 64 : 32)) return 0;
  const int64_t most = ((P + 63ll) / 64 + (n_keys_max + 63ll) / 64) / 4, want = 512 / wgs;
  const int64_t parts = want < 1 || most < 1 ? 1 : want > most ? most : want;
  return B <= 65535 && Hkv <= 65535 && blocks * parts <= 65535 ? (int)parts : 0;  // grid limits
}

template <int DT, int HD>
int launch_prefix_chain(const void* q, const void* kp, const void* vp, const void* kc, const void* vc, const float* key_bias, void* out,
                        float* ws, int B, int T, int H, int Hkv, int P, int64_t Pmax, int64_t Lmax, int past_len, int bias_stride,
                        int parts, hipStream_t s) {
  const int G = H / Hkv;
  const int64_t rows = (int64_t)T * G, all_rows = (int64_t)B * T * H;
  if ((all_rows + 3) / 4 > 0x7fffffff) return O355_EUNSUPPORTED;
  auto kern = attn_prefix_chain_kernel<DT, HD>;
  constexpr int lds = ChainLds<HD>::BYTES;  // more than a launch gets without asking
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
    return O355_ELAUNCH;
  hipLaunchKernelGGL(kern, dim3(Hkv, (unsigned)((rows + 127) / 128 * parts), B), dim3(256), lds, s, (const uint16_t*)q, (const uint16_t*)kp,
                     (const uint16_t*)vp, (const uint16_t*)kc, (const uint16_t*)vc, key_bias, (uint16_t*)out, ws, T, G, Hkv, P, Pmax,
                     Lmax, past_len, bias_stride, parts);
  if (parts > 1)
    hipLaunchKernelGGL((rows_combine_kernel<DT, HD>), dim3((unsigned)((all_rows + 3) / 4)), dim3(256), 0, s, (const float*)ws, out,
                       all_rows, parts);
  O355_CHECK_LAUNCH();
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int DT, int HD>
int launch_shared_prefix(const void* q, const void* kp, const void* vp, const void* kc, const void* vc, const float* key_bias, void* out,
                         float* ws, int B, int T, int H, int Hkv, int P, int64_t Pmax, int64_t Lmax, int past_len,
                         const int32_t* past_dev, int n_keys_max, int bias_stride, const PrefixPlan& plan, hipStream_t s) {
  const int64_t wgs = plan.wgs_p + plan.wgs_o, rows = (int64_t)B * T * H;
  if (wgs > 0x7fffffff || (rows + 3) / 4 > 0x7fffffff || Hkv > 65535) return O355_EUNSUPPORTED;  // grid limits
  const dim3 grid((unsigned)wgs, Hkv);
#define RUN(RTP, RTO)                                                                                                              \
  hipLaunchKernelGGL((attn_shared_prefix_kernel<DT, HD, RTP, RTO>), grid, dim3(256), 0, s, q, kp, vp, kc, vc, key_bias, \
                     ws, B, T, H / Hkv, Hkv, P, Pmax, Lmax, past_len, past_dev, n_keys_max, bias_stride, plan)
  if (plan.rtp == 1) RUN(1, 1);
  else if (plan.rtp == 2 && plan.rto == 1) RUN(2, 1);
  else RUN(2, 2);
#undef RUN
  hipLaunchKernelGGL((rows_combine_kernel<DT, HD>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, (const float*)ws, out, rows,
                     plan.splits_p + plan.splits_o);
  O355_CHECK_LAUNCH();
}

bool prefix_shape_ok(int B, int T, int H, int Hkv, int prefix_len, int n_keys_max) {
  return B > 0 && T > 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && prefix_len > 0 && n_keys_max >= T &&
         (int64_t)B * T * (H / Hkv) <= 0x7fffff00ll;
}

}  // namespace

extern "C" int64_t olmo355_attn_shared_prefix_workspace_bytes(int B, int T, int H, int Hkv, int hd, int prefix_len, int n_keys_max,
                                                              int dtype) {
  if (!prefix_shape_ok(B, T, H, Hkv, prefix_len, n_keys_max) || hd <= 0) return 0;
  if (const int parts = prefix_chain_parts(B, T, H, Hkv, hd, prefix_len, n_keys_max, dtype))
    return parts == 1 ? 0 : 4 * rows_parts_floats((int64_t)B * T * H, hd, parts);
  const PrefixPlan p = prefix_plan(B, T, H, Hkv, prefix_len, n_keys_max, true);
  return 4 * rows_parts_floats((int64_t)B * T * H, hd, p.most);
}

extern "C" int olmo355_attn_shared_prefix(const void* q, const void* kprefix, const void* vprefix, const void* kcache, const void* vcache,
                                          const float* key_bias, void* out, void* ws, int64_t ws_bytes, int B, int T, int H, int Hkv,
                                          int hd, int prefix_len, int Pmax, int Lmax, int past_len, const int32_t* past_len_dev,
                                          int n_keys_max, int bias_stride, int dtype, void* stream) {
  if (!q || !kprefix || !vprefix || !kcache || !vcache || !out) return O355_EINVAL;
  if (!prefix_shape_ok(B, T, H, Hkv, prefix_len, n_keys_max)) return O355_EINVAL;
  if (prefix_len > Pmax || n_keys_max > Lmax || past_len < 0) return O355_EINVAL;
  if (!past_len_dev && (int64_t)past_len + T > n_keys_max) return O355_EINVAL;
  if (key_bias && bias_stride < n_keys_max) return O355_EINVAL;
  for (const void* p : {q, kprefix, vprefix, kcache, vcache, (const void*)out, (const void*)ws})
    if (!aligned16(p)) return O355_EINVAL;
  if (past_len_dev && T != 1) return O355_EUNSUPPORTED;
  if (hd != 32 && hd != 64 && hd != 128) return O355_EUNSUPPORTED;
  if (dtype != O355_F32 && dtype != O355_BF16 && dtype != O355_F16) return O355_EUNSUPPORTED;
  const int64_t need = olmo355_attn_shared_prefix_workspace_bytes(B, T, H, Hkv, hd, prefix_len, n_keys_max, dtype);
  if (need && (!ws || ws_bytes < need)) return O355_EINVAL;
  if (const int parts = prefix_chain_parts(B, T, H, Hkv, hd, prefix_len, n_keys_max, dtype)) {
#define CHAIN(DTv, HDv)                                                                                                            \
  return launch_prefix_chain<DTv, HDv>(q, kprefix, vprefix, kcache, vcache, key_bias, out, (float*)ws, B, T, H, Hkv, prefix_len,    \
                                       Pmax, Lmax, past_len, bias_stride, parts, as_stream(stream))
    if (dtype == O355_BF16 && hd == 128) CHAIN(O355_BF16, 128);
    if (dtype == O355_BF16) CHAIN(O355_BF16, 64);
    if (hd == 128) CHAIN(O355_F16, 128);
    CHAIN(O355_F16, 64);
#undef CHAIN
  }
  const PrefixPlan plan = prefix_plan(B, T, H, Hkv, prefix_len, n_keys_max, !past_len_dev && past_len + T == n_keys_max);
#define PREFIX(DTv, HDv)                                                                                                           \
  return launch_shared_prefix<DTv, HDv>(q, kprefix, vprefix, kcache, vcache, key_bias, out, (float*)ws, B, T, H, Hkv, prefix_len,   \
                                        Pmax, Lmax, past_len, past_len_dev, n_keys_max, bias_stride, plan, as_stream(stream))
#define PREFIX_HD(DTv)             \
  do {                             \
    if (hd == 128) PREFIX(DTv, 128); \
    if (hd == 64) PREFIX(DTv, 64); \
    PREFIX(DTv, 32);               \
  } while (0)
  if (dtype == O355_F32) PREFIX_HD(O355_F32);
  if (dtype == O355_BF16) PREFIX_HD(O355_BF16);
  PREFIX_HD(O355_F16);
#undef PREFIX_HD
#undef PREFIX
}
