// The key/value cache in 8 bits: written together with the QK-norm and the rotation, read back, and attended to by the
// one new token of a decode step.
//
// A cached row (one token, one kv head, hd channels) is hd signed codes and one fp32 scale:
//   scale = max(max |x| / 127, FLT_MIN),  code = rint(x / scale) in -127 .. 127,  x ~ code * scale
// (the lower bound keeps the reciprocal finite; a row of zeros has codes 0).  The row's own maximum makes the error at most
// half a step of max / 127 whatever the row's size.  A row that holds an infinity or a NaN gets the scale NaN and codes 0:
// it reads back as NaN, and attention gives NaN unless the key is masked.
// Layout: codes int8 [B, Hkv, Lmax, hd], scales fp32 [B, Hkv, Lmax], keys rotated as in the unquantised cache.
#include "attn_rows.h"

namespace {

// eight activations: as they lie in memory (16 bytes of a 16-bit type, 32 of fp32), as floats, and back
template <int DT>
struct Raw8 {
  u32x4 w[DT == O355_F32 ? 2 : 1];
  __device__ __forceinline__ void ld(const void* p, int64_t e) {
    if constexpr (DT == O355_F32) {
      w[0] = reinterpret_cast<const u32x4*>((const float*)p + e)[0], w[1] = reinterpret_cast<const u32x4*>((const float*)p + e)[1];
    } else {
      w[0] = *reinterpret_cast<const u32x4*>((const uint16_t*)p + e);
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (DT == O355_F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[0][i]), f[4 + i] = __uint_as_float(w[1][i]);
    } else if constexpr (DT == O355_BF16) {
      unpack8(w[0], f);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)w[0][i]);
        f[2 * i] = (float)h[0], f[2 * i + 1] = (float)h[1];
      }
    }
  }
};
template <int DT>
__device__ __forceinline__ void ld8f(const void* p, int64_t e, float (&f)[8]) {
  Raw8<DT> r;
  r.ld(p, e);
  r.get(f);
}
template <int DT>
__device__ __forceinline__ void st8f(void* p, int64_t e, const float (&f)[8]) {
  if constexpr (DT == O355_F32) {
    reinterpret_cast<f32x4*>((float*)p + e)[0] = f32x4{f[0], f[1], f[2], f[3]};
    reinterpret_cast<f32x4*>((float*)p + e)[1] = f32x4{f[4], f[5], f[6], f[7]};
  } else if constexpr (DT == O355_BF16) {
    *reinterpret_cast<u32x4*>((uint16_t*)p + e) =
        u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
  } else {
    *reinterpret_cast<u32x4*>((uint16_t*)p + e) =
        u32x4{pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]), pack_f16x2(f[6], f[7])};
  }
}

// ---- write ----------------------------------------------------------------------------------------------------
// Part 0 normalises and rotates q, part 1 k, part 2 takes v: the sum of squares of q and of k are over the whole width
// (olmo/model.py:603-605), so whoever takes a part needs one of them and reads nothing twice.  A row's part is a workgroup's
// (WPR 4; grid (token rows, part)) or q_lanes / kv_lanes lanes' of a wave (WPR 1: no barrier; a wave takes as many rows as
// its 64 lanes hold; grid: part after part).  A lane owns channels j .. j + 7 of the first half of a head and the 8 they
// rotate with, CPT such pairs, which stay in registers as they were loaded; hd / 16 neighbouring lanes hold a head, whose
// maximum is a few register exchanges.  fp32 from the input to the code (q: to its one rounding).
template <int DT, int HD, int CPT, int WPR>
__global__ __launch_bounds__(256) void kv_write_q8_kernel(const void* __restrict__ qkv, const void* __restrict__ qw,
                                                          const void* __restrict__ kw, const float* __restrict__ sin_t,
                                                          const float* __restrict__ cos_t, void* __restrict__ q_out,
                                                          int8_t* __restrict__ kq, int8_t* __restrict__ vq, float* __restrict__ ks,
                                                          float* __restrict__ vs, void* __restrict__ kc, void* __restrict__ vc, int Lfull,
                                                          uint32_t rows, uint32_t T, int H, int Hkv, int Lmax, int n_pos, int past_len,
                                                          const int32_t* __restrict__ past_dev, float eps, int q_lanes, int kv_lanes,
                                                          uint32_t q_blocks, uint32_t kv_blocks) {
  constexpr int CPH = HD / 16, HALF = HD / 2, LANES = 64 * WPR;
  __shared__ float red[16];
  int part = blockIdx.y, me = threadIdx.x, lanes = LANES;
  uint32_t row = blockIdx.x;
  if constexpr (WPR == 1) {
    part = blockIdx.x < q_blocks ? 0 : blockIdx.x < q_blocks + kv_blocks ? 1 : 2;
    lanes = part == 0 ? q_lanes : kv_lanes;  // a power of two; below 64 only where it holds the whole row
    const uint32_t block = part == 0 ? blockIdx.x : blockIdx.x - q_blocks - (part - 1) * kv_blocks;
    row = block * (256u / (uint32_t)lanes) + (uint32_t)threadIdx.x / (uint32_t)lanes;
    me = threadIdx.x & (lanes - 1);
  }
  if (row >= rows) return;  // WPR 1: all lanes of a row
  const uint32_t b = row / T, t = row - b * T;
  const int dq = H * HD, dk = Hkv * HD;
  const int pos = (past_dev ? *past_dev : past_len) + (int)t;
  if (pos < 0 || pos >= Lmax || pos >= n_pos) return;  // a device-side position outside the cache: write nothing
  const int heads = part == 0 ? H : Hkv, n = heads * CPH;
  const int64_t in = (int64_t)row * (dq + 2 * dk) + (part == 0 ? 0 : part == 1 ? dq : dq + dk);
  const void* w = part == 0 ? qw : part == 1 ? kw : nullptr;
  Raw8<DT> x1[CPT], x2[CPT];
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    const int c = me + i * LANES;
    if (c < n) {
      const int64_t e = in + (c / CPH) * HD + (c % CPH) * 8;
      x1[i].ld(qkv, e);
      x2[i].ld(qkv, e + HALF);
    }
  }
  float rstd = 1.f;
  if (w) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < CPT; ++i)
      if (me + i * LANES < n) {
        float a[8], bb[8];
        x1[i].get(a), x2[i].get(bb);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + bb[e] * bb[e];
      }
    if constexpr (WPR == 1) {
      if (lanes == 64) ss = wave_sum(ss);
      else
        for (int o = lanes >> 1; o; o >>= 1) ss += __shfl_xor(ss, o, 64);
    } else {
      ss = block_sum(ss, red);
    }
    rstd = 1.f / sqrtf(ss / (float)(heads * HD) + eps);
  }
  const float* sn = sin_t + (int64_t)pos * HD;
  const float* cs = cos_t + (int64_t)pos * HD;
  const int j = (me % CPH) * 8;  // LANES is a multiple of CPH: the same channels of a head in every pair
  float c1[8], c2[8], s1[8], s2[8];
  if (part < 2) ld8f<O355_F32>(cs, j, c1), ld8f<O355_F32>(cs, j + HALF, c2), ld8f<O355_F32>(sn, j, s1), ld8f<O355_F32>(sn, j + HALF, s2);
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    const int c = me + i * LANES;
    if (c >= n) break;  // the lanes of a head leave together
    const int h = c / CPH;
    float a[8], bb[8];
    x1[i].get(a), x2[i].get(bb);
    if (w) {
      float w1[8], w2[8];
      ld8f<DT>(w, h * HD + j, w1);
      ld8f<DT>(w, h * HD + j + HALF, w2);
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = a[e] * rstd * w1[e], bb[e] = bb[e] * rstd * w2[e];
    }
    if (part < 2) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float u = a[e], v = bb[e];
        a[e] = u * c1[e] - v * s1[e];
        bb[e] = v * c2[e] + u * s2[e];
      }
    }
    if (part == 0) {
      st8f<DT>(q_out, (int64_t)row * dq + h * HD + j, a);
      st8f<DT>(q_out, (int64_t)row * dq + h * HD + j + HALF, bb);
      continue;
    }
    const int64_t bh = (int64_t)b * Hkv + h, at = bh * Lmax + pos;
    if (kc && pos < Lfull) {  // the row as the unquantised cache would hold it
      void* full = part == 1 ? kc : vc;
      const int64_t e = (bh * Lfull + pos) * HD + j;
      st8f<DT>(full, e, a);
      st8f<DT>(full, e + HALF, bb);
    }
    float amax = 0.f;
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = fabsf(a[e]), v = fabsf(bb[e]);
      finite = finite && u <= 3.4028234663852886e38f && v <= 3.4028234663852886e38f;
      amax = fmaxf(amax, fmaxf(u, v));
    }
    if (!finite) amax = INFINITY;
    amax = fmaxf(amax, dpp_lane<0xB1>(amax));                          // quad_perm [1,0,3,2]
    if constexpr (CPH >= 4) amax = fmaxf(amax, dpp_lane<0x4E>(amax));  // quad_perm [2,3,0,1]
    if constexpr (CPH >= 8) amax = fmaxf(amax, dpp_lane<0x141>(amax)); // row_half_mirror
    const bool ok = amax < INFINITY;
    const float scale = ok ? fmaxf(amax / 127.f, 1.1754943508222875e-38f) : __builtin_nanf("");
    // v / scale, correctly rounded, with one division a row: two refinements of v * (1 / scale) by its residual (P. Markstein: a
    // quotient within a unit of the last place, refined with the correctly rounded reciprocal and an exact residual, is the
    // rounded quotient).  `up` keeps the residuals of rows of tiny values exact.  v * (1 / scale) alone moves codes next to a
    // tie (a 16-bit value of half the row's maximum is at one); 8168 rows of 40 heads take 96 us with it, 103 so, 110 with a
    // division per value.
    const float up = scale < 0x1p-96f ? 0x1p96f : 1.f, s = scale * up, inv = 1.f / s;
    auto code = [&](float v) {
      v *= up;
      float t = v * inv;
      t = __builtin_fmaf(__builtin_fmaf(-t, s, v), inv, t);
      t = __builtin_fmaf(__builtin_fmaf(-t, s, v), inv, t);
      return ok ? (uint32_t)(uint8_t)(int8_t)(int)rintf(t) : 0u;
    };
    u32x2 p1, p2;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      p1[g] = code(a[4 * g]) | code(a[4 * g + 1]) << 8 | code(a[4 * g + 2]) << 16 | code(a[4 * g + 3]) << 24;
      p2[g] = code(bb[4 * g]) | code(bb[4 * g + 1]) << 8 | code(bb[4 * g + 2]) << 16 | code(bb[4 * g + 3]) << 24;
    }
    int8_t* codes = part == 1 ? kq : vq;
    *reinterpret_cast<u32x2*>(codes + at * HD + j) = p1;
    *reinterpret_cast<u32x2*>(codes + at * HD + j + HALF) = p2;
    if (j == 0) (part == 1 ? ks : vs)[at] = scale;
  }
}

// ---- read back --------------------------------------------------------------------------------------------------
// A thread turns 16 codes into 16 values; grid.y 0: keys, 1: values.
template <int DT, int HD>
__global__ __launch_bounds__(256) void kv_read_q8_kernel(const int8_t* __restrict__ kq, const int8_t* __restrict__ vq,
                                                         const float* __restrict__ ks, const float* __restrict__ vs,
                                                         void* __restrict__ kout, void* __restrict__ vout, int64_t pieces, int n,
                                                         int Lmax, int start, int Lout, int out_start) {
  constexpr int PPR = HD / 16;  // pieces per row
  const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (p >= pieces) return;
  const int8_t* codes = blockIdx.y ? vq : kq;
  const float* scales = blockIdx.y ? vs : ks;
  const int64_t r = p / PPR, bh = r / n, t = r - bh * n;
  const int c = (int)(p - r * PPR) * 16;
  const int64_t src = bh * Lmax + start + t, dst = (bh * Lout + out_start + t) * HD + c;
  const u32x4 w = *reinterpret_cast<const u32x4*>(codes + src * HD + c);
  const float s = scales[src];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(w[2 * g + (e >> 2)] >> (8 * (e & 3))) * s;
    st8f<DT>(blockIdx.y ? vout : kout, dst + 8 * g, f);
  }
}

// ---- decode attention over the codes ------------------------------------------------------------------------------
// Grid: (16 query heads of the group x run of keys, kv head, sequence).  See attn_rows.h for what a workgroup does.
template <int DT, int HD>
__global__ __launch_bounds__(256, 2) void attn_decode_q8_kernel(const void* __restrict__ q, const int8_t* __restrict__ kq,
                                                                const int8_t* __restrict__ vq, const float* __restrict__ ks,
                                                                const float* __restrict__ vs, const float* __restrict__ key_bias,
                                                                void* __restrict__ out, float* __restrict__ ws, int G, int Hkv,
                                                                int Lmax, int past_len, const int32_t* __restrict__ past_dev,
                                                                int n_keys_max, int bias_stride, int splits, int64_t rows) {
  __shared__ RowsLds<HD> lds;
  const uint32_t tile = blockIdx.x / (uint32_t)splits, split = blockIdx.x - tile * splits;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int64_t bh = (int64_t)b * Hkv + hk;
  const int keys = max(1, min((past_dev ? *past_dev : past_len) + 1, n_keys_max));
  RowsIn in;
  in.q = (const unsigned char*)q, in.tok0 = b, in.G = G, in.H = Hkv * G, in.head0 = hk * G;
  in.r0 = 16 * tile, in.nrows = min(G, in.r0 + 16);
  in.k = (const unsigned char*)kq + bh * Lmax * HD, in.v = (const unsigned char*)vq + bh * Lmax * HD;
  in.ks = ks + bh * Lmax, in.vs = vs + bh * Lmax;
  in.bias = key_bias ? key_bias + (int64_t)b * bias_stride : nullptr;
  in.keys = keys, in.past = -1;
  const Run run = run_of((uint32_t)(keys + 31) / 32, split, splits);
  RowsAcc<HD, 1> acc;
  walk_keys<DT, HD, 1, true, Q8Keys<DT, HD>>(in, run.lo + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), run.hi, 4, acc);
  merge_waves<HD, 1>(in, acc, lds, [&](int r, int c, auto& o, float m, float l) {
    constexpr int VC = HD / 16;
    const int64_t at = bh * G + r;
    if (splits == 1) {
      const float inv = 1.f / l;
#pragma unroll
      for (int j = 0; j < VC; ++j) o[j] *= inv;
      st_row<DT, VC>(out, at * HD + c, o);
    } else {
      st_row<O355_F32, VC>(ws, (split * rows + at) * HD + c, o);
      if (c == 0) {
        float* ml = ws + rows * splits * HD + (split * rows + at) * 2;
        ml[0] = m, ml[1] = l;
      }
    }
  });
}

// Runs of keys per (sequence, kv head, row tile), at least 128 keys each (one step per wave). A round of one workgroup per CU,
// no more, is best where it keeps the CUs busy: 4 x 4096 keys, 32 heads, 28.8 us with 256 workgroups, 29.4 with 512;
// 1 x 4096 12.4 against 13.0; 8 x 2048 26.0 against 29.0; 32 x 1000, 8 kv heads, 13.9 against 17.6 (one run each, no merge).
// Where the last round would leave a quarter of the CUs idle, long keys are cut finer, into as many runs as four workgroups per
// CU take: 9 x 4096, 32 heads, 74.8 us in whole runs, 63.6 in 3; 13 x 8000, 10 kv heads, 72 in whole runs, 58 in 3, 55 in the 7
// it takes. Up to 2048 keys that would cost more than it brings (5 x 2000, 32 heads, 19.0 in whole runs, 20.2 in 3). So beyond
// 128 (sequence, kv head, row tile) units keys stay whole, but for more than 2048 keys of 129-192 or 257-384 units.
// Never fewer runs with more keys: a workspace for n serves fewer.
int decode_q8_splits(int B, int H, int Hkv, int n_keys_max) {
  const int64_t units = (int64_t)B * Hkv * ((H / Hkv + 15) / 16), cus = 256;
  const int64_t whole = units < cus ? cus / units : 1, rounds = (units * whole + cus - 1) / cus;
  const bool idle = 4 * units * whole <= 3 * rounds * cus && n_keys_max > 2048;
  const int64_t fine = 4 * cus / units, want = idle && fine > whole ? fine : whole, most = (n_keys_max + 127) / 128;
  return (int)(want > most ? most : want);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

#define Q8_SWITCH_HD(hd, DTv, CALL) \
  switch (hd) {                     \
    case 32: CALL(DTv, 32); break;  \
    case 64: CALL(DTv, 64); break;  \
    case 128: CALL(DTv, 128); break; \
    default: return O355_EUNSUPPORTED; \
  }
#define Q8_SWITCH(dtype, hd, CALL)                             \
  switch (dtype) {                                             \
    case O355_F32: Q8_SWITCH_HD(hd, O355_F32, CALL) break;     \
    case O355_BF16: Q8_SWITCH_HD(hd, O355_BF16, CALL) break;   \
    case O355_F16: Q8_SWITCH_HD(hd, O355_F16, CALL) break;     \
    default: return O355_EUNSUPPORTED;                         \
  }

extern "C" int olmo355_qknorm_rope_kvwrite_q8(const void* qkv, const void* qw, const void* kw, const float* sin_tab,
                                              const float* cos_tab, void* q_out, int8_t* kq, int8_t* vq, float* kscale,
                                              float* vscale, void* kcache, void* vcache, int Lfull, int B, int T, int H, int Hkv, int hd,
                                              int Lmax, int n_pos, int past_len, const int32_t* past_len_dev, float eps, int dtype,
                                              void* stream) {
  if (!qkv || !sin_tab || !cos_tab || !q_out || !kq || !vq || !kscale || !vscale) return O355_EINVAL;
  if (B <= 0 || T <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || Lmax <= 0 || n_pos <= 0 || past_len < 0) return O355_EINVAL;
  if ((qw == nullptr) != (kw == nullptr) || (kcache == nullptr) != (vcache == nullptr)) return O355_EINVAL;
  if (kcache && (Lfull <= 0 || (!past_len_dev && (int64_t)past_len + T > Lfull))) return O355_EINVAL;
  if (!past_len_dev && ((int64_t)past_len + T > Lmax || (int64_t)past_len + T > n_pos)) return O355_EINVAL;
  for (const void* p : {qkv, qw, kw, (const void*)sin_tab, (const void*)cos_tab, (const void*)q_out, (const void*)kq, (const void*)vq,
                        (const void*)kcache, (const void*)vcache})
    if (!aligned16(p)) return O355_EINVAL;
  if (past_len_dev && T != 1) return O355_EUNSUPPORTED;
  if (hd != 32 && hd != 64 && hd != 128) return O355_EUNSUPPORTED;
  const int64_t chunks = (int64_t)H * hd / 16;
  if (chunks > 1024 || (int64_t)B * T > 0x7fffffff) return O355_EUNSUPPORTED;
  hipStream_t s = as_stream(stream);
  const uint32_t rows = (uint32_t)B * T;
  // Few rows: a workgroup to a row's part, whose loads all go out at once (32 heads of 128, 1 row 4.0 us against 7.3 with a wave
  // to it, 2048 rows 20.9 against 22.3); many rows: a wave (40 heads, 8168 rows 103 against 106; 40 / 8 heads, 8192 rows 53
  // against 65), or as many lanes as the row has pairs: the count of waves is what short rows cost (8 heads of 32, 8000 rows
  // 8.5 us against 18 with a wave and 35 with a workgroup to each; 16 / 2 heads of 64, 102032 rows 114 against 206 and 412).
  // 8168 rows of 40 heads: 4.1 TB/s of the 4.8 that a large copy reaches.  (Replays of a graph of such calls.)
  auto lanes_for = [hd](int heads) {
    int n = 2;
    while (n < 64 && n < heads * (hd / 16)) n *= 2;
    return n;
  };
  const int q_lanes = lanes_for(H), kv_lanes = lanes_for(Hkv);
  auto blocks_for = [rows](int lanes) { return (uint32_t)(((int64_t)rows * lanes + 255) / 256); };
  const uint32_t q_blocks = blocks_for(q_lanes), kv_blocks = blocks_for(kv_lanes);
#define WRITE(DTv, HDv, CPT, WPR)                                                                                                  \
  hipLaunchKernelGGL((kv_write_q8_kernel<DTv, HDv, CPT, WPR>), WPR == 1 ? dim3(q_blocks + 2 * kv_blocks) : dim3(rows, 3), dim3(256), 0, \
                     s, qkv, qw, kw, sin_tab, cos_tab, q_out, kq, vq, kscale, vscale, kcache, vcache, Lfull, rows, (uint32_t)T, H,    \
                     Hkv, Lmax, n_pos, past_len, past_len_dev, eps, q_lanes, kv_lanes, q_blocks, kv_blocks)
#define WRITE_CPT(DTv, HDv)                            \
  do {                                                 \
    if (rows < 4096 && chunks > 128) {                 \
      if (chunks <= 256) WRITE(DTv, HDv, 1, 4);        \
      else if (chunks <= 512) WRITE(DTv, HDv, 2, 4);   \
      else WRITE(DTv, HDv, 4, 4);                      \
    } else if (chunks <= 64) WRITE(DTv, HDv, 1, 1);    \
    else if (chunks <= 128) WRITE(DTv, HDv, 2, 1);     \
    else if (chunks <= 256) WRITE(DTv, HDv, 4, 1);     \
    else if (chunks <= 512) WRITE(DTv, HDv, 8, 1);     \
    else WRITE(DTv, HDv, 4, 4);                        \
  } while (0)
  Q8_SWITCH(dtype, hd, WRITE_CPT)
#undef WRITE_CPT
#undef WRITE
  O355_CHECK_LAUNCH();
}

extern "C" int olmo355_kv_read_q8(const int8_t* kq, const int8_t* vq, const float* kscale, const float* vscale, void* kout, void* vout,
                                  int B, int Hkv, int hd, int Lmax, int start, int n, int Lout, int out_start, int dtype, void* stream) {
  if (!kq || !vq || !kscale || !vscale || !kout || !vout) return O355_EINVAL;
  if (B <= 0 || Hkv <= 0 || Lmax <= 0 || Lout <= 0 || start < 0 || n <= 0 || out_start < 0) return O355_EINVAL;
  if ((int64_t)start + n > Lmax || (int64_t)out_start + n > Lout) return O355_EINVAL;
  for (const void* p : {(const void*)kq, (const void*)vq, (const void*)kout, (const void*)vout})
    if (!aligned16(p)) return O355_EINVAL;
  if (hd != 32 && hd != 64 && hd != 128) return O355_EUNSUPPORTED;
  const int64_t pieces = (int64_t)B * Hkv * n * (hd / 16), blocks = (pieces + 255) / 256;
  if (blocks > 0x7fffffff) return O355_EUNSUPPORTED;
  hipStream_t s = as_stream(stream);
#define READ(DTv, HDv)                                                                                                            \
  hipLaunchKernelGGL((kv_read_q8_kernel<DTv, HDv>), dim3((unsigned)blocks, 2), dim3(256), 0, s, kq, vq, kscale, vscale, kout, vout, \
                     pieces, n, Lmax, start, Lout, out_start)
  Q8_SWITCH(dtype, hd, READ)
#undef READ
  O355_CHECK_LAUNCH();
}

extern "C" int64_t olmo355_attn_decode_q8_workspace_bytes(int B, int H, int Hkv, int hd, int n_keys_max) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || hd <= 0 || n_keys_max <= 0) return 0;
  const int splits = decode_q8_splits(B, H, Hkv, n_keys_max);
  return splits == 1 ? 0 : 4 * rows_parts_floats((int64_t)B * H, hd, splits);
}

extern "C" int olmo355_attn_decode_q8(const void* q, const int8_t* kq, const int8_t* vq, const float* kscale, const float* vscale,
                                      const float* key_bias, void* out, void* ws, int64_t ws_bytes, int B, int H, int Hkv, int hd,
                                      int Lmax, int past_len, const int32_t* past_len_dev, int n_keys_max, int bias_stride, int dtype,
                                      void* stream) {
  if (!q || !kq || !vq || !kscale || !vscale || !out) return O355_EINVAL;
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || past_len < 0 || n_keys_max <= 0 || n_keys_max > Lmax) return O355_EINVAL;
  if (!past_len_dev && past_len >= n_keys_max) return O355_EINVAL;
  if (key_bias && bias_stride < n_keys_max) return O355_EINVAL;
  for (const void* p : {q, (const void*)kq, (const void*)vq, (const void*)out, (const void*)ws})
    if (!aligned16(p)) return O355_EINVAL;
  if (hd != 32 && hd != 64 && hd != 128) return O355_EUNSUPPORTED;
  const int64_t need = olmo355_attn_decode_q8_workspace_bytes(B, H, Hkv, hd, n_keys_max);
  if (need && (!ws || ws_bytes < need)) return O355_EINVAL;
  const int tiles = (H / Hkv + 15) / 16, splits = decode_q8_splits(B, H, Hkv, n_keys_max);
  const int64_t rows = (int64_t)B * H;
  if (B > 65535 || Hkv > 65535) return O355_EUNSUPPORTED;  // grid limits
  const dim3 grid(tiles * splits, Hkv, B);
  hipStream_t s = as_stream(stream);
#define DECODE(DTv, HDv)                                                                                                          \
  hipLaunchKernelGGL((attn_decode_q8_kernel<DTv, HDv>), grid, dim3(256), 0, s, q, kq, vq, kscale, vscale, key_bias, out,             \
                     (float*)ws, H / Hkv, Hkv, Lmax, past_len, past_len_dev, n_keys_max, bias_stride, splits, rows);               \
  if (splits > 1)                                                                                                                 \
  hipLaunchKernelGGL((rows_combine_kernel<DTv, HDv>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, (const float*)ws, out,   \
                     rows, splits)
  Q8_SWITCH(dtype, hd, DECODE)
#undef DECODE
  O355_CHECK_LAUNCH();
}
