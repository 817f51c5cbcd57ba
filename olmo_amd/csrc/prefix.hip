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
  int64_t wgs_p, wgs_o;    // workgroups per kv head
};

PrefixPlan prefix_plan(int B, int T, int H, int Hkv, int P, int n_keys_max, int dtype) {
  PrefixPlan p;
  const int64_t G = H / Hkv, rows_o = T * G, rows_p = B * rows_o;
  const int most = dtype == O355_F32 ? 2 : 4;  // fp32 operands are twice as wide
  p.rtp = rows_p <= 16 ? 1 : rows_p <= 32 ? 2 : most;
  p.rto = rows_o <= 16 ? 1 : p.rtp;
  p.tiles_p = (int)((rows_p + 16 * p.rtp - 1) / (16 * p.rtp));
  p.tiles_o = (int)((rows_o + 16 * p.rto - 1) / (16 * p.rto));
  auto splits = [](int64_t units, int keys, int target) {  // at least 128 keys per workgroup
    const int64_t most = (keys + 127) / 128, want = (target + units - 1) / units;
    return (int)(want < 1 ? 1 : want > most ? most : want);
  };
  p.splits_p = splits((int64_t)Hkv * p.tiles_p, P, 512);
  p.splits_o = splits((int64_t)B * Hkv * p.tiles_o, n_keys_max, 512);
  p.wgs_p = (int64_t)p.tiles_p * p.splits_p;
  p.wgs_o = (int64_t)B * p.tiles_o * p.splits_o;
  return p;
}

template <int DT, int HD, int RTP, int RTO>
__global__ __launch_bounds__(256, (RTP <= 2 && (DT != O355_F32 || HD < 128) ? 2 : 1)) void attn_shared_prefix_kernel(
    const void* __restrict__ q, const void* __restrict__ kp, const void* __restrict__ vp, const void* __restrict__ kc,
    const void* __restrict__ vc, const float* __restrict__ key_bias, float* __restrict__ ws, int B, int T, int G, int Hkv, int P,
    int64_t Pmax, int64_t Lmax, int past_len, const int32_t* __restrict__ past_dev, int n_keys_max, int bias_stride, PrefixPlan plan) {
  constexpr int ES = DT == O355_F32 ? 4 : 2, VC = HD / 16;
  __shared__ RowsLds<HD> lds;
  const int H = Hkv * G;
  const int64_t rows = (int64_t)B * T * H;
  const int parts = plan.splits_p + plan.splits_o;
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
    const uint32_t tile = i / (uint32_t)plan.splits_p;
    part = (int)(i - tile * plan.splits_p);
    in.tok0 = 0, in.head0 = hk * G;
    in.r0 = tile * 16 * RTP, in.nrows = B * T * G;
    in.k = (const unsigned char*)kp + hk * Pmax * HD * ES, in.v = (const unsigned char*)vp + hk * Pmax * HD * ES;
    in.bias = nullptr, in.keys = P, in.past = -1;
    share_steps(in, (uint32_t)(P + 31) / 32, part, plan.splits_p);
    attend_rows<DT, HD, RTP, false, RawKeys<DT, HD>>(in, lds, emit);
    return;
  }
  i -= (uint32_t)plan.wgs_p;
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
  share_steps(in, (uint32_t)(last + 32) / 32, split, plan.splits_o);
  attend_rows<DT, HD, RTO, false, RawKeys<DT, HD>>(in, lds, emit);
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
  else if (plan.rtp == 2) RUN(2, 2);
  else if constexpr (DT != O355_F32) {
    if (plan.rto == 1) RUN(4, 1);
    else RUN(4, 4);
  }
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
  const PrefixPlan p = prefix_plan(B, T, H, Hkv, prefix_len, n_keys_max, dtype);
  return 4 * rows_parts_floats((int64_t)B * T * H, hd, p.splits_p + p.splits_o);
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
  const PrefixPlan plan = prefix_plan(B, T, H, Hkv, prefix_len, n_keys_max, dtype);
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
