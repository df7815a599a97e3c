// Decode over a KV cache that also adds the attention weights to the keys'
// running totals, on gfx950.
//
// As kat_attn_decode (attn_decode.hip), for one query per (batch, head) against
// n = lengths[b] cached rows, the query in row n - 1, with p_j the rows'
// positions (their index, or given: the rows of an evicted cache):
//   s_j = scale <q, k_j> - slope_h (p_{n-1} - p_j),  f_j = sigma(s_j)^4
//   L = sum_j f_j,  o = sum_j f_j v_j / (L + eps)
//   total_j += f_j / (L + eps)   (j < n)
//
// Design: HBM bounds it (2 D dtype bytes per row and 8 for its total). Where the
// (b, h) fill the chip, or their rows are few, a block takes all rows of one, keeps
// the f in LDS and finishes o, L and the totals itself. Else the decode's split over
// the rows: L is known only after every chunk, so the chunks leave their f in the
// workspace (8 more bytes per row), and the second kernel, which adds the chunks'
// sums, adds f / (L + eps) to the totals in blocks beside those that write o. The
// chunks are sized by the rows that are filled, so a short sequence in a long cache
// spreads over all blocks. No atomics: every total belongs to one thread.
// B=16, H=16, T=4096, D=128, bf16: 86 us = 6.3 TB/s; four scores per lane instead of
// one, with a load per position and a store per f of each, took 105 us.

#include <algorithm>
#include <type_traits>

#include "attn_cache.h"
#include "kat_internal.h"

namespace kat {

using namespace mfma;

struct AccumArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* L;                  // [B*H] or nullptr
  const float* slopes;       // [H]
  float* total;              // [B, H, T] by stot
  const int32_t* lengths;    // [B] or nullptr (all T)
  const int32_t* positions;  // [B, H, T] by spos, or nullptr
  int B, H, T, D;
  int64_t sq[2], sk[3], sv[3], so[2], stot[2], spos[2];
  float scale, eps;
  int splits;
  float* part;   // [B*H][splits][W] sums f v (W the layout width), 16 sigma^4 as f
  float* lpart;  // [B*H][splits] sums f
  float* f;      // [B*H][T]
};

constexpr int kAccThreads = 256;
constexpr int kAccWaves = kAccThreads / 64;
constexpr int kAccInFlight = 4;  // rows per lane in flight
constexpr int kAccRowsPerBlock = 4 * kAccThreads;  // totals per block of the second kernel
constexpr int kOneWaves = 16;    // one launch: waves of the block of a (b, h)
constexpr int kOneRows = 8192;   // most rows of it (their f stay in LDS)

template <typename T, int W> struct AccShape {
  static constexpr int EPL = 16 / (int)sizeof(T);     // elements per lane
  static constexpr int LPR = W / EPL;                 // lanes per row
  static constexpr int RPW = 64 / LPR;                // rows per wave per load
  static constexpr int RPI = RPW * kAccInFlight;      // consecutive rows per wave per pass
  static_assert(LPR >= 4 && LPR <= 64, "a row is at least a quad of lanes");
};

// lane permutations within quads (DPP)
template <int CTRL> __device__ __forceinline__ float quad(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}

// A pass of a wave takes four loads of RPW rows; lane (sub, grp) holds piece sub of
// rows 4 loads x RPW + grp. The four partial dot products are added over the row's
// lanes so that lane q of every quad ends with load q's (two exchanges within the
// quad halve the values at every step, then one sum per further step): each lane
// maps one score instead of four, loads one position and the first quad of a row
// stores one f.
// ONE: the block takes all rows of its (b, h) and writes o, L and the totals itself.
template <typename T, int W, bool POS, bool ONE>
__global__ __launch_bounds__(64 * (ONE ? kOneWaves : kAccWaves)) void attn_accum_part_k(AccumArgs a) {
  typedef AccShape<T, W> S;
  constexpr int EPL = S::EPL, LPR = S::LPR, RPW = S::RPW, RPI = S::RPI, U = kAccInFlight;
  constexpr int NW = ONE ? kOneWaves : kAccWaves, NT = 64 * NW;
  constexpr int RPP = RPI * NW;  // rows per block per pass
  static_assert(U == 4, "a load per lane of a quad");
  __shared__ float sh_acc[NW][W];
  __shared__ float sh_l[NW];
  __shared__ float sh_f[ONE ? kOneRows : 1];
  const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
  const int split = blockIdx.x;
  const int lane = threadIdx.x & 63, w = wave_id();
  const int sub = lane % LPR, grp = lane / LPR, qd = lane & 3;
  int n = a.lengths ? a.lengths[b] : a.T;
  n = min(max(n, 0), a.T);  // a bad length cannot move a read out of the cache
  const int splits = ONE ? 1 : a.splits;
  const int per = ((n + RPP - 1) / RPP + splits - 1) / splits * RPP;
  const int j0 = split * per, j1 = min(j0 + per, n);
  const float slope = a.slopes[h];
  const int32_t* pp = POS ? a.positions + b * a.spos[0] + h * a.spos[1] : nullptr;
  const int qpos = POS ? (n > 0 ? pp[n - 1] : 0) : n - 1;

  const bool din = sub * EPL < a.D;  // lanes past the head dim: zero query, the row's first piece
  const int col0 = din ? sub * EPL : 0;
  float qv[EPL];
  load_acc<T, EPL>((const T*)a.q + b * a.sq[0] + h * a.sq[1] + col0, qv);
#pragma unroll
  for (int e = 0; e < EPL; ++e) qv[e] = din ? qv[e] * a.scale : 0.f;
  const T* kp = (const T*)a.k + b * a.sk[0] + h * a.sk[1] + col0;
  const T* vp = (const T*)a.v + b * a.sv[0] + h * a.sv[1] + col0;
  float* fp = a.f + (int64_t)bh * a.T;

  float acc[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
  float l = 0.f;
  for (int base = j0 + w * RPI; base < j1; base += RPP) {
    VecT<T, EPL> kr[U], vr[U];
    const int mine = base + qd * RPW + grp;  // the row whose score this lane maps
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = min(base + u * RPW + grp, j1 - 1);  // rows past the chunk re-read its last
      kr[u] = __builtin_bit_cast(VecT<T, EPL>, ld_piece_nt((const char*)(kp + (int64_t)j * a.sk[2])));
      vr[u] = __builtin_bit_cast(VecT<T, EPL>, ld_piece_nt((const char*)(vp + (int64_t)j * a.sv[2])));
    }
    const int pos = POS ? pp[min(mine, j1 - 1)] : mine;
    float d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      d[u] = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) d[u] = fmaf(qv[e], to_acc(kr[u].v[e]), d[u]);
    }
    const bool o1 = lane & 1, o2 = lane & 2;
    const float x = (o1 ? d[1] : d[0]) + quad<0xB1>(o1 ? d[0] : d[1]);  // quad_perm: xor 1
    const float y = (o1 ? d[3] : d[2]) + quad<0xB1>(o1 ? d[2] : d[3]);
    float s = (o2 ? y : x) + quad<0x4E>(o2 ? x : y);  // xor 2
#pragma unroll
    for (int off = 4; off < LPR; off <<= 1) s += __shfl_xor(s, off, 64);
    const float t = sig2_pow4(s - slope * (float)(qpos - pos));
    const float f = mine < j1 ? t : 0.f;
    if (sub < 4 && mine < j1) {
      if constexpr (ONE) sh_f[mine] = f;
      else fp[mine] = f;
    }
    l += f;
    const float fu[U] = {quad<0x00>(f), quad<0x55>(f), quad<0xAA>(f), quad<0xFF>(f)};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < EPL; ++e) acc[e] = fmaf(fu[u], to_acc(vr[u].v[e]), acc[e]);
  }
  l += quad<0xB1>(l);
  l += quad<0x4E>(l);
  // lanes with the same `sub` hold the same columns: add across the row groups
#pragma unroll
  for (int off = LPR; off < 64; off <<= 1) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] += __shfl_xor(acc[e], off, 64);
    l += __shfl_xor(l, off, 64);
  }
  if (grp == 0) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) sh_acc[w][sub * EPL + e] = acc[e];
    if (sub == 0) sh_l[w] = l;
  }
  if constexpr (ONE) {
    // the totals' loads run beside the exchange
    float* tp = a.total + b * a.stot[0] + h * a.stot[1];
    float old = (int)threadIdx.x < n ? tp[threadIdx.x] : 0.f;
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int ww = 0; ww < NW; ++ww) l += sh_l[ww];
    const float inv = inv_sum(l + 16.f * a.eps);
    if (threadIdx.x == 0 && a.L) a.L[bh] = l * 0.0625f;
    if ((int)threadIdx.x < a.D) {
      float t = 0.f;
#pragma unroll
      for (int ww = 0; ww < NW; ++ww) t += sh_acc[ww][threadIdx.x];
      ((T*)a.o)[b * a.so[0] + h * a.so[1] + threadIdx.x] = from_acc<T>(t * inv);
    }
    for (int j = threadIdx.x; j < n; j += NT) {
      if (j >= NT) old = tp[j];
      tp[j] = fmaf(sh_f[j], inv, old);
    }
  } else {
    __syncthreads();
    const int64_t p = (int64_t)bh * a.splits + split;
    for (int d = threadIdx.x; d <= W; d += NT) {
      float t = 0.f;
#pragma unroll
      for (int ww = 0; ww < NW; ++ww) t += d < W ? sh_acc[ww][d] : sh_l[ww];
      if (d < W) a.part[p * W + d] = t;
      else a.lpart[p] = t;
    }
  }
}

// Block (0, bh): L and o. Block (1 + i, bh): the totals of rows i
// kAccRowsPerBlock .. Every block adds the chunks' row sums itself, in the same
// order.
template <typename T, int W> __global__ __launch_bounds__(kAccThreads) void attn_accum_finish_k(AccumArgs a) {
  __shared__ float sh[kAccWaves];
  const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
  const int S = a.splits;
  const float* lp = a.lpart + (int64_t)bh * S;
  float l = 0.f;
  for (int s = threadIdx.x; s < S; s += kAccThreads) l += lp[s];
  l = wave_sum(l);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = l;
  // the loads of the block's own part run beside the sum
  float t[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int col = threadIdx.x;
  const bool first = blockIdx.x == 0;
  if (first && col < W) {  // (a missing split loads the last one again: no branch between the loads)
    const float* p = a.part + (int64_t)bh * S * W + col;
    for (int s = 0; s < S; s += 8) {
      float x[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) x[r] = p[(int64_t)min(s + r, S - 1) * W];
#pragma unroll
      for (int r = 0; r < 8; ++r) t[r] += s + r < S ? x[r] : 0.f;
    }
  }
  int n = a.lengths ? a.lengths[b] : a.T;
  n = min(max(n, 0), a.T);
  const int r0 = ((int)blockIdx.x - 1) * kAccRowsPerBlock + threadIdx.x;
  float* tp = a.total + b * a.stot[0] + h * a.stot[1];
  constexpr int R = kAccRowsPerBlock / kAccThreads;
  float f[R], old[R];
  if (!first) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = r0 + r * kAccThreads;
      f[r] = j < n ? a.f[(int64_t)bh * a.T + j] : 0.f;
      old[r] = j < n ? tp[j] : 0.f;
    }
  }
  __syncthreads();
  l = (sh[0] + sh[1]) + (sh[2] + sh[3]);
  const float inv = inv_sum(l + 16.f * a.eps);
  if (first) {
    if (col == 0 && a.L) a.L[bh] = l * 0.0625f;
    if (col < a.D)
      ((T*)a.o)[b * a.so[0] + h * a.so[1] + col] =
          from_acc<T>((((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]))) * inv);
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = r0 + r * kAccThreads;
      if (j < n) tp[j] = fmaf(f[r], inv, old[r]);
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

static int accum_rpp(int W, int dtype) { return 64 / (W * dtype_size(dtype) / 16) * kAccInFlight * kAccWaves; }

// One launch, a block of 16 waves per (b, h): saves the second launch and the f in
// memory, but a CU streams no more than some 35 GB/s into one block. Taken where the
// (b, h) fill half the CUs, or their rows take less than the second launch: with c =
// 0.56 CUs, bytes per (b, h) x (c - BH) below 20 MB (rates of 35 kB/us per block and
// 5 MB/us in all, 4 us for the launch). bf16, two launches / one, us: 12 heads of 64, T=576
// 7.0 / 4.8; 96 heads, T=1152 11.9 / 10.7, T=2304 16.8 / 19.6; 16 heads of 128, T=1000 6.4
// / 13.0; 256 heads of 128, T=1024 27.6 / 23.6, T=4096 94.2 / 86.5; 384 of 64, T=2304
// 43 / 44; fp32, 48 heads of 64, T=512 7.0 / 8.7.
static bool accum_one(int64_t B, int64_t H, int64_t T, int W, int dtype) {
  const double row = 2.0 * W * dtype_size(dtype);
  return T <= kOneRows && row * T * (0.56 * num_cus() - (double)(B * H)) < 20e6;
}

// chunks per (b, h): three blocks per CU, none smaller than one block pass (1 / 2 / 3 /
// 4 blocks: B=16, H=16, T=4096, D=128 110 / 98 / 96 / 100 us, B=4, H=12, T=2048, D=64 in
// fp32 16.6 / 14.1 / 12.5 / 14.7)
static int accum_splits(int64_t B, int64_t H, int64_t T, int W, int dtype) {
  const int64_t want = (3 * (int64_t)num_cus() + B * H - 1) / (B * H), rpp = accum_rpp(W, dtype);
  return (int)std::max<int64_t>(1, std::min(want, (T + rpp - 1) / rpp));
}

template <typename T, int W, bool POS> static int launch_accum(const AccumArgs& a, bool one, hipStream_t st) {
  if (one) {
    hipLaunchKernelGGL((attn_accum_part_k<T, W, POS, true>), dim3(1, (unsigned)(a.B * a.H)), dim3(64 * kOneWaves), 0, st, a);
    return check_launch("kat_attn_decode_accum");
  }
  hipLaunchKernelGGL((attn_accum_part_k<T, W, POS, false>), dim3((unsigned)a.splits, (unsigned)(a.B * a.H)),
                     dim3(kAccThreads), 0, st, a);
  if (int rc = check_launch("kat_attn_decode_accum (partials)")) return rc;
  const unsigned nb = 1 + (unsigned)((a.T + kAccRowsPerBlock - 1) / kAccRowsPerBlock);
  hipLaunchKernelGGL((attn_accum_finish_k<T, W>), dim3(nb, (unsigned)(a.B * a.H)), dim3(kAccThreads), 0, st, a);
  return check_launch("kat_attn_decode_accum (totals)");
}
template <typename T> static int accum_w(const AccumArgs& a, int W, hipStream_t st) {
  const bool one = accum_one(a.B, a.H, a.T, W, sizeof(T) == 4 ? KAT_F32 : KAT_BF16);
  auto go = [&](auto w) {
    constexpr int kW = decltype(w)::value;
    return a.positions ? launch_accum<T, kW, true>(a, one, st) : launch_accum<T, kW, false>(a, one, st);
  };
  switch (W) {
    case 32: if constexpr (sizeof(T) == 4) return go(std::integral_constant<int, 32>{}); break;
    case 64: return go(std::integral_constant<int, 64>{});
    case 128: return go(std::integral_constant<int, 128>{});
    case 256: if constexpr (sizeof(T) == 2) return go(std::integral_constant<int, 256>{}); break;
  }
  return fail(KAT_EUNSUPPORTED, "kat_attn_decode_accum: head dim %d", a.D);
}

}  // namespace kat

using namespace kat;

extern "C" size_t kat_attn_decode_accum_workspace_size(int64_t B, int64_t H, int64_t T, int64_t D, int dtype) {
  const int W = cache_layout(D, dtype);
  if (B <= 0 || H <= 0 || T <= 0 || !W || accum_one(B, H, T, W, dtype)) return 0;
  return (size_t)(B * H) * ((size_t)accum_splits(B, H, T, W, dtype) * (W + 1) + T) * sizeof(float);
}

extern "C" int kat_attn_decode_accum(const void* q, const void* k, const void* v, void* out, float* L,
                                     const float* slopes, float* weights, const int32_t* lengths,
                                     const int32_t* positions, const int64_t* wp_strides, void* workspace,
                                     size_t workspace_bytes, int64_t B, int64_t H, int64_t T, int64_t D,
                                     const int64_t* strides, float scale, float eps, int dtype, void* stream) {
  const char* nm = "kat_attn_decode_accum";
  if (B < 0 || H < 0 || T < 0 || D < 0) return fail(KAT_EINVAL, "%s: negative size", nm);
  if (B > 0xffff || H > 0xffff || B * H > 0xffff || T > 0x3fffffff)
    return fail(KAT_EUNSUPPORTED, "%s: B*H or T too large", nm);
  const int W = cache_layout(D, dtype);
  if (!W) return fail(KAT_EUNSUPPORTED, "%s: head dim %lld with dtype %d", nm, (long long)D, dtype);
  if (B * H == 0) return KAT_OK;
  if (!q || !out || !slopes || !strides || !wp_strides || (T > 0 && (!k || !v || !weights)))
    return fail(KAT_EINVAL, "%s: null pointer", nm);
  const int esz = dtype_size(dtype);
  const int64_t size[10] = {B, H, B, H, T, B, H, T, B, H};
  int64_t st10[10];
  for (int t = 0; t < 10; ++t) {
    st10[t] = dim_stride(strides[t], size[t]);
    if ((st10[t] * esz) % 16 != 0) return fail(KAT_EUNSUPPORTED, "%s: strides must keep rows 16-byte aligned", nm);
  }
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(KAT_EUNSUPPORTED, "%s: tensors must be 16-byte aligned", nm);
  if (T > 1 && (st10[4] < D || st10[7] < D)) return fail(KAT_EINVAL, "%s: cache row stride < D", nm);
  AccumArgs a = {};
  a.q = q;
  a.k = k;
  a.v = v;
  a.o = out;
  a.L = L;
  a.slopes = slopes;
  a.total = weights;
  a.lengths = lengths;
  a.positions = positions;
  a.B = (int)B;
  a.H = (int)H;
  a.T = (int)T;
  a.D = (int)D;
  for (int i = 0; i < 2; ++i) {
    a.sq[i] = st10[i];
    a.so[i] = st10[8 + i];
    a.stot[i] = wp_strides[i];
    a.spos[i] = wp_strides[2 + i];
  }
  for (int i = 0; i < 3; ++i) {
    a.sk[i] = st10[2 + i];
    a.sv[i] = st10[5 + i];
  }
  a.scale = scale;
  a.eps = eps;
  a.splits = accum_splits(B, H, std::max<int64_t>(T, 1), W, dtype);
  const size_t need = kat_attn_decode_accum_workspace_size(B, H, std::max<int64_t>(T, 1), D, dtype);
  if (need && (!workspace || workspace_bytes < need))
    return fail(KAT_EINVAL, "%s: workspace %zu bytes < required %zu", nm, workspace_bytes, need);
  a.part = (float*)workspace;
  a.lpart = a.part + (size_t)(B * H) * a.splits * W;
  a.f = a.lpart + (size_t)(B * H) * a.splits;
  const hipStream_t st = as_stream(stream);
  switch (dtype) {
    case KAT_F32: return accum_w<float>(a, W, st);
    case KAT_BF16: return accum_w<bf16>(a, W, st);
    case KAT_F16: return accum_w<f16>(a, W, st);
  }
  return fail(KAT_EUNSUPPORTED, "%s: unsupported dtype %d", nm, dtype);
}
