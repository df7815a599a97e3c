// Eviction from a KV cache by accumulated attention weight on gfx950.
//
// Of the n = lengths[b] filled rows of each (b, h), m = min(n, keep) stay: those
// whose position is among the newest (position > position of row n - 1 -
// recent), then those with the largest total weight, ties to the lower row (a
// NaN total ranks above every number). Two forms:
//   into another cache: the kept rows of k, v, weights and positions go to rows
//     0 .. m - 1 of the outputs in their order; rows behind stay as they are
//   in place: kept rows below m stay where they are, and the kept rows at or
//     past m move, in order, into the rows below m that are given up. Rows are
//     read at or past m and written below it, so blocks need no order, and only
//     what has to move is moved. (Attention over the cache goes by the rows'
//     positions, not by their order.)
// lengths[b] becomes m.
//
// Design: a plan kernel, one block per (b, h), selects and writes the list of
// moves; a second kernel moves the rows, many blocks per (b, h). The selection is
// latency-bound (a few KB per head): totals become unsigned keys in the order
// of the numbers, held in registers (each wave a contiguous run of rows), and
// the m-th largest key is found bit by bit: one ballot and scalar popcount per 64
// keys and one block barrier per bit, no atomics, no sort. Ties and the list
// order come from ballots and prefix sums over the waves' runs.

#include <algorithm>

#include "attn_cache.h"
#include "kat_internal.h"

namespace kat {

struct EvictArgs {
  const char* k;
  const char* v;
  const float* w;
  const int32_t* pos;
  const int32_t* len;  // [B] or nullptr (all T)
  char* ko;
  char* vo;
  float* wo;
  int32_t* po;
  int32_t* lo;  // [B] or nullptr
  int B, H, T, keep, recent, in_place;
  int pieces;  // 16-byte pieces of a row
  // bytes: k, v, ko, vo (b, h, t); elements: w, pos, wo, po (b, h)
  int64_t sk[3], sv[3], sko[3], svo[3], sw[2], spos[2], swo[2], spo[2];
  int32_t* src;  // [B*H][keep] rows to move, in order
  int32_t* dst;  // [B*H][keep] where to (in place)
  int32_t* cnt;  // [B*H]
};

constexpr int kEvThreads = 1024;
constexpr int kEvWaves = kEvThreads / 64;

// the number of rows of a wave whose bit is set, as a wave-uniform value
__device__ __forceinline__ int bits(bool x) { return __popcll(__builtin_amdgcn_ballot_w64(x)); }
// set bits of the lanes below this one
__device__ __forceinline__ int bits_below(bool x, int lane) {
  return __popcll(__builtin_amdgcn_ballot_w64(x) & ((1ull << lane) - 1ull));
}

// R: keys per thread held in registers (T <= 1024 R); 0: any T, the keys are
// formed again from memory each time
template <int R> __global__ __launch_bounds__(kEvThreads) void kv_evict_plan_k(EvictArgs a) {
  __shared__ int cnt[2][kEvWaves];
  __shared__ int tot[3][kEvWaves];
  const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H;
  const int lane = threadIdx.x & 63, wv = mfma::wave_id();
  int n = a.len ? a.len[b] : a.T;
  n = min(max(n, 0), a.T);
  const int m = min(n, a.keep);
  const float* w = a.w + b * a.sw[0] + h * a.sw[1];
  const int32_t* pos = a.pos + b * a.spos[0] + h * a.spos[1];
  // rows with a position above this are the newest
  const int64_t edge = n > 0 ? (int64_t)pos[n - 1] - a.recent : 0;

  // wave wv owns rows run .. run + seg - 1, 64 at a time
  const int seg = R ? 64 * R : ((n + kEvThreads - 1) / kEvThreads) * 64;
  const int run = wv * seg;
  const int end = min(run + seg, n);
  auto key_of = [&](int j) __attribute__((always_inline)) -> uint32_t {
    if (j >= end) return 0u;  // below every row's key
    if ((int64_t)pos[j] > edge) return 0xffffffffu;
    const uint32_t u = __builtin_bit_cast(uint32_t, w[j] + 0.f);  // -0 as 0
    const uint32_t o = (u >> 31) ? ~u : (u | 0x80000000u);
    return (u & 0x7fffffffu) > 0x7f800000u ? 0xfffffffeu : min(max(o, 1u), 0xfffffffeu);
  };
  uint32_t kr[R ? R : 1];
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) kr[i] = key_of(run + i * 64 + lane);
  }
  // f(key, row) for the wave's rows in order, all lanes together
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i) f(kr[i], run + i * 64 + lane);
    } else {
      for (int j = run; j < end; j += 64) f(key_of(j + lane), j + lane);
    }
  };

  // the m-th largest key
  uint32_t tau = 0;
  int above = 0;  // keys above tau
  if (m < n) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t cand = tau | (1u << bit);
      int c = 0;
      each([&](uint32_t x, int) { c += bits(x >= cand); });
      if (lane == 0) cnt[bit & 1][wv] = c;
      __syncthreads();
      c = 0;
#pragma unroll
      for (int i = 0; i < kEvWaves; ++i) c += cnt[bit & 1][i];
      if (c >= m) tau = cand;
      else above = c;
    }
  } else {
    tau = 1;  // every filled row
  }
  // of the rows with that key, the first `ties` stay
  const int ties = m < n ? m - above : n;
  int eq = 0;
  each([&](uint32_t x, int) { eq += bits(x == tau); });
  if (lane == 0) tot[0][wv] = eq;
  __syncthreads();
  int eq0 = 0;
  for (int i = 0; i < wv; ++i) eq0 += tot[0][i];
  auto kept = [&](uint32_t x, int& e) __attribute__((always_inline)) {
    const bool q = x == tau;
    const bool y = x > tau || (q && e + bits_below(q, lane) < ties);
    e += bits(q);
    return y;
  };
  int e = eq0, nm = 0, nh = 0;  // moves and (in place) holes of this wave
  each([&](uint32_t x, int j) {
    const bool y = kept(x, e);
    nm += bits(y && (!a.in_place || j >= m));
    nh += bits(!y && j < m);
  });
  if (lane == 0) {
    tot[1][wv] = nm;
    tot[2][wv] = nh;
  }
  __syncthreads();
  int m0 = 0, h0 = 0;
  for (int i = 0; i < wv; ++i) {
    m0 += tot[1][i];
    h0 += tot[2][i];
  }
  if (wv == kEvWaves - 1 && lane == 0) a.cnt[bh] = m0 + nm;
  int32_t* src = a.src + (int64_t)bh * a.keep;
  int32_t* dst = a.dst + (int64_t)bh * a.keep;
  e = eq0;
  each([&](uint32_t x, int j) {
    const bool y = kept(x, e);
    const bool mv = y && (!a.in_place || j >= m), ho = !y && j < m;
    if (mv) src[m0 + bits_below(mv, lane)] = j;
    if (a.in_place && ho) dst[h0 + bits_below(ho, lane)] = j;
    m0 += bits(mv);
    h0 += bits(ho);
  });
}

constexpr int kMvThreads = 256;
constexpr int kMvRows = 32;  // rows per block

__global__ __launch_bounds__(kMvThreads) void kv_evict_move_k(EvictArgs a) {
  const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
  const int t = threadIdx.x;
  if (blockIdx.x == 0 && h == 0 && t == 0 && a.lo) {
    const int n = a.len ? a.len[b] : a.T;
    a.lo[b] = min(min(max(n, 0), a.T), a.keep);
  }
  const int r0 = (int)blockIdx.x * kMvRows, r1 = min(r0 + kMvRows, a.cnt[bh]);
  if (r0 >= r1) return;
  const int32_t* src = a.src + (int64_t)bh * a.keep;
  const int32_t* dst = a.dst + (int64_t)bh * a.keep;
  auto to = [&](int r) __attribute__((always_inline)) { return a.in_place ? dst[r] : r; };
  if (r0 + t < r1) {
    const int s = src[r0 + t], d = to(r0 + t);
    a.wo[b * a.swo[0] + h * a.swo[1] + d] = a.w[b * a.sw[0] + h * a.sw[1] + s];
    a.po[b * a.spo[0] + h * a.spo[1] + d] = a.pos[b * a.spos[0] + h * a.spos[1] + s];
  }
  const char* k = a.k + b * a.sk[0] + h * a.sk[1];
  const char* v = a.v + b * a.sv[0] + h * a.sv[1];
  char* ko = a.ko + b * a.sko[0] + h * a.sko[1];
  char* vo = a.vo + b * a.svo[0] + h * a.svo[1];
  const int per = a.pieces, all = (r1 - r0) * per;
  for (int i = t; i < all; i += kMvThreads) {
    const int r = i / per, p = i - r * per;
    const int s = src[r0 + r], d = to(r0 + r);
    const mfma::i16x8 x = ld_piece_nt(k + (int64_t)s * a.sk[2] + 16 * p);
    const mfma::i16x8 y = ld_piece_nt(v + (int64_t)s * a.sv[2] + 16 * p);
    *reinterpret_cast<mfma::i16x8*>(ko + (int64_t)d * a.sko[2] + 16 * p) = x;
    *reinterpret_cast<mfma::i16x8*>(vo + (int64_t)d * a.svo[2] + 16 * p) = y;
  }
}

template <int R> static int launch_evict(const EvictArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((kv_evict_plan_k<R>), dim3((unsigned)(a.B * a.H)), dim3(kEvThreads), 0, st, a);
  if (int rc = check_launch("kat_kv_evict (plan)")) return rc;
  const int64_t most = a.in_place ? std::min<int64_t>(a.keep, std::max(0, a.T - a.keep)) : std::min(a.keep, a.T);
  const unsigned nb = (unsigned)std::max<int64_t>(1, (most + kMvRows - 1) / kMvRows);
  hipLaunchKernelGGL(kv_evict_move_k, dim3(nb, (unsigned)(a.B * a.H)), dim3(kMvThreads), 0, st, a);
  return check_launch("kat_kv_evict (move)");
}

}  // namespace kat

using namespace kat;

extern "C" size_t kat_kv_evict_workspace_size(int64_t B, int64_t H, int64_t keep) {
  if (B <= 0 || H <= 0 || keep < 0) return 0;
  return (size_t)(B * H) * (2 * (size_t)keep + 1) * sizeof(int32_t);
}

extern "C" int kat_kv_evict(const void* k, const void* v, const float* weights, const int32_t* positions,
                            const int32_t* lengths, void* k_out, void* v_out, float* weights_out,
                            int32_t* positions_out, int32_t* lengths_out, void* workspace, size_t workspace_bytes,
                            int64_t B, int64_t H, int64_t T, int64_t D, int64_t keep, int64_t recent, int in_place,
                            const int64_t* strides, int dtype, void* stream) {
  const char* nm = "kat_kv_evict";
  if (B < 0 || H < 0 || T < 0 || D < 0 || keep < 0 || recent < 0) return fail(KAT_EINVAL, "%s: negative size", nm);
  if (recent > keep) return fail(KAT_EINVAL, "%s: recent %lld > keep %lld", nm, (long long)recent, (long long)keep);
  if (B > 0xffff || H > 0xffff || B * H > 0xffff || T > 0x3fffffff || keep > 0x3fffffff)
    return fail(KAT_EUNSUPPORTED, "%s: B*H, T or keep too large", nm);
  const int esz = dtype_size(dtype);
  if (!esz || D == 0 || (D * esz) % 16 != 0)
    return fail(KAT_EUNSUPPORTED, "%s: head dim %lld with dtype %d (rows of whole 16-byte pieces)", nm, (long long)D, dtype);
  if (B * H == 0) return KAT_OK;
  if (!k || !v || !weights || !positions || !k_out || !v_out || !weights_out || !positions_out || !strides)
    return fail(KAT_EINVAL, "%s: null pointer", nm);
  if (in_place && (k != k_out || v != v_out || weights != weights_out || positions != positions_out))
    return fail(KAT_EINVAL, "%s: in place, but the outputs are other tensors", nm);
  for (int t = 0; t < 12; ++t)
    if ((strides[t] * esz) % 16 != 0) return fail(KAT_EUNSUPPORTED, "%s: strides must keep rows 16-byte aligned", nm);
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_out) || !aligned16(v_out))
    return fail(KAT_EUNSUPPORTED, "%s: tensors must be 16-byte aligned", nm);
  const size_t need = kat_kv_evict_workspace_size(B, H, keep);
  if (!workspace || workspace_bytes < need)
    return fail(KAT_EINVAL, "%s: workspace %zu bytes < required %zu", nm, workspace_bytes, need);
  EvictArgs a = {};
  a.k = (const char*)k;
  a.v = (const char*)v;
  a.w = weights;
  a.pos = positions;
  a.len = lengths;
  a.ko = (char*)k_out;
  a.vo = (char*)v_out;
  a.wo = weights_out;
  a.po = positions_out;
  a.lo = lengths_out;
  a.B = (int)B;
  a.H = (int)H;
  a.T = (int)T;
  a.keep = (int)keep;
  a.recent = (int)recent;
  a.in_place = in_place != 0;
  a.pieces = (int)(D * esz / 16);
  for (int i = 0; i < 3; ++i) {
    a.sk[i] = strides[i] * esz;
    a.sv[i] = strides[3 + i] * esz;
    a.sko[i] = strides[6 + i] * esz;
    a.svo[i] = strides[9 + i] * esz;
  }
  for (int i = 0; i < 2; ++i) {
    a.sw[i] = strides[12 + i];
    a.spos[i] = strides[14 + i];
    a.swo[i] = strides[16 + i];
    a.spo[i] = strides[18 + i];
  }
  a.src = (int32_t*)workspace;
  a.dst = a.src + (size_t)(B * H) * keep;
  a.cnt = a.dst + (size_t)(B * H) * keep;
  const hipStream_t st = as_stream(stream);
  if (T <= 1024) return launch_evict<1>(a, st);
  if (T <= 4096) return launch_evict<4>(a, st);
  if (T <= 16384) return launch_evict<16>(a, st);
  if (T <= 32768) return launch_evict<32>(a, st);
  return launch_evict<0>(a, st);
}
