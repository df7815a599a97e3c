// The attention weight that each key of a prompt receives, summed over the
// queries, on gfx950:
//   w_j = sum_{i >= j, i >= T - last} f_ij / (L_i + eps),   f_ij = sigma(s_ij)^4,
//   s_ij = scale <q_i, k_j> - slope_h (i - j)
// with L the row sums that the forward (kat_attn_fwd) stored. With a token mask,
// a dropped token neither gives nor receives weight. This is what an eviction
// policy needs of a prompt before its keys go into a smaller cache.
//
// Design (MI355X). One matrix product and 8 VALU operations per (query, key)
// pair and no output but T floats per head: instruction issue (MFMA + VALU)
// bounds it, not memory. Like the backward's dK/dV pass a block keeps its keys'
// fragments in registers and streams the queries through LDS (64-row tiles,
// double-buffered LDS-DMA, the swizzled tiles of attn_mfma_dev.h):
//   S[q][key] = Q K^T   A = Q rows (ds_read_b128), B = K (registers)
// and a lane holds queries 4 g + j of its key li, so the column sums stay in
// registers until the end (lane groups added by two shuffles). Every Q fragment
// read feeds the products of KS 16-key subtiles. Grids short of the chip split the
// queries over the waves of a block or over blocks, whose sums are added in a
// fixed order (keyw_plan has the rules and what they measured). No atomics.

#include <algorithm>
#include <type_traits>

#include "attn_cache.h"
#include "kat_internal.h"

namespace kat {

using namespace mfma;

struct KeywArgs {
  const void* q;
  const void* k;
  const float* L;       // [B, H, T] by sl
  float* out;           // [B, H, T] by so
  const float* slopes;  // [H]
  const uint8_t* mask;  // [B, T]: row b at mask + b * smask; or nullptr
  int B, H, T, D;
  int lo;               // first query that counts
  int qc, chunks;       // queries per block; most chunks of a key block
  int64_t sq[3], sk[3], sl[3], so[2], smask;
  float scale, eps;
  float* part;          // [chunks][B*H][T], or nullptr (one chunk)
};

constexpr int kKwWaves = 4;
// a row in 16-bit units
template <typename T, int W> constexpr int kw_units() { return W * (int)sizeof(T) / 2; }
// query rows per LDS tile
template <int U> constexpr int kw_rows() { return U == 512 ? 32 : 64; }

// KS: 16-key subtiles per wave (their fragments take U / 8 registers each). QW > 1:
// the block's QW waves share their keys and split a tile's queries (16 rows each).
// KK: 64-byte column blocks that hold columns (the tiles are U / 32 wide)
template <typename T, int W, int KK, bool KM, int KS, int QW>
__global__ __launch_bounds__(64 * (QW > 1 ? QW : kKwWaves), (kw_units<T, W>() == 512 ? 1 : 2)) void attn_keyw_k(KeywArgs a) {
  constexpr int ES = (int)sizeof(T), U = kw_units<T, W>(), NW = QW > 1 ? QW : kKwWaves, QR = QW > 1 ? 16 * QW : kw_rows<U>();
  constexpr int KWV = NW / QW;   // waves with keys of their own
  constexpr int BK = 16 * KS * KWV;    // keys per block
  constexpr int WR = QR / QW;          // rows of a tile per wave
  constexpr bool kBiasC = ES == 2;     // the bias enters the product as its C operand
  __shared__ short sq[2][QR * U];
  __shared__ float sc[2][QR];  // 1 / (16 (L + eps)) of the tile's queries; 0: the query does not count
  __shared__ float sw[QW][BK];

  int bh, kb;
  block_order((int)blockIdx.x, a.B * a.H, bh, kb);
  const int b = bh / a.H, h = bh - b * a.H;
  const int T_ = a.T;
  const int r0 = std::max(a.lo, kb * BK) + (int)blockIdx.y * a.qc;
  const int r1 = std::min(T_, r0 + a.qc);
  if (r0 >= r1) return;  // fewer chunks than the longest key block has
  const int lane = threadIdx.x & 63, w = wave_id();
  const int g = lane >> 4, li = lane & 15;
  const int kw = kb * BK + (w % KWV) * 16 * KS;  // the wave's first key
  const int w0 = (w / KWV) * WR;                 // its first row of a tile

  const char* qp = (const char*)((const T*)a.q + b * a.sq[0] + h * a.sq[1]);
  const char* kp = (const char*)((const T*)a.k + b * a.sk[0] + h * a.sk[1]);
  const int64_t sqb = a.sq[2] * ES, skb = a.sk[2] * ES;
  const float* lp = a.L + b * a.sl[0] + h * a.sl[1];
  const uint8_t* mp = KM ? a.mask + b * a.smask : nullptr;
  const float slope = a.slopes[h];
  // (a scale below 2^-60 moves no score, but the bias is divided by it)
  const float scale = !kBiasC || fabsf(a.scale) >= 0x1p-60f ? a.scale : copysignf(0x1p-60f, a.scale);
  const int cols = a.D * ES / 16;
  // A block whose keys all are dropped is done (every wave reads all of its keys'
  // mask, so they agree), and a wave without a key that counts (!live) only loads.
  // With tiles skipped whose queries all are dropped, prompts padded on the left by
  // 0 .. T/2 tokens: fp16, 120 heads, T=2217 107 us without, 77 with; fp32, 12 heads,
  // T=1000 18.9 / 10.5; bf16, 48 heads, T=256, 64 queries 3.7 / 4.0. (The test after
  // the first loads are issued: 82.5 / 11.9 / 3.9.)
  bool live = true;
  if constexpr (KM) {
    uint64_t in = 0;
    live = false;
#pragma unroll
    for (int i = 0; i < BK; i += 64) {
      const int key = kb * BK + i + lane;
      const uint64_t m = __builtin_amdgcn_ballot_w64(i + lane < BK && key < T_ && mp[std::min(key, T_ - 1)] != 0);
      in |= m;
      const int k0 = kw - kb * BK - i;  // the wave's keys are bits k0 .. k0 + 16 KS - 1 of one of these words
      if (k0 >= 0 && k0 < 64) live = (m >> k0 & (1ull << 16 * KS) - 1) != 0;
    }
    if (in == 0) {
      const int key = kb * BK + (int)threadIdx.x;
      if ((int)threadIdx.x < BK && key < T_) {
        if (a.part) a.part[((int64_t)blockIdx.y * a.B * a.H + bh) * T_ + key] = 0.f;
        else a.out[b * a.so[0] + h * a.so[1] + key] = 0.f;
      }
      return;
    }
  }

  TileDma<U, NW, QR> dq;
  dq.init(w, lane, (uint32_t)(sqb / 2), a.D * ES / 2);
  auto issue = [&](short* tile, int row) __attribute__((always_inline)) {
    const int64_t left = (int64_t)(T_ - 1 - row) * sqb + a.D * ES;  // bytes from this row to the last one's end
    dq.issue_rows(tile, qp + (int64_t)row * sqb, (uint32_t)std::min<int64_t>(left, 0x7fffffff), w);
  };
  auto cinv = [&](int row) __attribute__((always_inline)) {
    const bool in = row < r1 && (!KM || mp[std::min(row, T_ - 1)] != 0);
    const float l = lp[(int64_t)std::min(row, T_ - 1) * a.sl[2]];
    return in ? inv_sum(16.f * (l + a.eps)) : 0.f;
  };

  issue(sq[0], r0);
  i16x8 kf[KS][KK];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int p = 4 * kk + g;
      kf[ks][kk] = i16x8{0, 0, 0, 0, 0, 0, 0, 0};
      if (p < cols)
        kf[ks][kk] = *reinterpret_cast<const i16x8*>(kp + (int64_t)std::min(kw + 16 * ks + li, T_ - 1) * skb + 16 * p);
    }
  if (threadIdx.x < QR) sc[0][threadIdx.x] = cinv(r0 + (int)threadIdx.x);
  // slope (key - q) of a 16 x 16 piece: the lane's part, for the product divided
  // by the scale (fp32: added after it, or it would set the rounding of the sums)
  f32x4 bl;
#pragma unroll
  for (int j = 0; j < 4; ++j) bl[j] = (kBiasC ? slope / scale : slope) * (float)(li - 4 * g - j);
  f32x4 acc[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) acc[ks] = f32x4{0.f, 0.f, 0.f, 0.f};

  // the wave's rows of a tile, row .. row + WR - 1, against its keys. MASKED: they
  // touch the diagonal or hold a query that does not count (whose values may be
  // anything)
  auto tile = [&](auto masked_tag, int row, const short* qt, const float* ct) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const float base = slope * (float)(kw - row);
#pragma unroll
    for (int hr = 0; hr < WR; hr += 16) {
      f32x4 s_[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s_[ks] = kBiasC ? bl : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const i16x8 qa = lds16(qt + soff<U>(hr + li, 32 * kk + 8 * g));
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s_[ks] = dot64<T>(qa, kf[ks][kk], s_[ks]);
      }
      const f32x4 c = *reinterpret_cast<const f32x4*>(ct + hr + 4 * g);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const float tterm = fmaf(slope, (float)(16 * ks - hr), base);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float s = fmaf(s_[ks][j], scale, kBiasC ? tterm : bl[j] + tterm);
          const float r = __builtin_amdgcn_rcpf(fabsf(s) + 1.f);
          const float t = fmaf(s, r, 1.f);
          const float t2 = t * t;
          const float f = t2 * t2;
          if constexpr (MASKED) {
            const bool in = c[j] != 0.f && kw + 16 * ks + li <= row + hr + 4 * g + j;
            acc[ks][j] = fmaf(in ? f : 0.f, in ? c[j] : 0.f, acc[ks][j]);
          } else {
            acc[ks][j] = fmaf(f, c[j], acc[ks][j]);
          }
        }
      }
    }
  };

  dma_wait();
  __syncthreads();
  auto step = [&](int row, auto buf_tag) __attribute__((always_inline)) {
    constexpr int buf = decltype(buf_tag)::value;
    const bool more = row + QR < r1;
    float cn = 0.f;
    if (more) {
      issue(sq[buf ^ 1], row + QR);
      if (threadIdx.x < QR) cn = cinv(row + QR + (int)threadIdx.x);
    }
    const int rw = row + w0;
    if (rw + WR - 1 >= kw) {  // else every key of the wave lies past its queries
      bool plain = rw >= kw + 16 * KS - 1, some = true;
      if constexpr (KM) {
        const uint64_t out = __builtin_amdgcn_ballot_w64(sc[buf][w0 + lane % WR] == 0.f);
        plain = plain && out == 0;
        some = live && out != ~0ull;
      }
      if (!some) {  // a dropped key, or queries that do not count: no weight
      } else if (plain) tile(std::false_type{}, rw, sq[buf] + w0 * U, sc[buf] + w0);
      else tile(std::true_type{}, rw, sq[buf] + w0 * U, sc[buf] + w0);
    }
    if (more && threadIdx.x < QR) sc[buf ^ 1][threadIdx.x] = cn;
    dma_wait();
    __syncthreads();
  };
  for (int row = r0; row < r1; row += 2 * QR) {
    step(row, std::integral_constant<int, 0>{});
    if (row + QR < r1) step(row + QR, std::integral_constant<int, 1>{});
  }

#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    float t = (acc[ks][0] + acc[ks][1]) + (acc[ks][2] + acc[ks][3]);
    t += __shfl_xor(t, 16, 64);
    t += __shfl_xor(t, 32, 64);
    if (g == 0) sw[w / KWV][(w % KWV) * 16 * KS + 16 * ks + li] = t;
  }
  __syncthreads();
  const int key = kb * BK + (int)threadIdx.x;
  if ((int)threadIdx.x < BK && key < T_) {
    float t = sw[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < QW; ++i) t += sw[i][threadIdx.x];
    if (KM && mp[key] == 0) t = 0.f;
    if (a.part) a.part[((int64_t)blockIdx.y * a.B * a.H + bh) * T_ + key] = t;
    else a.out[b * a.so[0] + h * a.so[1] + key] = t;
  }
}

// adds the chunks of each key in order (a missing chunk loads the last one again:
// no branch between the loads)
__global__ __launch_bounds__(256) void attn_keyw_sum_k(KeywArgs a, int bk) {
  const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
  const int key = blockIdx.x * 256 + threadIdx.x;
  if (key >= a.T) return;
  const int rows = a.T - std::max(a.lo, key / bk * bk);
  const int nc = (rows + a.qc - 1) / a.qc;
  const int64_t step = (int64_t)a.B * a.H * a.T;
  const float* p = a.part + (int64_t)bh * a.T + key;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < nc; c += 4) {
    float x[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = p[std::min(c + r, nc - 1) * step];
#pragma unroll
    for (int r = 0; r < 4; ++r) t[r] += c + r < nc ? x[r] : 0.f;
  }
  a.out[b * a.so[0] + h * a.so[1] + key] = (t[0] + t[1]) + (t[2] + t[3]);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// layout widths: 64, 128, 256 (16-bit types: D a multiple of 8 up to 256), 32
// .. 256 (fp32: multiples of 4 up to 256), the head dims of the MFMA forward
static int keyw_layout(int64_t D, int dtype) {
  if (dtype == KAT_F32 && D > 128 && D <= 256 && D % 4 == 0) return 256;
  return cache_layout(D, dtype);
}
// How a call is laid out: keys per block (ks 16-key subtiles per wave, qw waves
// per key set), queries per block and their number of chunks. Measured (GPU time,
// us, causal, every query unless said):
//  - Own keys per wave, 16 or (16-bit types, large calls) 32 of them: more keys per Q
//    read against more waves per SIMD. bf16 16 / 32 / 64 keys: 64 heads, T=4096, D=128
//    214 / 194 / 219; 192 heads, T=2048, D=64 119 / 114 / 122, of which the last 64
//    queries 15.8 / 13.9 / 14.6; 48 heads, T=2048 35 / 37 / 43; 64 heads, T=1000, D=96
//    19.4 / 21.5 / 25. fp32, T=2048: 32 heads of 128 172 / 180, 12 of 64 44.8 / 44.9.
//  - With fewer than three such blocks per CU the queries are split too. Up to 1024
//    rows over the four waves of a block that share 16 keys, in one launch: bf16, D=64,
//    chunks / waves: 12 heads, T=256 5.9 / 4.3; 48 heads, T=512 9.3 / 7.6; 24 heads,
//    T=1000 12.3 / 10.9 (12 heads 9.6 / 9.9, and 16.6 / 18.4 at T=2048); over eight
//    waves while there are fewer than three such blocks per CU (four / eight waves: 12
//    heads, T=512, D=128 7.2 / 6.3, T=1000, D=64 10.0 / 7.8; 24 heads, T=512, D=64 6.3 /
//    6.4, in fp32 11.3 / 12.9; 96 heads, T=256 6.2 / 8.4). Beyond 1024 rows, in
//    chunks over blocks, about four per CU, and a second launch: fp32, 12 heads,
//    T=2048 53 us in two chunks, 44.8 in six.
//  - Else one block takes all its queries, the longest first (64 heads, T=4096: 194 us
//    whole, 207 in two chunks; 96 heads, T=512 8.9 whole, 11.7 split over four waves).
struct KeywPlan {
  int ks, qw, bk, qc, chunks;
};
static KeywPlan keyw_plan(int64_t B, int64_t H, int64_t T, int64_t lo, int W, int dtype) {
  const int64_t cus = num_cus(), bh = B * H;
  KeywPlan p = {1, 1, 0, 0, 0};
  const double pairs = (double)bh * ((double)(T - lo) * lo + 0.5 * (T - lo) * (T - lo));
  if (dtype != KAT_F32 && (pairs >= 0x1p27 || (T + 127) / 128 * bh >= 8 * cus)) p.ks = 2;
  p.bk = 16 * p.ks * kKwWaves;
  int64_t rows = 0;  // (key block, query row) pairs of one head
  for (int64_t k = 0; k < T; k += p.bk) rows += T - std::max(lo, k);
  int64_t c = T - lo;
  if ((T + p.bk - 1) / p.bk * bh < 3 * cus) c = std::max<int64_t>(64, (rows * bh + 4 * cus - 1) / (4 * cus));
  c = (c + 63) / 64 * 64;  // whole tiles
  if (c < T - lo && p.ks == 1 && T <= 1024) {
    p.qw = (T + 15) / 16 * bh < 3 * cus && W * dtype_size(dtype) <= 512 ? 8 : 4;
    p.bk = 16;
    c = (T - lo + 63) / 64 * 64;
  }
  p.chunks = (int)((T - lo + c - 1) / c);
  p.qc = (int)c;
  return p;
}

template <typename T, int W, int KK, int KS, int QW> static int launch_keyw(const KeywArgs& a, hipStream_t st) {
  constexpr int BK = 16 * KS * (QW > 1 ? 1 : kKwWaves);
  const dim3 grid((unsigned)((a.T + BK - 1) / BK * a.B * a.H), (unsigned)a.chunks), block(64 * (QW > 1 ? QW : kKwWaves));
  if (a.mask) hipLaunchKernelGGL((attn_keyw_k<T, W, KK, true, KS, QW>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((attn_keyw_k<T, W, KK, false, KS, QW>), grid, block, 0, st, a);
  if (int rc = check_launch("kat_attn_key_weights")) return rc;
  if (!a.part) return KAT_OK;
  hipLaunchKernelGGL(attn_keyw_sum_k, dim3((unsigned)((a.T + 255) / 256), (unsigned)(a.B * a.H)), dim3(256), 0, st, a, BK);
  return check_launch("kat_attn_key_weights (sum)");
}
template <typename T, int W, int KK> static int keyw_mode(const KeywArgs& a, const KeywPlan& p, hipStream_t st) {
  if constexpr (kw_units<T, W>() <= 256) {
    if (p.qw == 8) return launch_keyw<T, W, KK, 1, 8>(a, st);
  }
  if (p.qw == 4) return launch_keyw<T, W, KK, 1, 4>(a, st);
  if constexpr (sizeof(T) == 2) {
    if (p.ks == 2) return launch_keyw<T, W, KK, 2, 1>(a, st);
  }
  return launch_keyw<T, W, KK, 1, 1>(a, st);
}
// Column blocks: all of a layout's, or the first three quarters where the head
// dim ends there (96, 192; 48 in fp32), so that no zeros are multiplied. All / three
// quarters, us: fp32, 128 heads, T=1245, D=80 246 / 203; fp32, 144 heads, T=2048,
// D=48 355 / 295; bf16, 64 heads, T=2048, D=96 64.6 / 58.1; bf16, 48 heads, T=1000,
// D=192 24.1 / 22.2.
template <typename T, int W> static int keyw_cols(const KeywArgs& a, const KeywPlan& p, hipStream_t st) {
  constexpr int KK = kw_units<T, W>() / 32;
  if constexpr (KK >= 4) {
    if (a.D <= W / 4 * 3) return keyw_mode<T, W, KK / 4 * 3>(a, p, st);
  }
  return keyw_mode<T, W, KK>(a, p, st);
}
template <typename T> static int keyw_w(const KeywArgs& a, int W, const KeywPlan& p, hipStream_t st) {
  switch (W) {
    case 32: if constexpr (sizeof(T) == 4) return keyw_cols<T, 32>(a, p, st); break;
    case 64: return keyw_cols<T, 64>(a, p, st);
    case 128: return keyw_cols<T, 128>(a, p, st);
    case 256: return keyw_cols<T, 256>(a, p, st);
  }
  return fail(KAT_EUNSUPPORTED, "kat_attn_key_weights: head dim %d", a.D);
}

}  // namespace kat

using namespace kat;

extern "C" size_t kat_attn_key_weights_workspace_size(int64_t B, int64_t H, int64_t T, int64_t D, int64_t last,
                                                      int dtype) {
  const int W = keyw_layout(D, dtype);
  if (B <= 0 || H <= 0 || T <= 0 || last < 0 || !W) return 0;
  const int chunks = keyw_plan(B, H, T, last == 0 ? 0 : std::max<int64_t>(0, T - last), W, dtype).chunks;
  return chunks == 1 ? 0 : (size_t)chunks * B * H * T * sizeof(float);
}

extern "C" int kat_attn_key_weights(const void* q, const void* k, const float* L, float* weights,
                                    const float* slopes, const uint8_t* token_mask, int64_t mask_stride_b,
                                    void* workspace, size_t workspace_bytes, int64_t B, int64_t H, int64_t T,
                                    int64_t D, int64_t last, const int64_t* strides, float scale, float eps,
                                    int dtype, void* stream) {
  const char* nm = "kat_attn_key_weights";
  if (B < 0 || H < 0 || T < 0 || D < 0 || last < 0) return fail(KAT_EINVAL, "%s: negative size", nm);
  if (B > 0xffff || H > 0xffff || B * H > 0xffff || T > 0x3fffff)
    return fail(KAT_EUNSUPPORTED, "%s: B*H or T too large", nm);
  const int W = keyw_layout(D, dtype);
  if (!W) return fail(KAT_EUNSUPPORTED, "%s: head dim %lld with dtype %d", nm, (long long)D, dtype);
  if (B * H * T == 0) return KAT_OK;
  if (!q || !k || !L || !weights || !slopes || !strides) return fail(KAT_EINVAL, "%s: null pointer", nm);
  const int esz = dtype_size(dtype);
  int64_t st6[6];
  for (int t = 0; t < 6; ++t) {
    const int64_t size[3] = {B, H, T};
    st6[t] = dim_stride(strides[t], size[t % 3]);
    if ((st6[t] * esz) % 16 != 0) return fail(KAT_EUNSUPPORTED, "%s: strides must keep rows 16-byte aligned", nm);
  }
  if (!aligned16(q) || !aligned16(k)) return fail(KAT_EUNSUPPORTED, "%s: tensors must be 16-byte aligned", nm);
  if (T > 1 && (st6[2] < D || st6[5] < D)) return fail(KAT_EINVAL, "%s: row stride < D", nm);
  // a tile's rows are addressed by 31-bit byte offsets
  if (st6[2] > 0x7fffffff / (64 * esz)) return fail(KAT_EUNSUPPORTED, "%s: q row stride too large", nm);
  KeywArgs a = {};
  a.q = q;
  a.k = k;
  a.L = L;
  a.out = weights;
  a.slopes = slopes;
  a.mask = token_mask;
  a.smask = mask_stride_b;
  a.B = (int)B;
  a.H = (int)H;
  a.T = (int)T;
  a.D = (int)D;
  a.lo = last == 0 ? 0 : (int)std::max<int64_t>(0, T - last);
  for (int i = 0; i < 3; ++i) {
    a.sq[i] = st6[i];
    a.sk[i] = st6[3 + i];
    a.sl[i] = strides[6 + i];
  }
  if (T == 1) a.sq[2] = D;
  a.so[0] = strides[9];
  a.so[1] = strides[10];
  a.scale = scale;
  a.eps = eps;
  const KeywPlan p = keyw_plan(B, H, T, a.lo, W, dtype);
  a.qc = p.qc;
  a.chunks = p.chunks;
  const size_t need = kat_attn_key_weights_workspace_size(B, H, T, D, last, dtype);
  if (need && (!workspace || workspace_bytes < need))
    return fail(KAT_EINVAL, "%s: workspace %zu bytes < required %zu", nm, workspace_bytes, need);
  a.part = need ? (float*)workspace : nullptr;
  if (a.chunks > 0xffff || (T + 15) / 16 * B * H > 0x7fffffff) return fail(KAT_EUNSUPPORTED, "%s: B*H*T too large", nm);
  const hipStream_t st = as_stream(stream);
  switch (dtype) {
    case KAT_F32: return keyw_w<float>(a, W, p, st);
    case KAT_BF16: return keyw_w<bf16>(a, W, p, st);
    case KAT_F16: return keyw_w<f16>(a, W, p, st);
  }
  return fail(KAT_EUNSUPPORTED, "%s: unsupported dtype %d", nm, dtype);
}
