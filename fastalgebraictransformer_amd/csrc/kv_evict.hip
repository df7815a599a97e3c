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
// Design: a selection per (b, h), then its moves at the copy rate. Into another
// cache it is one launch: every block of a (b, h) selects for itself (the selection
// takes no longer for being done on several CUs at once) and moves its share of
// the rows. In place the blocks would write the totals that others still read, so
// there a plan kernel writes the list of moves and a second one moves the rows.
// The selection is latency-bound (8 bytes per row): totals become unsigned
// keys in the order of the numbers, held in registers (each wave a contiguous run
// of rows), and the m-th largest key is found in three histograms of its bits
// (11, 11 and 10 bits, most significant first; LDS integer atomics, whose order
// does not matter). The first digit takes the sign, the exponent and two bits of
// the significand, so that totals within a few octaves do not all meet in one
// counter. Ties and the list's order come from ballots and prefix sums over the
// waves' runs. Finding the key bit by bit instead (a ballot per 64 keys and a
// barrier per bit) took 68 us for 32768 rows and 11.5 us for 640; plan and moves
// in two launches 21 us at B=16, H=12, T=2048, D=64, keep 512 and 105 us at B=4,
// H=16, T=32768, D=128, keep 4096 (bf16).

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
  int B, H, T, keep, recent;
  int pieces;  // 16-byte pieces of a row
  // bytes: k, v, ko, vo (b, h, t); elements: w, pos, wo, po (b, h)
  int64_t sk[3], sv[3], sko[3], svo[3], sw[2], spos[2], swo[2], spo[2];
  int share;     // rows per block, in one launch
  int32_t* src;  // [B*H][keep] rows to move, in order
  int32_t* dst;  // [B*H][keep] where to (in place)
  int32_t* cnt;  // [B*H]
};

// set bits of the lanes below this one
__device__ __forceinline__ int bits_below(uint64_t m) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// x plus the lanes below (DPP: shifts within rows of 16 lanes, then the rows'
// last lanes broadcast onwards)
__device__ __forceinline__ uint32_t scan_lanes(uint32_t x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ int sum_lanes(int x) { return __builtin_amdgcn_readlane((int)scan_lanes((uint32_t)x), 63); }

// rows first .. last - 1 of a (b, h)'s list of moves, by NT threads from thread t
// on: source rows src[r - first], destinations dst (nullptr: the place in the list)
template <int NT>
__device__ __forceinline__ void move_rows(const EvictArgs& a, int b, int h, int first, int last, const int32_t* src,
                                          const int32_t* dst) {
  const int t = threadIdx.x;
  auto to = [&](int i) __attribute__((always_inline)) { return dst ? dst[i] : first + i; };
  const int rows = last - first;
  // the totals and positions: their loads run beside those of the first pieces
  const float* w = a.w + b * a.sw[0] + h * a.sw[1];
  const int32_t* pos = a.pos + b * a.spos[0] + h * a.spos[1];
  float* wo = a.wo + b * a.swo[0] + h * a.swo[1];
  int32_t* po = a.po + b * a.spo[0] + h * a.spo[1];
  float w0 = 0.f;
  int32_t p0 = 0;
  if (t < rows) {
    w0 = w[src[t]];
    p0 = pos[src[t]];
  }
  const char* k = a.k + b * a.sk[0] + h * a.sk[1];
  const char* v = a.v + b * a.sv[0] + h * a.sv[1];
  char* ko = a.ko + b * a.sko[0] + h * a.sko[1];
  char* vo = a.vo + b * a.svo[0] + h * a.svo[1];
  constexpr int U = 4;  // pieces in flight per thread, of k and of v
  const int per = a.pieces;
  const int all = rows * per;  // (at most kEvShare rows of 2^15 pieces)
  for (int i0 = t; i0 < all; i0 += NT * U) {
    mfma::i16x8 x[U], y[U];
    int at[U], pc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * NT;
      const bool in = i < all;
      const int r = in ? (int)((uint32_t)i / (uint32_t)per) : 0;
      pc[u] = in ? i - r * per : -1;
      at[u] = to(r);
      if (in) {
        const int s = src[r];
        x[u] = ld_piece_nt(k + (int64_t)s * a.sk[2] + 16 * pc[u]);
        y[u] = ld_piece_nt(v + (int64_t)s * a.sv[2] + 16 * pc[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (pc[u] >= 0) {
        *reinterpret_cast<mfma::i16x8*>(ko + (int64_t)at[u] * a.sko[2] + 16 * pc[u]) = x[u];
        *reinterpret_cast<mfma::i16x8*>(vo + (int64_t)at[u] * a.svo[2] + 16 * pc[u]) = y[u];
      }
  }
  if (t < rows) {
    wo[to(t)] = w0;
    po[to(t)] = p0;
  }
  for (int i = t + NT; i < rows; i += NT) {
    wo[to(i)] = w[src[i]];
    po[to(i)] = pos[src[i]];
  }
}

constexpr int kEvBins = 2048;
constexpr int kEvShare = 4096;  // most rows that a block moves in one launch

// NT threads; R: keys per thread held in registers (T <= NT R); 0: any T, the
// keys are formed again from memory each time. ONE: one launch, block (share,
// b h) moves rows share a.share .. to the outputs; else, in place, block (0, b h)
// writes the list of moves
template <int NT, int R, bool ONE> __global__ __launch_bounds__(NT) void kv_evict_plan_k(EvictArgs a) {
  constexpr int NW = NT / 64, BPT = kEvBins / NT;  // waves; bins per thread
  __shared__ uint32_t hist[kEvBins];
  __shared__ uint32_t wsum[NW];
  __shared__ uint32_t found[3];
  __shared__ int tot[3][NW];
  __shared__ int32_t list[ONE ? kEvShare : 1];
  const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
  const int lane = threadIdx.x & 63, wv = mfma::wave_id();
  int n = a.len ? a.len[b] : a.T;
  n = min(max(n, 0), a.T);
  const int m = min(n, a.keep);
  const float* w = a.w + b * a.sw[0] + h * a.sw[1];
  const int32_t* pos = a.pos + b * a.spos[0] + h * a.spos[1];
  // rows with a position from `edge` on are the newest (positions as unsigned
  // numbers in their order; past the last one: none)
  const int64_t edge64 = n > 0 ? (int64_t)pos[n - 1] - a.recent + 1 + 0x80000000ll : 0;
  const uint32_t edge = (uint32_t)min(max(edge64, (int64_t)0), (int64_t)0xffffffffll);
  const bool newest = edge64 <= 0xffffffffll;

  // wave wv owns rows run .. run + seg - 1, 64 at a time
  const int seg = R ? 64 * R : ((n + NT - 1) / NT) * 64;
  const int run = wv * seg;
  const int end = min(run + seg, n);
  auto rank = [&](float x, int32_t p) __attribute__((always_inline)) -> uint32_t {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 as 0
    uint32_t o = (u >> 31) ? ~u : (u | 0x80000000u);
    o = min(max(o, 1u), 0xfffffffeu);  // 0: no row; 2^32 - 1: a newest one
    if ((u & 0x7fffffffu) > 0x7f800000u) o = 0xfffffffeu;
    return newest && ((uint32_t)p ^ 0x80000000u) >= edge ? 0xffffffffu : o;
  };
  uint32_t kr[R ? R : 1];
  if constexpr (R > 0) {
    float x[R];
    int32_t p[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int j = min(run + i * 64 + lane, a.T - 1);  // (does not wait for the length)
      x[i] = w[j];
      p[i] = pos[j];
    }
#pragma unroll
    for (int i = 0; i < R; ++i) kr[i] = run + i * 64 + lane < end ? rank(x[i], p[i]) : 0u;
  }
  // f(key, row) for the wave's rows in order, all lanes together
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i) f(kr[i], run + i * 64 + lane);
    } else {
      for (int j = run; j < end; j += 64) f(j + lane < end ? rank(w[j + lane], pos[j + lane]) : 0u, j + lane);
    }
  };

  // the m-th largest key, and how many rows with that key stay, of how many
  uint32_t tau = 1;
  int ties = n, equal = n;
  if (m == 0) {
    tau = 0xffffffffu;
    ties = 0;
  } else if (m < n) {
    int need = m;
    tau = 0;
#pragma unroll
    for (int round = 0; round < 3; ++round) {
      constexpr int kShift[3] = {21, 10, 0};
      const int sh = kShift[round], nb = round == 2 ? 1024 : 2048;
      for (int i = threadIdx.x; i < nb; i += NT) hist[i] = 0;
      __syncthreads();
      // counters in falling order of the digit
      each([&](uint32_t x, int) {
        if (x != 0u && (round == 0 || (x >> kShift[round ? round - 1 : 0]) == (tau >> kShift[round ? round - 1 : 0])))
          atomicAdd(&hist[nb - 1 - ((x >> sh) & (nb - 1))], 1u);
      });
      __syncthreads();
      uint32_t c[BPT], s = 0;
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        const int bin = threadIdx.x * BPT + i;
        c[i] = bin < nb ? hist[bin] : 0u;
        s += c[i];
      }
      const uint32_t incl = scan_lanes(s);  // over the threads up to this one
      if (lane == 63) wsum[wv] = incl;
      __syncthreads();
      uint32_t before = incl - s;
#pragma unroll
      for (int i = 0; i < NW; ++i) before += i < wv ? wsum[i] : 0u;
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        if (before < (uint32_t)need && (uint32_t)need <= before + c[i]) {  // one bin of one thread
          found[0] = nb - 1 - (threadIdx.x * BPT + i);
          found[1] = before;
          found[2] = c[i];
        }
        before += c[i];
      }
      __syncthreads();
      tau |= found[0] << sh;
      need -= (int)found[1];
      equal = (int)found[2];
    }
    ties = need;
  }

  // the moves: kept rows (in place: those at or past m), in order; and in place
  // the rows below m that are given up
  int eq0 = 0;  // rows with the key tau in the waves before
  if (ties != equal) {
    int eq = 0;
    each([&](uint32_t x, int) { eq += x == tau; });
    eq = sum_lanes(eq);
    if (lane == 0) tot[0][wv] = eq;
    __syncthreads();
    for (int i = 0; i < wv; ++i) eq0 += tot[0][i];
  }
  // f(kept, row); rows with the key tau stay while fewer than `ties` came before
  auto each_kept = [&](auto f) __attribute__((always_inline)) {
    if (ties == equal) {
      each([&](uint32_t x, int j) { f(x >= tau, j); });
    } else {
      int e = eq0;
      each([&](uint32_t x, int j) {
        const uint64_t q = __builtin_amdgcn_ballot_w64(x == tau);
        f(x > tau || (x == tau && e + bits_below(q) < ties), j);
        e += __popcll(q);
      });
    }
  };
  // the place of a wave's first move (hole): those of the waves before
  auto before = [&](int mine, int* t) __attribute__((always_inline)) {
    mine = sum_lanes(mine);
    if (lane == 0) t[wv] = mine;
    __syncthreads();
    int c = 0;
    for (int i = 0; i < wv; ++i) c += t[i];
    return c;
  };
  if constexpr (ONE) {
    int nm = 0;
    each_kept([&](bool y, int) { nm += y; });
    int m0 = before(nm, tot[1]);
    const int m1 = m0 + tot[1][wv];
    const int first = (int)blockIdx.x * a.share, last = min(first + a.share, m);
    if (m0 < last && m1 > first) {  // else this wave's rows are other blocks'
      each_kept([&](bool y, int j) {
        const uint64_t mm = __builtin_amdgcn_ballot_w64(y);
        const int r = m0 + bits_below(mm) - first;
        if (y && r >= 0 && r < last - first) list[r] = j;
        m0 += __popcll(mm);
      });
    }
    __syncthreads();
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0 && a.lo) a.lo[b] = m;
    move_rows<NT>(a, b, h, first, last, list, nullptr);
  } else {
    int nm = 0, nh = 0;
    each_kept([&](bool y, int j) {
      nm += y && j >= m;
      nh += !y && j < m;
    });
    int m0 = before(nm, tot[1]), h0 = before(nh, tot[2]);
    int32_t* src = a.src + (int64_t)bh * a.keep;
    int32_t* dst = a.dst + (int64_t)bh * a.keep;
    each_kept([&](bool y, int j) {
      const bool mv = y && j >= m, ho = !y && j < m;
      const uint64_t mm = __builtin_amdgcn_ballot_w64(mv), hm = __builtin_amdgcn_ballot_w64(ho);
      if (mv) src[m0 + bits_below(mm)] = j;
      if (ho) dst[h0 + bits_below(hm)] = j;
      m0 += __popcll(mm);
      h0 += __popcll(hm);
    });
    if (wv == NW - 1 && lane == 0) a.cnt[bh] = m0;
  }
}

constexpr int kMvThreads = 256;
constexpr int kMvRows = 32;  // rows per block

__global__ __launch_bounds__(kMvThreads) void kv_evict_move_k(EvictArgs a) {
  const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0 && a.lo) {
    const int n = a.len ? a.len[b] : a.T;
    a.lo[b] = min(min(max(n, 0), a.T), a.keep);
  }
  const int r0 = (int)blockIdx.x * kMvRows, r1 = min(r0 + kMvRows, a.cnt[bh]);
  if (r0 >= r1) return;
  const int64_t at = (int64_t)bh * a.keep + r0;
  move_rows<kMvThreads>(a, b, h, r0, r1, a.src + at, a.dst + at);
}

template <int NT, int R> static int launch_evict(const EvictArgs& a, bool one, hipStream_t st) {
  const unsigned bh = (unsigned)(a.B * a.H);
  if (one) {
    const unsigned nb = (unsigned)std::max(1, (std::min(a.keep, a.T) + a.share - 1) / a.share);
    hipLaunchKernelGGL((kv_evict_plan_k<NT, R, true>), dim3(nb, bh), dim3(NT), 0, st, a);
    return check_launch("kat_kv_evict");
  }
  hipLaunchKernelGGL((kv_evict_plan_k<NT, R, false>), dim3(1, bh), dim3(NT), 0, st, a);
  if (int rc = check_launch("kat_kv_evict (plan)")) return rc;
  const int64_t most = std::min<int64_t>(a.keep, std::max(0, a.T - a.keep));  // holes, and rows past them
  const unsigned nb = (unsigned)std::max<int64_t>(1, (most + kMvRows - 1) / kMvRows);
  hipLaunchKernelGGL(kv_evict_move_k, dim3(nb, bh), dim3(kMvThreads), 0, st, a);
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
  if (!esz || D == 0 || D > 0xffff || (D * esz) % 16 != 0)
    return fail(KAT_EUNSUPPORTED, "%s: head dim %lld with dtype %d (rows of whole 16-byte pieces)", nm, (long long)D, dtype);
  if (B * H * T == 0) return KAT_OK;
  if (!k || !v || !weights || !positions || !k_out || !v_out || !weights_out || !positions_out || !strides)
    return fail(KAT_EINVAL, "%s: null pointer", nm);
  if (in_place && (k != k_out || v != v_out || weights != weights_out || positions != positions_out))
    return fail(KAT_EINVAL, "%s: in place, but the outputs are other tensors", nm);
  int64_t st12[12];
  for (int t = 0; t < 12; ++t) {
    const int64_t size[3] = {B, H, t < 6 ? T : std::min(keep, T)};
    st12[t] = dim_stride(strides[t], size[t % 3]);
    if ((st12[t] * esz) % 16 != 0) return fail(KAT_EUNSUPPORTED, "%s: strides must keep rows 16-byte aligned", nm);
  }
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_out) || !aligned16(v_out))
    return fail(KAT_EUNSUPPORTED, "%s: tensors must be 16-byte aligned", nm);
  if (!in_place && lengths_out && lengths_out == lengths)
    return fail(KAT_EINVAL, "%s: lengths_out must be another tensor than lengths, unless in place", nm);
  const size_t need = in_place ? kat_kv_evict_workspace_size(B, H, keep) : 0;
  if (need && (!workspace || workspace_bytes < need))
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
  a.pieces = (int)(D * esz / 16);
  for (int i = 0; i < 3; ++i) {
    a.sk[i] = st12[i] * esz;
    a.sv[i] = st12[3 + i] * esz;
    a.sko[i] = st12[6 + i] * esz;
    a.svo[i] = st12[9 + i] * esz;
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
  const bool one = !in_place;
  // a block per CU (each selects anew, so a second one on a CU costs more than it
  // brings: 23 against 18.6 us at B=16, H=12, T=2048, keep 512), at least 32 rows each
  const int64_t want = std::max<int64_t>(1, num_cus() / (B * H)), rows = std::max<int64_t>(1, std::min(keep, T));
  a.share = (int)std::min<int64_t>(kEvShare, std::max<int64_t>(32, (rows + want - 1) / want));
  // waves enough that a thread holds few keys (640 rows: 256 threads of 4 keys 6.6 us,
  // 512 of 2 5.9, 1024 of 1 6.3; 2048 rows: 1024 of 2 7.1, 512 of 8 7.8, 256 of 16 9.7)
  if (T <= 1024) return launch_evict<512, 2>(a, one, st);
  if (T <= 2048) return launch_evict<1024, 2>(a, one, st);
  if (T <= 4096) return launch_evict<1024, 4>(a, one, st);
  if (T <= 16384) return launch_evict<1024, 16>(a, one, st);
  if (T <= 32768) return launch_evict<1024, 32>(a, one, st);
  return launch_evict<1024, 0>(a, one, st);
}
