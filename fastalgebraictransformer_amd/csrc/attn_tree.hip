// Attention of a tree of drafted tokens over a KV cache on gfx950: the pass
// that scores all drafted tokens of speculative decoding at once.
//
// Per (b, h) the cache holds n = lengths[b] rows, the last N of them the keys
// and values of the drafted tokens: token i sits in row c + i, c = n - N. Token
// i hangs on token parents[i] < i, or on the context (-1); any other value
// marks an absent token, and so is every token below one. With anc(i) the
// tokens from the root to i (i included), token i attends to the rows j < c and
// to c + j, j in anc(i):
//   s = scale <q_i, k_j> - slope_h (p_i - p_j),  f = sigma(s)^4,
//   L_i = sum f,  o_i = sum f v_j / (L_i + eps)
// where a row's position p is its index (context) or c + depth (tokens), or is
// given (caches whose rows have been evicted). One token, N = 1, is the decode.
// Absent tokens get o = 0, L = 0.
//
// Design (MI355X). Every cache row is read once for all N queries, so HBM
// bounds the call: 2 D dtype bytes and 4 N D flops per row, N = 64 in bf16 64
// flops per byte against the card's ~230. As in the decode, the rows are split
// into chunks, one block each, and sigma^4 needs no running maximum: blocks
// write plain sums and a second kernel adds them in a fixed order.
//
// A block streams its rows through LDS in tiles of 64 (LDS-DMA, a ring of
// NS stages, non-temporal: each row is used once), so rows in flight hold no
// registers. Its waves form QG query groups of 16 QT queries and KG row groups of a
// tile:
//   S^T[row][q] = K Q^T    A = K (LDS rows)             B = Q^T (registers)
//   f of S^T               lane (g, li) holds rows 4 g + j, query li
//   O^T[d][q] += V^T f^T   A = V^T (LDS, transposed reads)  B = f in two parts of
//                          the dtype (Split), or fp32
// A first version gave every wave whole rows for all queries, loaded straight
// into registers: at 64 queries the accumulators and fragments (192 registers)
// left no room for the rows in flight, and it spilled (578 us at B=8, H=16, N=64,
// T=8192, D=128, bf16).
// Only tiles that reach the tokens' rows (two or three) look at the ancestor
// masks, which each block derives from the parents by pointer doubling, one
// lane per token.

#include <algorithm>
#include <type_traits>

#include "attn_cache.h"
#include "kat_internal.h"

namespace kat {

using namespace mfma;

struct TreeArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* L;                  // [B*H*N] or nullptr
  const float* slopes;       // [H]
  const int32_t* parents;    // [B, N]: row b at parents + b * spar
  const int32_t* lengths;    // [B] or nullptr (all T)
  const int32_t* positions;  // [B, H, T] or nullptr
  int B, H, N, T, D;
  int64_t sq[3], sk[3], sv[3], so[3], spar, spos[2];
  float scale, eps;
  int splits;
  float* part;   // [B*H*splits][N][W] sums f v (W the layout width), 16 sigma^4 as f
  float* lpart;  // [B*H*splits][N] sums f
};

constexpr int kTreeMax = 64;  // tokens: one ancestor mask is one 64-bit word
// How a block is laid out, by a row's 16-bit units U and the number NQ of 16-query
// subtiles (1, 2 or 4): rows of a tile, waves, stages of the ring (a stage is 4 U
// bytes per row, of the CU's 160 KB of LDS), blocks per CU, and subtiles per wave.
//  - Eight waves run on a CU, in one block where the registers allow it: it streams one
//    ring four stages deep and leaves half the partial sums. B=8, H=16, N=64, T=8192,
//    D=128, bf16 (weights rounded once): one block of eight 90 us, two of four waves
//    with rings of two stages 103. At U = 256 eight waves of 64 queries would spill, and
//    with 32 queries at U = 128 they leave each wave few rows: four waves there, on
//    tiles of 32 rows. B=4, H=16, N=64, T=2048, D=256 tiles of 32 / 64 rows 41 / 43; B=3,
//    H=16, N=25, T=1999, D=96 four / eight waves 16.8 / 19.1. A wave has 16 rows of a
//    tile at least.
//  - With 64 queries two subtiles per wave, which share its reads of K and V (one / two:
//    B=16, H=12, T=4096, D=64 63.5 / 61.2, B=8, H=16, T=8192, D=128 107 / 105).
struct TreeShape {
  int rows, waves, stages, blocks, qt;
};
constexpr TreeShape tree_shape(int U, int NQ) {
  return U <= 64 ? TreeShape{64, NQ == 1 ? 4 : 8, 4, NQ == 1 ? 2 : 1, NQ == 4 ? 2 : 1}
         : NQ == 1 ? TreeShape{64, 4, 2, U == 128 ? 2 : 1, 1}
         : U == 128 && NQ == 4 ? TreeShape{64, 8, 4, 1, 2}
                               : TreeShape{32, 4, 4, U == 128 ? 2 : 1, 1};
}
constexpr int tree_nq(int64_t N) { return N <= 16 ? 1 : N <= 32 ? 2 : 4; }

// Two fp32 weights as packed pairs of T, the rounded values and what the rounding
// left: the product with V then has the weights to 16 bits (bf16; 22 in fp16) and o
// is rounded once, when it is stored. With the rounded weights alone, one rounding of
// a weight near 1 moves a whole row of o by up to half a step of T (1.4 to 1.7 times
// the error of o against 64 bits). B=8, H=16, T=8192, D=128, bf16, rounded / split: 64
// tokens 95 / 103 us, 32 99 / 99, 16 94 / 94.
template <typename T> struct Split {
  uint32_t hi, lo;
  __device__ __forceinline__ Split(float x, float y) {
    hi = mfma::Mfma<T>::pack2(x, y);
    if constexpr (__is_same(T, bf16)) {
      lo = mfma::Mfma<T>::pack2(x - __builtin_bit_cast(float, hi << 16), y - __builtin_bit_cast(float, hi & 0xffff0000u));
    } else {
      const VecT<f16, 2> h = __builtin_bit_cast(VecT<f16, 2>, hi);
      lo = mfma::Mfma<T>::pack2(x - (float)h.v[0], y - (float)h.v[1]);
    }
  }
};

template <typename T, int W, int NQ> constexpr TreeShape tree_at() { return tree_shape(W * (int)sizeof(T) / 2, NQ); }

template <typename T, int W, int NQ, bool POS>
__global__ __launch_bounds__((64 * tree_at<T, W, NQ>().waves), (tree_at<T, W, NQ>().waves * tree_at<T, W, NQ>().blocks / 4))
void attn_tree_k(TreeArgs a) {
  constexpr int ES = (int)sizeof(T);
  constexpr int U = W * ES / 2;          // a row in 16-bit units, the unit of the tile helpers
  constexpr int KK = U / 32;             // 64-byte column blocks
  constexpr int DS = W / 16;             // 16-wide d subtiles
  constexpr TreeShape S = tree_at<T, W, NQ>();
  constexpr int NW = S.waves, TR = S.rows, NS = S.stages, QT = S.qt;
  constexpr int QG = NQ / QT;            // query groups
  constexpr int KG = NW / QG;            // row groups of a tile
  constexpr int TK = TR / KG;            // rows of a wave's group
  typedef TileDma<U, NW, TR> Dma;
  constexpr int OPS = 2 * Dma::SEGS + (POS ? 1 : 0);  // a wave's DMA operations per tile
  constexpr int RING = NS * 2 * TR * U;
  static_assert(TK >= 16 && RING * 2 >= NW * DS * QT * 1024, "the ring holds the waves' sums");
  __shared__ __align__(16) short ring[RING];
  __shared__ int spos[POS ? NS : 1][NW][64];  // (a DMA writes 64 words)
  __shared__ float sl[NW][16 * QT];
  __shared__ uint64_t sanc[kTreeMax];  // ancestors of token i, itself included; 0 if absent
  __shared__ int sdep[kTreeMax];       // depth of token i below the context

  const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
  const int split = blockIdx.x;
  const int lane = threadIdx.x & 63, w = wave_id();
  const int g = lane >> 4, li = lane & 15;
  const int qg = w % QG, kg = w / QG;
  const int N = a.N;
  const float slope = a.slopes[h], scale = a.scale;
  // what does not wait for the length: the queries and the parents
  const int cols = a.D * ES / 16;  // 16-byte pieces of a row that hold columns
  const int qi = 16 * QT * qg + li;  // the lane's token of the first subtile; + 16 of the next
  i16x8 qf[QT][KK];
#pragma unroll
  for (int qs = 0; qs < QT; ++qs)
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int p = 4 * kk + g, i = qi + 16 * qs;
      qf[qs][kk] = i16x8{0, 0, 0, 0, 0, 0, 0, 0};
      if (i < N && p < cols)
        qf[qs][kk] = *reinterpret_cast<const i16x8*>(
            (const char*)((const T*)a.q + b * a.sq[0] + h * a.sq[1] + i * a.sq[2]) + 16 * p);
    }
  const int parent = w == 0 && lane < N ? a.parents[b * a.spar + lane] : -2;
  int n = a.lengths ? a.lengths[b] : a.T;
  n = min(n, a.T);
  const int c = n - N;       // rows of the context
  if (c < 0) n = 0;          // no room for the tokens: the row holds no draft

  const char* kp = (const char*)((const T*)a.k + b * a.sk[0] + h * a.sk[1]);
  const char* vp = (const char*)((const T*)a.v + b * a.sv[0] + h * a.sv[1]);
  const int64_t skb = a.sk[2] * ES, svb = a.sv[2] * ES;
  const int32_t* pp = POS ? a.positions + b * a.spos[0] + h * a.spos[1] : nullptr;

  // this split's tiles
  const int nt = (n + TR - 1) / TR;
  const int per = (nt + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(t0 + per, nt);

  Dma dk, dv;
  dk.init(w, lane, (uint32_t)(skb / 2), a.D * ES / 2);
  dv.init(w, lane, (uint32_t)(svb / 2), a.D * ES / 2);
  // rows past the last filled one, and columns past the head dim, read as zeros
  auto issue = [&](int t) __attribute__((always_inline)) {
    const int row = t * TR, st = (t - t0) % NS;
    short* const kt = ring + st * 2 * TR * U;
    const int64_t left = (int64_t)(n - 1 - row), lim = 0x7fffffff;
    dk.template issue_rows<true>(kt, kp + row * skb, (uint32_t)min(left * skb + a.D * ES, lim), w);
    dv.template issue_rows<true>(kt + TR * U, vp + row * svb, (uint32_t)min(left * svb + a.D * ES, lim), w);
    if constexpr (POS)
      dma4(rsrc_words(pp + row, (uint32_t)min(left + 1, (int64_t)TR) * 4), lds_addr(&spos[st][w][0]), (uint32_t)lane * 4);
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (t0 + i < t1) issue(t0 + i);

  if (w == 0) {
    // pointer doubling: after step i, anc holds the 2^i nearest ancestors and
    // up the one above them (-1: the context is reached)
    int up = parent;
    bool ok = c >= 0 && up >= -1 && up < lane;
    if (!ok) up = -1;
    uint64_t anc = 1ull << lane;
#pragma unroll
    for (int st = 0; st < 6; ++st) {
      const int src = up < 0 ? lane : up;
      const uint32_t lo = __shfl((uint32_t)anc, src, 64), hi = __shfl((uint32_t)(anc >> 32), src, 64);
      const int up2 = __shfl(up, src, 64);
      const bool ok2 = (bool)__shfl((int)ok, src, 64);
      if (up >= 0) {
        anc |= ((uint64_t)hi << 32) | lo;
        ok = ok && ok2;
        up = up2;
      }
    }
    sanc[lane] = ok ? anc : 0ull;
    sdep[lane] = __popcll(anc) - 1;
  }

  __syncthreads();  // masks and depths
  uint64_t anc[QT];
  int qpos[QT];
#pragma unroll
  for (int qs = 0; qs < QT; ++qs) {
    const int i = qi + 16 * qs;
    anc[qs] = i < N ? sanc[i] : 0ull;
    qpos[qs] = 0;
    if (i < N && n > 0) qpos[qs] = POS ? pp[c + i] : c + sdep[i];
  }

  const float sj[4] = {0.f, slope, 2.f * slope, 3.f * slope};
  f32x4 oacc[DS][QT];
  float lsum[QT];
#pragma unroll
  for (int qs = 0; qs < QT; ++qs) {
    lsum[qs] = 0.f;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) oacc[ds][qs] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // 16 rows at tile row hr (row k0 + hr of the cache) against the wave's
  // queries: f of S^T. TAIL: the tile reaches the tokens' rows or the end
  auto scores = [&](auto tail_tag, int k0, int hr, const short* kt, const int* pt, f32x4 (&f)[QT]) __attribute__((always_inline)) {
    constexpr bool TAIL = decltype(tail_tag)::value;
#pragma unroll
    for (int qs = 0; qs < QT; ++qs) f[qs] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const i16x8 kf = lds16(kt + soff<U>(hr + li, 32 * kk + 8 * g));
#pragma unroll
      for (int qs = 0; qs < QT; ++qs) f[qs] = dot64<T>(kf, qf[qs][kk], f[qs]);
    }
    i32x4 kpos;
    if constexpr (POS) kpos = *reinterpret_cast<const i32x4*>(pt + hr + 4 * g);
#pragma unroll
    for (int qs = 0; qs < QT; ++qs) {
      // (context rows that are positions: the lane's first one; the others lie j on)
      const float bias0 = -slope * (float)(qpos[qs] - (k0 + hr + 4 * g));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tok = k0 + hr + 4 * g + j - c;  // the drafted token in this row, if >= 0
        float bias;
        if constexpr (POS) bias = -slope * (float)(qpos[qs] - kpos[j]);
        else if constexpr (TAIL) bias = -slope * (float)(qpos[qs] - (tok < 0 ? c + tok : c + sdep[min(tok, kTreeMax - 1)]));
        else bias = j ? bias0 + sj[j] : bias0;
        const float s = fmaf(f[qs][j], scale, bias);
        float x;
        if constexpr (ES == 4) {
          x = sig2_pow4(s);
        } else {
          // 1 + s r: two instructions less (B=8, H=16, N=64, T=8192, D=128 103 us, 110
          // with sig2); its relative error, some 2^-22 (1 + |s|), grows only where f is
          // small against the sums it enters
          const float t = fmaf(s, __builtin_amdgcn_rcpf(fabsf(s) + 1.f), 1.f), t2 = t * t;
          x = t2 * t2;
        }
        if constexpr (TAIL) {
          const bool seen = tok < 0 ? anc[qs] != 0ull : tok < N && ((anc[qs] >> (tok & 63)) & 1ull);
          x = seen ? x : 0.f;
        }
        f[qs][j] = x;
      }
      lsum[qs] += (f[qs][0] + f[qs][1]) + (f[qs][2] + f[qs][3]);
    }
  };
  // O^T += V^T f^T over the 32 rows at tile row hr (x: the first 16, y), or over 16
  auto product32 = [&](int hr, const f32x4 (&x)[QT], const f32x4 (&y)[QT], const short* vt) __attribute__((always_inline)) {
    if constexpr (ES == 2) {
      i16x8 ph[QT], pl[QT];
#pragma unroll
      for (int qs = 0; qs < QT; ++qs) {
        const Split<T> a0(x[qs][0], x[qs][1]), a1(x[qs][2], x[qs][3]), b0(y[qs][0], y[qs][1]), b1(y[qs][2], y[qs][3]);
        ph[qs] = pack_frag(a0.hi, a1.hi, b0.hi, b1.hi);
        pl[qs] = pack_frag(a0.lo, a1.lo, b0.lo, b1.lo);
      }
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        const i16x8 vf = frag_tr<U>(vt, hr, 16 * ds, g, li);
#pragma unroll
        for (int qs = 0; qs < QT; ++qs) oacc[ds][qs] = Mfma<T>::mma(vf, ph[qs], oacc[ds][qs]);
#pragma unroll
        for (int qs = 0; qs < QT; ++qs) oacc[ds][qs] = Mfma<T>::mma(vf, pl[qs], oacc[ds][qs]);
      }
    }
  };
  auto product16 = [&](int hr, const f32x4 (&x)[QT], const short* vt) __attribute__((always_inline)) {
    if constexpr (ES == 4) {
#pragma unroll
      for (int ds = 0; ds < DS; ++ds)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float vf = *reinterpret_cast<const float*>(vt + soff<U>(hr + 4 * g + j, 32 * ds + 2 * li));
#pragma unroll
          for (int qs = 0; qs < QT; ++qs)
            oacc[ds][qs] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf, x[qs][j], oacc[ds][qs], 0, 0, 0);
        }
    } else {
      // one product takes both parts of the weights: 32 k-indices, the rows twice
      i16x8 p[QT];
#pragma unroll
      for (int qs = 0; qs < QT; ++qs) {
        const Split<T> a0(x[qs][0], x[qs][1]), a1(x[qs][2], x[qs][3]);
        p[qs] = pack_frag(a0.hi, a1.hi, a0.lo, a1.lo);
      }
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        const i16x4 v = lds_tr(vt + soff<U>(hr + 4 * g + (li >> 2), 16 * ds + 4 * (li & 3)));
        const i16x8 vf = i16x8{v[0], v[1], v[2], v[3], v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int qs = 0; qs < QT; ++qs) oacc[ds][qs] = Mfma<T>::mma(vf, p[qs], oacc[ds][qs]);
      }
    }
  };
  // the same without 0 x inf: rows with f = 0 add nothing
  auto product_checked = [&](int hr, const f32x4 (&x)[QT], const short* vt) __attribute__((always_inline)) {
    for (int r = 0; r < 16; ++r) {
      const int src = (r >> 2) * 16 + li;  // the lane that holds this row's f of query li
#pragma unroll
      for (int qs = 0; qs < QT; ++qs) {
        float y = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float z = __shfl(x[qs][j], src, 64);
          if ((r & 3) == j) y = z;
        }
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const T z = *reinterpret_cast<const T*>(vt + soff<U>(hr + r, (16 * ds + 4 * g + j) * ES / 2));
            if (y != 0.f) oacc[ds][qs][j] = fmaf(y, (float)z, oacc[ds][qs][j]);
          }
      }
    }
  };

  for (int t = t0; t < t1; ++t) {
    // tile t has arrived once only the NS - 2 younger ones are in flight
    if (t + NS - 2 < t1) dma_wait_but<(NS - 2) * OPS>();
    else dma_wait();
    __syncthreads();  // and every wave has left tile t - 1, whose stage is next
    if (t + NS - 1 < t1) issue(t + NS - 1);
    const int st = (t - t0) % NS, k0 = t * TR, h0 = kg * TK;
    const short* const kt = ring + st * 2 * TR * U;
    const short* const vt = kt + TR * U;
    const int* const pt = &spos[POS ? st : 0][w][0];
    if (k0 + TR <= c) {
      if constexpr (TK >= 32 && ES == 2) {
#pragma unroll
        for (int hr = 0; hr < TK; hr += 32) {
          f32x4 x[QT], y[QT];
          scores(std::false_type{}, k0, h0 + hr, kt, pt, x);
          scores(std::false_type{}, k0, h0 + hr + 16, kt, pt, y);
          product32(h0 + hr, x, y, vt);
        }
      } else {
#pragma unroll
        for (int hr = 0; hr < TK; hr += 16) {
          f32x4 x[QT];
          scores(std::false_type{}, k0, h0 + hr, kt, pt, x);
          product16(h0 + hr, x, vt);
        }
      }
    } else {
      for (int hr = h0; hr < h0 + TK; hr += 16) {
        f32x4 x[QT];
        scores(std::true_type{}, k0, hr, kt, pt, x);
        // values that some query must not see may be anything, and 0 x inf is
        // not 0: rows that hold a value that is not finite go one by one. (An
        // infinity in a row of the context, which every token sees, gives NaN.)
        bool odd = false;
#pragma unroll
        for (int u = 0; u < U / 32; ++u) {  // (the rows as they lie, 1 KB at a time: no bank conflicts)
          const VecT<T, 16 / ES> z = __builtin_bit_cast(VecT<T, 16 / ES>, lds16(vt + hr * U + 8 * (64 * u + lane)));
#pragma unroll
          for (int e = 0; e < 16 / ES; ++e) odd = odd || !(fabsf((float)z.v[e]) <= 3.4028234e38f);
        }
        if (__builtin_amdgcn_ballot_w64(odd) == 0ull) product16(hr, x, vt);
        else product_checked(hr, x, vt);
      }
    }
  }

  // L: over the lane groups; then, with the sums, over the row groups in order
  const bool whole = a.splits == 1;
  f32x4* const sx = reinterpret_cast<f32x4*>(ring);
#pragma unroll
  for (int qs = 0; qs < QT; ++qs) {
    lsum[qs] += __shfl_xor(lsum[qs], 16, 64);
    lsum[qs] += __shfl_xor(lsum[qs], 32, 64);
    if (KG > 1 && g == 0) sl[w][16 * qs + li] = lsum[qs];
  }
  if constexpr (KG > 1) {
    __syncthreads();  // the ring is idle
#pragma unroll
    for (int ds = 0; ds < DS; ++ds)
#pragma unroll
      for (int qs = 0; qs < QT; ++qs) sx[((w * DS + ds) * QT + qs) * 64 + lane] = oacc[ds][qs];
    __syncthreads();
  }
#pragma unroll
  for (int qs = 0; qs < QT; ++qs) {
    const int i = qi + 16 * qs;
    float l = lsum[qs];
    if constexpr (KG > 1) {
      l = 0.f;
#pragma unroll
      for (int r = 0; r < KG; ++r) l += sl[r * QG + qg][16 * qs + li];
    }
    const bool absent = anc[qs] == 0ull;
    if (absent) l = 0.f;
    const float inv = inv_sum(l + 16.f * a.eps);
    if (i >= N) continue;
    const int64_t prow = ((int64_t)bh * a.splits + split) * N + i;
    T* const op = (T*)a.o + b * a.so[0] + h * a.so[1] + i * a.so[2];
    if (kg == 0 && g == 0) {
      if (!whole) a.lpart[prow] = l;
      else if (a.L) a.L[(int64_t)bh * N + i] = l * 0.0625f;
    }
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) {
      if (KG > 1 && ds % KG != kg) continue;  // a row group writes every KG-th subtile
      f32x4 t = oacc[ds][qs];
      if constexpr (KG > 1) {
        t = sx[((qg * DS + ds) * QT + qs) * 64 + lane];
#pragma unroll
        for (int r = 1; r < KG; ++r) t += sx[(((r * QG + qg) * DS + ds) * QT + qs) * 64 + lane];
      }
      if (absent) t = f32x4{0.f, 0.f, 0.f, 0.f};  // (its products with rows it does not see may be NaN)
      const int d = 16 * ds + 4 * g;
      if (!whole) {
        *reinterpret_cast<f32x4*>(a.part + prow * W + d) = t;
      } else if (d < a.D) {
        const float y[4] = {t[0] * inv, t[1] * inv, t[2] * inv, t[3] * inv};
        store_acc<T, 4>(op + d, y);
      }
    }
  }
}

// o = sum over the splits / (L + eps): a thread per 4 columns of a query row,
// eight independent loads in flight, added in split order in eight running sums
// (deterministic). The last splits load as the others do, a missing one the last
// split again: with a branch around each they waited in turn, up to a microsecond
// a load (bf16, 12 heads, 57 tokens, T=2016: D=64 15.9 -> 14.0 us, D=128 20.6 -> 18.8)
constexpr int kTreeCombThreads = 256;
template <typename T, int W> __global__ __launch_bounds__(kTreeCombThreads) void attn_tree_combine_k(TreeArgs a) {
  constexpr int TPR = W / 4, RPB = kTreeCombThreads / TPR;  // threads per row, rows per block
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;  // (b * H + h) * N + i
  const int d = (threadIdx.x % TPR) * 4;
  if (row >= (int64_t)a.B * a.H * a.N) return;
  const int i = (int)(row % a.N);
  const int bh = (int)(row / a.N), b = bh / a.H, h = bh - b * a.H;
  const int64_t p0 = (int64_t)bh * a.splits * a.N + i;
  f32x4 t[8];
  float l[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    t[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    l[r] = 0.f;
  }
  for (int s = 0; s < a.splits; s += 8) {
    f32x4 x[8];
    float y[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int64_t p = p0 + (int64_t)std::min(s + r, a.splits - 1) * a.N;
      x[r] = *reinterpret_cast<const f32x4*>(a.part + p * W + d);
      y[r] = a.lpart[p];
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const bool in = s + r < a.splits;
#pragma unroll
      for (int j = 0; j < 4; ++j) t[r][j] += in ? x[r][j] : 0.f;
      l[r] += in ? y[r] : 0.f;
    }
  }
  const f32x4 x = ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
  const float y = ((l[0] + l[1]) + (l[2] + l[3])) + ((l[4] + l[5]) + (l[6] + l[7]));
  if (d == 0 && a.L) a.L[row] = y * 0.0625f;
  if (d < a.D) {
    const float inv = inv_sum(y + 16.f * a.eps);
    const float z[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
    store_acc<T, 4>((T*)a.o + b * a.so[0] + h * a.so[1] + i * a.so[2] + d, z);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// Blocks per (b, h): no more than the CUs hold at once (B=3, H=16, N=25, T=1999, D=96:
// 8 splits 16.8 us, 12, past what fits, 23.5; 4 splits 20.0), none without a tile; of
// those the number with the least time in tiles one after another and in the combine,
// whose rounds of eight splits take about three tiles' time each. Most that fit / this
// rule, bf16, 12 heads: N=64, D=64, T=1344 12.6 (21) / 10.9 us (8), T=4032 14.2 / 12.6
// (16); N=57, D=256, T=4000 30.5 (21) / 25.6 (16), T=16000 52 (21, as here) against 54.6
// (16); N=8, D=64, T=8192 13.7 (42) / 11.3 (16); one head, N=16, D=64, T=65536 47.5 (512) /
// 17.7; four heads, N=57, D=128, T=32768 28.7 (64) / 29.6 (40).
static int tree_splits(int64_t B, int64_t H, int64_t N, int64_t T, int W, int dtype) {
  const TreeShape s = tree_shape(W * dtype_size(dtype) / 2, tree_nq(N));
  const int64_t tiles = (T + s.rows - 1) / s.rows;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(s.blocks * (int64_t)num_cus() / (B * H), tiles));
  auto cost = [&](int64_t n) { return (tiles + n - 1) / n + 3 * ((n + 7) / 8); };
  int64_t best = most;
  for (int64_t n = (most - 1) / 8 * 8; n > 0; n -= 8)
    if (cost(n) < cost(best)) best = n;
  return (int)best;
}

template <typename T, int W, int NQ, bool POS> static int launch_tree(const TreeArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((attn_tree_k<T, W, NQ, POS>), dim3((unsigned)a.splits, (unsigned)(a.B * a.H)),
                     dim3(64 * tree_at<T, W, NQ>().waves), 0, st, a);
  if (int rc = check_launch("kat_attn_tree")) return rc;
  if (a.splits == 1) return KAT_OK;
  const int64_t rows = (int64_t)a.B * a.H * a.N, rpb = kTreeCombThreads / (W / 4);
  hipLaunchKernelGGL((attn_tree_combine_k<T, W>), dim3((unsigned)((rows + rpb - 1) / rpb)), dim3(kTreeCombThreads), 0,
                     st, a);
  return check_launch("kat_attn_tree (combine)");
}
template <typename T, int W> static int tree_n(const TreeArgs& a, hipStream_t st) {
  const bool pos = a.positions != nullptr;
  switch (tree_nq(a.N)) {
    case 1: return pos ? launch_tree<T, W, 1, true>(a, st) : launch_tree<T, W, 1, false>(a, st);
    case 2: return pos ? launch_tree<T, W, 2, true>(a, st) : launch_tree<T, W, 2, false>(a, st);
    default: return pos ? launch_tree<T, W, 4, true>(a, st) : launch_tree<T, W, 4, false>(a, st);
  }
}
template <typename T> static int tree_w(const TreeArgs& a, int W, hipStream_t st) {
  switch (W) {
    case 32: if constexpr (sizeof(T) == 4) return tree_n<T, 32>(a, st); break;
    case 64: return tree_n<T, 64>(a, st);
    case 128: return tree_n<T, 128>(a, st);
    case 256: if constexpr (sizeof(T) == 2) return tree_n<T, 256>(a, st); break;
  }
  return fail(KAT_EUNSUPPORTED, "kat_attn_tree: head dim %d", a.D);
}

}  // namespace kat

using namespace kat;

extern "C" size_t kat_attn_tree_workspace_size(int64_t B, int64_t H, int64_t N, int64_t T, int64_t D, int dtype) {
  const int W = cache_layout(D, dtype);
  if (B <= 0 || H <= 0 || T <= 0 || N <= 0 || N > kTreeMax || !W) return 0;
  const int splits = tree_splits(B, H, N, T, W, dtype);
  return splits == 1 ? 0 : (size_t)(B * H) * splits * N * (W + 1) * sizeof(float);
}

extern "C" int kat_attn_tree(const void* q, const void* k, const void* v, void* out, float* L, const float* slopes,
                             const int32_t* parents, int64_t parents_stride_b, const int32_t* lengths,
                             const int32_t* positions, const int64_t* pos_strides, void* workspace,
                             size_t workspace_bytes, int64_t B, int64_t H, int64_t N, int64_t T, int64_t D,
                             const int64_t* strides, float scale, float eps, int dtype, void* stream) {
  const char* nm = "kat_attn_tree";
  if (B < 0 || H < 0 || N < 0 || T < 0 || D < 0) return fail(KAT_EINVAL, "%s: negative size", nm);
  if (N > kTreeMax) return fail(KAT_EUNSUPPORTED, "%s: %lld tokens, at most %d are supported", nm, (long long)N, kTreeMax);
  if (B > 0xffff || H > 0xffff || B * H > 0xffff || T > 0x3fffffff)
    return fail(KAT_EUNSUPPORTED, "%s: B*H or T too large", nm);
  const int W = cache_layout(D, dtype);
  if (!W) return fail(KAT_EUNSUPPORTED, "%s: head dim %lld with dtype %d", nm, (long long)D, dtype);
  if (B * H * N == 0) return KAT_OK;
  if (!q || !out || !slopes || !parents || !strides || (positions && !pos_strides) || (T > 0 && (!k || !v)))
    return fail(KAT_EINVAL, "%s: null pointer", nm);
  const int esz = dtype_size(dtype);
  int64_t st12[12];
  for (int t = 0; t < 12; ++t) {
    const int64_t size[3] = {B, H, t < 3 || t >= 9 ? N : T};
    st12[t] = dim_stride(strides[t], size[t % 3]);
    if ((st12[t] * esz) % 16 != 0) return fail(KAT_EUNSUPPORTED, "%s: strides must keep rows 16-byte aligned", nm);
  }
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(KAT_EUNSUPPORTED, "%s: tensors must be 16-byte aligned", nm);
  if (T > 1 && (st12[5] < D || st12[8] < D)) return fail(KAT_EINVAL, "%s: cache row stride < D", nm);
  // a tile's rows are addressed by 31-bit byte offsets
  if (T > 1 && std::max(st12[5], st12[8]) > 0x7fffffff / (64 * esz))
    return fail(KAT_EUNSUPPORTED, "%s: cache row stride too large", nm);
  TreeArgs a = {};
  a.q = q;
  a.k = k;
  a.v = v;
  a.o = out;
  a.L = L;
  a.slopes = slopes;
  a.parents = parents;
  a.lengths = lengths;
  a.positions = positions;
  a.B = (int)B;
  a.H = (int)H;
  a.N = (int)N;
  a.T = (int)T;
  a.D = (int)D;
  for (int i = 0; i < 3; ++i) {
    a.sq[i] = st12[i];
    a.sk[i] = st12[3 + i];
    a.sv[i] = st12[6 + i];
    a.so[i] = st12[9 + i];
  }
  if (T <= 1) a.sk[2] = a.sv[2] = D;
  a.spar = parents_stride_b;
  if (positions) {
    a.spos[0] = pos_strides[0];
    a.spos[1] = pos_strides[1];
  }
  a.scale = scale;
  a.eps = eps;
  a.splits = tree_splits(B, H, N, std::max<int64_t>(T, 1), W, dtype);
  const size_t need = kat_attn_tree_workspace_size(B, H, N, T, D, dtype);
  if (need && (!workspace || workspace_bytes < need))
    return fail(KAT_EINVAL, "%s: workspace %zu bytes < required %zu", nm, workspace_bytes, need);
  a.part = (float*)workspace;
  a.lpart = a.part + (size_t)(B * H) * a.splits * N * W;
  const hipStream_t st = as_stream(stream);
  switch (dtype) {
    case KAT_F32: return tree_w<float>(a, W, st);
    case KAT_BF16: return tree_w<bf16>(a, W, st);
    case KAT_F16: return tree_w<f16>(a, W, st);
  }
  return fail(KAT_EUNSUPPORTED, "%s: unsupported dtype %d", nm, dtype);
}
