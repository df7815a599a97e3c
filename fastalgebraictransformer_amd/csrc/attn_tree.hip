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
// write plain sums and a second kernel adds them in a fixed order. Inside a block
// every wave takes row groups of its own (32 rows; 16 in fp32) for all queries,
// so K and V pass through no shared tile and the loop has no barrier:
//   S^T[row][q] = K Q^T    A = K straight from memory to registers (lane (g,
//                          li) loads 16 bytes of row li), B = Q^T (registers)
//   f of S^T               lane (g, li) holds rows 4 g + j, query li
//   O^T[d][q] += V^T f^T   A = V^T: the wave's rows go through an LDS tile of
//                          its own and come back transposed; B = f packed to
//                          the dtype (as the forward does), or fp32
// The next group's rows are loaded before the current group is worked on.
// Only groups that reach the tokens' rows (at most three) look at the ancestor
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
constexpr int kTreeWaves = 4;

// rows of one wave's group
template <typename T> constexpr int tree_group() { return sizeof(T) == 2 ? 32 : 16; }

template <typename T, int W, int QT, bool POS>
__global__ __launch_bounds__(64 * kTreeWaves, QT == 4 || W == 256 ? 1 : 2) void attn_tree_k(TreeArgs a) {
  constexpr int ES = (int)sizeof(T);
  constexpr int RB = W * ES;             // bytes of a row
  constexpr int KK = RB / 64;            // 64-byte column blocks
  constexpr int G = tree_group<T>();     // rows of a group
  constexpr int HH = G / 16;             // 16-row halves
  constexpr int CPR = RB / 16;           // 16-byte pieces of a row
  constexpr int NV = G * CPR / 64;       // V pieces per lane
  constexpr int RPL = 64 / CPR;          // V rows per load instruction
  constexpr int DS = W / 16;             // 16-wide d subtiles
  constexpr int U = RB / 2;              // a row in 16-bit units, the unit of the tile helpers
  static_assert(CPR <= 64 && NV >= 1, "row layout");
  __shared__ short sv[kTreeWaves][G * U];
  __shared__ f32x4 sx[kTreeWaves * DS * 64];  // the waves' sums of one query subtile
  __shared__ float sl[kTreeWaves][16 * QT];
  __shared__ uint64_t sanc[kTreeMax];  // ancestors of token i, itself included; 0 if absent
  __shared__ int sdep[kTreeMax];       // depth of token i below the context

  const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
  const int split = blockIdx.x;
  const int lane = threadIdx.x & 63, w = wave_id();
  const int g = lane >> 4, li = lane & 15;
  const int N = a.N;
  int n = a.lengths ? a.lengths[b] : a.T;
  n = min(n, a.T);
  const int c = n - N;       // rows of the context
  if (c < 0) n = 0;          // no room for the tokens: the row holds no draft

  if (w == 0) {
    // pointer doubling: after step i, anc holds the 2^i nearest ancestors and
    // up the one above them (-1: the context is reached)
    int up = lane < N ? a.parents[b * a.spar + lane] : -2;
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

  const float slope = a.slopes[h], scale = a.scale;
  const char* kp = (const char*)((const T*)a.k + b * a.sk[0] + h * a.sk[1]);
  const char* vp = (const char*)((const T*)a.v + b * a.sv[0] + h * a.sv[1]);
  const int64_t skb = a.sk[2] * ES, svb = a.sv[2] * ES;
  const int32_t* pp = POS ? a.positions + b * a.spos[0] + h * a.spos[1] : nullptr;
  const int cols = a.D * ES / 16;  // pieces of a row that hold columns

  // this split's groups, dealt to the waves in turn
  const int ng = (n + G - 1) / G;
  const int per = (ng + a.splits - 1) / a.splits;
  const int g0 = split * per, g1 = min(g0 + per, ng);

  // pieces at or past the head dim re-read the row's first one (the query is
  // zero there, and their output columns are not stored); rows past the last
  // filled one re-read it
  i16x8 kr[HH][KK], vr[NV];
  auto load = [&](int gi) __attribute__((always_inline)) {
#pragma unroll
    for (int hh = 0; hh < HH; ++hh) {
      const char* row = kp + (int64_t)min(gi * G + 16 * hh + li, n - 1) * skb;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) kr[hh][kk] = ld_piece_nt(row + 16 * (4 * kk + g < cols ? 4 * kk + g : 0));
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int r = u * RPL + lane / CPR, p = lane % CPR;
      vr[u] = ld_piece_nt(vp + (int64_t)min(gi * G + r, n - 1) * svb + 16 * (p < cols ? p : 0));
    }
  };
  int gi = g0 + w;
  if (gi < g1) load(gi);

  i16x8 qf[QT][KK];
#pragma unroll
  for (int qs = 0; qs < QT; ++qs)
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int i = 16 * qs + li, p = 4 * kk + g;
      qf[qs][kk] = i16x8{0, 0, 0, 0, 0, 0, 0, 0};
      if (i < N && p < cols)
        qf[qs][kk] = *reinterpret_cast<const i16x8*>((const char*)((const T*)a.q + b * a.sq[0] + h * a.sq[1] + i * a.sq[2]) +
                                                     16 * p);
    }
  __syncthreads();  // masks and depths
  uint64_t anc[QT];
  int qpos[QT];
#pragma unroll
  for (int qs = 0; qs < QT; ++qs) {
    const int i = 16 * qs + li;
    anc[qs] = i < N ? sanc[i] : 0ull;
    qpos[qs] = 0;
    if (i < N && n > 0) qpos[qs] = POS ? pp[c + i] : c + sdep[i];
  }

  f32x4 oacc[DS][QT];
  float lsum[QT];
#pragma unroll
  for (int qs = 0; qs < QT; ++qs) {
    lsum[qs] = 0.f;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) oacc[ds][qs] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  short* const vt = sv[w];

  // one group from the loaded rows; TAIL: it reaches the tokens' rows or ends
  // past the last filled row
  auto work = [&](auto tail_tag, int k0, const i16x8 (&kc)[HH][KK]) __attribute__((always_inline)) {
    constexpr bool TAIL = decltype(tail_tag)::value;
    f32x4 f[HH][QT];
#pragma unroll
    for (int hh = 0; hh < HH; ++hh)
#pragma unroll
      for (int qs = 0; qs < QT; ++qs) {
        f[hh][qs] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) f[hh][qs] = dot64<T>(kc[hh][kk], qf[qs][kk], f[hh][qs]);
      }
#pragma unroll
    for (int hh = 0; hh < HH; ++hh)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = k0 + 16 * hh + 4 * g + j;
        const int tok = row - c;  // the drafted token in this row, if >= 0
        int kpos = row;
        if constexpr (POS) kpos = pp[TAIL ? min(row, n - 1) : row];
        else if constexpr (TAIL) kpos = tok < 0 ? row : c + sdep[min(tok, kTreeMax - 1)];
#pragma unroll
        for (int qs = 0; qs < QT; ++qs) {
          const float s = fmaf(f[hh][qs][j], scale, -slope * (float)(qpos[qs] - kpos));
          float x = sig2_pow4(s);
          if constexpr (TAIL) {
            const bool seen = tok < 0 ? anc[qs] != 0ull : tok < N && ((anc[qs] >> (tok & 63)) & 1ull);
            x = seen ? x : 0.f;
          }
          f[hh][qs][j] = x;
          lsum[qs] += x;
        }
      }
    bool plain = true;
    if constexpr (TAIL) {
      // values that some query must not see may be anything, and 0 x inf is not
      // 0: a group holding a value that is not finite takes the products one by one
      bool odd = false;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const VecT<T, 16 / ES> x = __builtin_bit_cast(VecT<T, 16 / ES>, vr[u]);
#pragma unroll
        for (int e = 0; e < 16 / ES; ++e) odd = odd || !(fabsf((float)x.v[e]) <= 3.4028234e38f);
      }
      plain = __builtin_amdgcn_ballot_w64(odd) == 0ull;
    }
    if (plain) {
      if constexpr (ES == 2) {
        i16x8 pf[QT];
#pragma unroll
        for (int qs = 0; qs < QT; ++qs) {
          const f32x4 x = f[0][qs], y = f[1][qs];
          pf[qs] = pack_frag(Mfma<T>::pack2(x[0], x[1]), Mfma<T>::pack2(x[2], x[3]), Mfma<T>::pack2(y[0], y[1]),
                             Mfma<T>::pack2(y[2], y[3]));
        }
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) {
          const i16x8 vf = frag_tr<U>(vt, 0, 16 * ds, g, li);
#pragma unroll
          for (int qs = 0; qs < QT; ++qs) oacc[ds][qs] = Mfma<T>::mma(vf, pf[qs], oacc[ds][qs]);
        }
      } else {
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = *reinterpret_cast<const float*>(vt + soff<U>(4 * g + j, 32 * ds + 2 * li));
#pragma unroll
            for (int qs = 0; qs < QT; ++qs)
              oacc[ds][qs] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, f[0][qs][j], oacc[ds][qs], 0, 0, 0);
          }
      }
    } else {
      for (int r = 0; r < G; ++r) {
        const int src = ((r & 15) >> 2) * 16 + li;  // the lane that holds this row's f of query li
#pragma unroll
        for (int qs = 0; qs < QT; ++qs) {
          float x = 0.f;
#pragma unroll
          for (int hh = 0; hh < HH; ++hh)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float y = __shfl(f[hh][qs][j], src, 64);
              if (r == 16 * hh + (r & 12) + j) x = y;
            }
#pragma unroll
          for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int d = 16 * ds + 4 * g + j;
              const T y = *reinterpret_cast<const T*>(reinterpret_cast<const char*>(vt + soff<U>(r, d * ES / 2)));
              if (x != 0.f) oacc[ds][qs][j] = fmaf(x, (float)y, oacc[ds][qs][j]);
            }
        }
      }
    }
  };

  for (; gi < g1; gi += kTreeWaves) {
    const int k0 = gi * G;
    i16x8 kc[HH][KK];
#pragma unroll
    for (int hh = 0; hh < HH; ++hh)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) kc[hh][kk] = kr[hh][kk];
#pragma unroll
    for (int u = 0; u < NV; ++u)
      *reinterpret_cast<i16x8*>(vt + soff<U>(u * RPL + lane / CPR, 8 * (lane % CPR))) = vr[u];
    if (k0 + G > c) {
      work(std::true_type{}, k0, kc);
      if (gi + kTreeWaves < g1) load(gi + kTreeWaves);
    } else {
      if (gi + kTreeWaves < g1) load(gi + kTreeWaves);
      work(std::false_type{}, k0, kc);
    }
  }

  // sums over the lane groups (l), then over the waves, in wave order
#pragma unroll
  for (int qs = 0; qs < QT; ++qs) {
    lsum[qs] += __shfl_xor(lsum[qs], 16, 64);
    lsum[qs] += __shfl_xor(lsum[qs], 32, 64);
    if (g == 0) sl[w][16 * qs + li] = lsum[qs];
  }
  const bool whole = a.splits == 1;
  const int64_t prow = ((int64_t)bh * a.splits + split) * N;
#pragma unroll
  for (int qs = 0; qs < QT; ++qs) {
    __syncthreads();
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) sx[(w * DS + ds) * 64 + lane] = oacc[ds][qs];
    __syncthreads();
    const int i = 16 * qs + li;
    float l = 0.f;
#pragma unroll
    for (int ww = 0; ww < kTreeWaves; ++ww) l += sl[ww][i];
    const bool absent = anc[qs] == 0ull;
    if (absent) l = 0.f;
    const float inv = 1.f / (l + 16.f * a.eps);
    if (i < N && w == 0 && g == 0) {
      if (!whole) a.lpart[prow + i] = l;
      else if (a.L) a.L[(int64_t)bh * N + i] = l * 0.0625f;
    }
    for (int ds = w; ds < DS; ds += kTreeWaves) {
      f32x4 t = sx[ds * 64 + lane];
#pragma unroll
      for (int ww = 1; ww < kTreeWaves; ++ww) t += sx[(ww * DS + ds) * 64 + lane];
      if (absent) t = f32x4{0.f, 0.f, 0.f, 0.f};  // (their products with rows they do not see may be NaN)
      const int d = 16 * ds + 4 * g;
      if (i >= N) continue;
      if (!whole) {
        *reinterpret_cast<f32x4*>(a.part + (prow + i) * W + d) = t;
      } else if (d < a.D) {
        T* o = (T*)a.o + b * a.so[0] + h * a.so[1] + i * a.so[2] + d;
        const float y[4] = {t[0] * inv, t[1] * inv, t[2] * inv, t[3] * inv};
        store_acc<T, 4>(o, y);
      }
    }
  }
}

// o = sum over the splits / (L + eps): a thread per 4 columns of a query row,
// eight independent loads in flight, added in split order in eight running sums
// (deterministic)
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
  int s = 0;
  for (; s + 8 <= a.splits; s += 8) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int64_t p = p0 + (int64_t)(s + r) * a.N;
      t[r] += *reinterpret_cast<const f32x4*>(a.part + p * W + d);
      l[r] += a.lpart[p];
    }
  }
#pragma unroll
  for (int r = 0; r < 7; ++r)
    if (s + r < a.splits) {
      const int64_t p = p0 + (int64_t)(s + r) * a.N;
      t[r] += *reinterpret_cast<const f32x4*>(a.part + p * W + d);
      l[r] += a.lpart[p];
    }
  const f32x4 x = ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
  const float y = ((l[0] + l[1]) + (l[2] + l[3])) + ((l[4] + l[5]) + (l[6] + l[7]));
  if (d == 0 && a.L) a.L[row] = y * 0.0625f;
  if (d < a.D) {
    const float inv = 1.f / (y + 16.f * a.eps);
    const float z[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
    store_acc<T, 4>((T*)a.o + b * a.so[0] + h * a.so[1] + i * a.so[2] + d, z);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// blocks per (b, h): enough to fill the CUs twice, none without a row group
// per wave
static int tree_splits(int64_t B, int64_t H, int64_t T, int dtype) {
  const int per_block = kTreeWaves * (dtype == KAT_F32 ? 16 : 32);
  const int64_t want = (2 * (int64_t)num_cus() + B * H - 1) / (B * H);
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, (T + per_block - 1) / per_block));
}

template <typename T, int W, int QT, bool POS> static int launch_tree(const TreeArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((attn_tree_k<T, W, QT, POS>), dim3((unsigned)a.splits, (unsigned)(a.B * a.H)),
                     dim3(64 * kTreeWaves), 0, st, a);
  if (int rc = check_launch("kat_attn_tree")) return rc;
  if (a.splits == 1) return KAT_OK;
  const int64_t rows = (int64_t)a.B * a.H * a.N, rpb = kTreeCombThreads / (W / 4);
  hipLaunchKernelGGL((attn_tree_combine_k<T, W>), dim3((unsigned)((rows + rpb - 1) / rpb)), dim3(kTreeCombThreads), 0,
                     st, a);
  return check_launch("kat_attn_tree (combine)");
}
template <typename T, int W> static int tree_qt(const TreeArgs& a, hipStream_t st) {
  const bool pos = a.positions != nullptr;
  if (a.N <= 16) return pos ? launch_tree<T, W, 1, true>(a, st) : launch_tree<T, W, 1, false>(a, st);
  if (a.N <= 32) return pos ? launch_tree<T, W, 2, true>(a, st) : launch_tree<T, W, 2, false>(a, st);
  return pos ? launch_tree<T, W, 4, true>(a, st) : launch_tree<T, W, 4, false>(a, st);
}
template <typename T> static int tree_w(const TreeArgs& a, int W, hipStream_t st) {
  switch (W) {
    case 32: if constexpr (sizeof(T) == 4) return tree_qt<T, 32>(a, st); break;
    case 64: return tree_qt<T, 64>(a, st);
    case 128: return tree_qt<T, 128>(a, st);
    case 256: if constexpr (sizeof(T) == 2) return tree_qt<T, 256>(a, st); break;
  }
  return fail(KAT_EUNSUPPORTED, "kat_attn_tree: head dim %d", a.D);
}

}  // namespace kat

using namespace kat;

extern "C" size_t kat_attn_tree_workspace_size(int64_t B, int64_t H, int64_t N, int64_t T, int64_t D, int dtype) {
  const int W = cache_layout(D, dtype);
  if (B <= 0 || H <= 0 || T <= 0 || N <= 0 || N > kTreeMax || !W) return 0;
  const int splits = tree_splits(B, H, T, dtype);
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
  for (int t = 0; t < 12; ++t)
    if ((strides[t] * esz) % 16 != 0) return fail(KAT_EUNSUPPORTED, "%s: strides must keep rows 16-byte aligned", nm);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(KAT_EUNSUPPORTED, "%s: tensors must be 16-byte aligned", nm);
  if (T > 1 && (strides[5] < D || strides[8] < D)) return fail(KAT_EINVAL, "%s: cache row stride < D", nm);
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
    a.sq[i] = strides[i];
    a.sk[i] = strides[3 + i];
    a.sv[i] = strides[6 + i];
    a.so[i] = strides[9 + i];
  }
  a.spar = parents_stride_b;
  if (positions) {
    a.spos[0] = pos_strides[0];
    a.spos[1] = pos_strides[1];
  }
  a.scale = scale;
  a.eps = eps;
  a.splits = tree_splits(B, H, std::max<int64_t>(T, 1), dtype);
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
