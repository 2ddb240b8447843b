// RMS norm of every query / key head and the rotary position embedding in one pass (gfx950).
//
//   n = x * rsqrt(mean(x^2) + eps) * w,   y = R(pos) n   (rotates pairs of n's first `rot` values)
//   dn = R(pos)^T dy,  xh = x * rsqrt(...),  g = dn * w,  dw = sum dn * xh,  dx = rsqrt(...) (g - xh mean(g xh))
//
// Memory bound: each value is read and written once (backward: x and dy read, dx written), everything in
// between is fp32 in registers.
//  * A lane holds 4 rotation pairs (8 values) of one head, so no value changes lanes for the rotation: with
//    split halves it loads 4 values of the first and the 4 partners of the second half, interleaved pairs are
//    8 neighbours, values past `rot` travel as pairs that are not turned.
//  * A wave owns a token and walks its heads, 64 / (lanes of a head) at a time: the angles and the norm weights
//    stay in registers for all of them, and the only reductions are over the lanes of a head.
//  * Weight gradients: every lane sums its own columns over all its rows, the workgroup joins them in LDS and
//    writes one partial row, a second small kernel adds the rows in order (no atomics, same bits every run).
#include "bh/api.h"
#include "bh/device.h"
#include "bh/qk_rope_api.h"

#include <algorithm>
#include <stdexcept>
#include <string>
#include <type_traits>

namespace bh {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;

template <typename T> BH_DEVICE void load4(const T* p, float (&r)[8], int at) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  const t4 v = *reinterpret_cast<const t4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[at + i] = to_f<T>(v[i]);
}
template <typename T> BH_DEVICE void store4(T* p, const float (&r)[8], int at) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<t4*>(p) = t4{from_f<T>(r[at]), from_f<T>(r[at + 1]), from_f<T>(r[at + 2]), from_f<T>(r[at + 3])};
}

// The 4 pairs of a lane. VEC: two runs of 4 values from e0 and e1; with split halves (and in the part that is not
// rotated) registers i and 4 + i are a pair, interleaved registers 2 i and 2 i + 1 (the runs are neighbours).
template <bool VEC> struct Slots {
  int e0, e1;        // VEC: start of the two runs
  int first, half;   // first pair, rot / 2
  int hn;
  bool inter, live;  // live: the lane has a pair below hn / 2
  BH_DEVICE Slots(int c, int hn_, int rot, bool il) : first(4 * c), half(rot >> 1), hn(hn_), inter(il) {
    live = 8 * c < hn;
    const bool halves = !il && 8 * c < rot;
    e0 = halves ? 4 * c : 8 * c;
    e1 = halves ? half + 4 * c : 8 * c + 4;
  }
  // element of register k (0..7) on the scalar path; -1: none
  BH_DEVICE int elem(int k) const {
    const int pair = first + (inter ? k >> 1 : k & 3), second = inter ? k & 1 : k >> 2;
    if (2 * pair >= hn) return -1;
    return !inter && pair < half ? pair + (second ? half : 0) : 2 * pair + second;
  }
  template <typename T> BH_DEVICE void load(const T* p, float (&r)[8]) const {
    if (!live) {
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = 0.f;
      return;
    }
    if (VEC) {
      load4<T>(p + e0, r, 0);
      load4<T>(p + e1, r, 4);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = elem(k);
        r[k] = e >= 0 ? to_f<T>(p[e]) : 0.f;
      }
    }
  }
  template <typename T> BH_DEVICE void store(T* p, const float (&r)[8]) const {
    if (!live) return;
    if (VEC) {
      store4<T>(p + e0, r, 0);
      store4<T>(p + e1, r, 4);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = elem(k);
        if (e >= 0) p[e] = from_f<T>(r[k]);
      }
    }
  }
};

// sum over the LPR lanes of a head (8 lanes and more): moves inside 16 lanes are DPP operands of the adds
template <int CTRL> BH_DEVICE float add_dpp(float v) {
  const int x = __builtin_bit_cast(int, v);
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, true));
}
template <int LPR> BH_DEVICE float row_sum(float v) {
  v = add_dpp<0xB1>(v);                  // quad_perm 1 0 3 2
  v = add_dpp<0x4E>(v);                  // quad_perm 2 3 0 1
  v = add_dpp<0x141>(v);                 // row_half_mirror
  if (LPR >= 16) v = add_dpp<0x140>(v);  // row_mirror
  if (LPR >= 32) v += __shfl_xor(v, 16, kWave);
  if (LPR >= 64) v += __shfl_xor(v, 32, kWave);
  return v;
}

// the lane's 4 angles at the token's position; a position outside the tables gives NaN, never a read there
BH_DEVICE void angles(const QkRopeArgs& a, int t, int b, int first, float (&c)[4], float (&s)[4]) {
  int64_t pos = a.offset + t;
  if (a.pos) {
    const int64_t i = (int64_t)t * a.pos_st + (int64_t)b * a.pos_sb;
    pos = a.pos_i64 ? reinterpret_cast<const int64_t*>(a.pos)[i] : (int64_t)reinterpret_cast<const int*>(a.pos)[i];
  }
  const bool ok = pos >= 0 && pos < a.n_pos;
  const int half = a.rot >> 1;
  const int64_t row = ok ? pos * half : 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool turned = first + i < half;
    c[i] = !turned ? 1.f : ok ? a.cos[row + first + i] : __builtin_nanf("");
    s[i] = !turned ? 0.f : ok ? a.sin[row + first + i] : __builtin_nanf("");
  }
}
// pairs turned by +angle (SIGN 1) or -angle (SIGN -1)
template <int SIGN> BH_DEVICE void turn(float (&r)[8], const float (&c)[4], const float (&s)[4], bool inter) {
  auto pair = [&](int i, float& x, float& y) {
    const float q = SIGN > 0 ? s[i] : -s[i], u = x, v = y;
    x = u * c[i] - v * q;
    y = v * c[i] + u * q;
  };
  if (inter) {
#pragma unroll
    for (int i = 0; i < 4; ++i) pair(i, r[2 * i], r[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) pair(i, r[i], r[4 + i]);
  }
}
template <bool VEC> BH_DEVICE void load_weights(const QkRopeArgs& a, const Slots<VEC>& sl, int k, float (&w)[8]) {
  switch (a.w_dt) {
    case kF16: sl.load(reinterpret_cast<const f16*>(a.w[k]), w); break;
    case kBF16: sl.load(reinterpret_cast<const bf16*>(a.w[k]), w); break;
    default: sl.load(reinterpret_cast<const float*>(a.w[k]), w);
  }
}

template <typename T> BH_DEVICE T* row_ptr(const HeadView& v, int t, int b, int h) {
  return reinterpret_cast<T*>(v.p) + (int64_t)t * v.st + (int64_t)b * v.sb + (int64_t)h * v.sh;
}

// A token's passes: query heads in groups of HPW (the first nq), then key heads. f gets the operand as a constant,
// so its weights and sums are registers that are never selected.
template <typename F> BH_DEVICE void passes(int nq, int p0, int p1, F&& f) {
  f(std::integral_constant<int, 0>{}, p0, min(p1, nq));
  f(std::integral_constant<int, 1>{}, max(p0, nq) - nq, p1 - nq);
}

template <typename T, int LPR, bool VEC, bool NORM>
__global__ __launch_bounds__(kThreads) void k_qk_rope_fwd(QkRopeArgs a, int ppw) {
  constexpr int HPW = kWave / LPR;
  const int lane = threadIdx.x & (kWave - 1), c = lane % LPR, sub = lane / LPR;
  const int64_t tok = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (tok >= (int64_t)a.s * a.b) return;
  const int t = (int)(tok / a.b), b = (int)(tok - (int64_t)t * a.b);
  const Slots<VEC> sl(c, a.hn, a.rot, a.interleaved);
  const int nq = (a.heads[0] + HPW - 1) / HPW, np = nq + (a.heads[1] + HPW - 1) / HPW;
  const int p0 = blockIdx.y * ppw, p1 = min(p0 + ppw, np);
  const float inv_n = 1.f / (float)a.hn;
  float co[4], si[4];
  if (a.rot) angles(a, t, b, sl.first, co, si);
  auto run = [&](auto kk, int q0, int q1) {
    constexpr int k = decltype(kk)::value;
    if (q0 >= q1) return;
    float w[8];
    if (NORM) load_weights(a, sl, k, w);
    int h = q0 * HPW + sub;
    const T* x = row_ptr<const T>(a.x[k], t, b, 0) + (int64_t)h * a.x[k].sh;
    T* y = row_ptr<T>(a.y[k], t, b, 0) + (int64_t)h * a.y[k].sh;
    const int64_t sx = HPW * a.x[k].sh, sy = HPW * a.y[k].sh;
    auto head = [&](const T* xp, T* yp, bool on) {
      float v[8];
      sl.load(xp, v);
      if (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
        const float r = rsqrtf(row_sum<LPR>(ss) * inv_n + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * r * w[i];
      }
      if (a.rot) turn<1>(v, co, si, sl.inter);
      if (on) sl.store(yp, v);
    };
    int q = q0;
    const int full = a.heads[k] / HPW;  // passes whose every lane has a head
#pragma unroll 4
    for (; q < min(q1, full); ++q, x += sx, y += sy) head(x, y, true);
    if (q < q1) {
      const bool on = q * HPW + sub < a.heads[k];
      head(on ? x : row_ptr<const T>(a.x[k], t, b, 0), y, on);
    }
  };
  passes(nq, p0, p1, run);
}

template <typename T, int LPR, bool VEC, bool NORM>
__global__ __launch_bounds__(kThreads) void k_qk_rope_bwd(QkRopeArgs a, int ppw, float* __restrict__ part) {
  constexpr int HPW = kWave / LPR;
  __shared__ float sh[NORM ? kWaves : 1][NORM ? 2 * 8 * LPR : 1];
  const int lane = threadIdx.x & (kWave - 1), c = lane % LPR, sub = lane / LPR;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t toks = (int64_t)a.s * a.b;
  const Slots<VEC> sl(c, a.hn, a.rot, a.interleaved);
  const int nq = (a.heads[0] + HPW - 1) / HPW, np = nq + (a.heads[1] + HPW - 1) / HPW;
  const int p0 = blockIdx.y * ppw, p1 = min(p0 + ppw, np);
  const float inv_n = 1.f / (float)a.hn;
  float w[2][8], dw[2][8];
  if (NORM) {
    load_weights(a, sl, 0, w[0]);
    load_weights(a, sl, 1, w[1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[0][i] = dw[1][i] = 0.f;
  }
  for (int64_t tok = (int64_t)blockIdx.x * kWaves + wave; tok < toks; tok += (int64_t)gridDim.x * kWaves) {
    const int t = (int)(tok / a.b), b = (int)(tok - (int64_t)t * a.b);
    float co[4], si[4];
    if (a.rot) angles(a, t, b, sl.first, co, si);
    auto run = [&](auto kk, int q0, int q1) {
      constexpr int k = decltype(kk)::value;
      if (q0 >= q1) return;
      const int h = q0 * HPW + sub;
      const T* x = row_ptr<const T>(a.x[k], t, b, 0) + (int64_t)h * a.x[k].sh;
      const T* dy = row_ptr<const T>(a.dy[k], t, b, 0) + (int64_t)h * a.dy[k].sh;
      T* y = row_ptr<T>(a.y[k], t, b, 0) + (int64_t)h * a.y[k].sh;
      const int64_t sx = HPW * a.x[k].sh, sd = HPW * a.dy[k].sh, sy = HPW * a.y[k].sh;
      auto head = [&](const T* xp, const T* dp, T* yp, bool on) {
        float v[8], g[8];
        sl.load(dp, g);
        if (NORM) sl.load(xp, v);
        if (a.rot) turn<-1>(g, co, si, sl.inter);
        if (NORM) {
          float ss = 0.f, gx = 0.f, gw[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            gw[i] = g[i] * w[k][i];
            ss = fmaf(v[i], v[i], ss);
            gx = fmaf(gw[i], v[i], gx);
          }
          ss = row_sum<LPR>(ss);
          gx = row_sum<LPR>(gx);
          const float r = rsqrtf(ss * inv_n + a.eps), m = gx * r * r * inv_n, keep = on ? r : 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dw[k][i] = fmaf(g[i], v[i] * keep, dw[k][i]);
            g[i] = r * (gw[i] - v[i] * m);
          }
        }
        if (on) sl.store(yp, g);
      };
      int q = q0;
      const int full = a.heads[k] / HPW;
#pragma unroll 4
      for (; q < min(q1, full); ++q, x += sx, dy += sd, y += sy) head(x, dy, y, true);
      if (q < q1) {
        const bool on = q * HPW + sub < a.heads[k];
        head(on ? x : row_ptr<const T>(a.x[k], t, b, 0), on ? dy : row_ptr<const T>(a.dy[k], t, b, 0), y, on);
      }
    };
    passes(nq, p0, p1, run);
  }
  if (NORM) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = dw[k][i];
#pragma unroll
        for (int o = LPR; o < kWave; o <<= 1) v += __shfl_xor(v, o, kWave);
        if (sub == 0) sh[wave][(k * LPR + c) * 8 + i] = v;
      }
    __syncthreads();
    float* row = part + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * a.hn;
    if (wave < 2 && sub == 0 && sl.live) {  // wave k writes the sums of operand k to their columns
      const int k = wave;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = 0.f;
#pragma unroll
        for (int q = 0; q < kWaves; ++q) v[i] += sh[q][(k * LPR + c) * 8 + i];
      }
      sl.template store<float>(row + k * a.hn, v);
    }
  }
}

// Weight gradients of the query (blockIdx.y 0) and the key (1): sums over the partial rows, each column by 16 lanes
// that take every 16th row, joined in order through LDS. A block has 64 columns.
template <typename W>
__global__ __launch_bounds__(1024) void k_qk_rope_dw(const float* __restrict__ part, int rows, int hn, W* __restrict__ dwq,
                                                     W* __restrict__ dwk) {
  __shared__ float sh[16][64];
  const int col = threadIdx.x & 63, lane = threadIdx.x >> 6, c = blockIdx.x * 64 + col;
  const float* p = part + (int64_t)blockIdx.y * hn + c;
  float acc = 0.f;
  if (c < hn) {
#pragma unroll 8
    for (int r = lane; r < rows; r += 16) acc += p[(int64_t)r * 2 * hn];
  }
  sh[lane][col] = acc;
  __syncthreads();
  if (lane == 0 && c < hn) {
    float t = 0.f;
#pragma unroll
    for (int l = 0; l < 16; ++l) t += sh[l][col];
    (blockIdx.y ? dwk : dwq)[c] = from_f<W>(t);
  }
}

inline void check_launch(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw std::runtime_error(std::string(what) + ": " + hipGetErrorString(e));
}
template <typename T> struct TypeTag { using type = T; };
template <typename F> void dispatch(int dt, const QkRopeArgs& a, F&& f) {
  auto by_norm = [&](auto t, auto lpr, auto vec) {
    if (a.w[0]) f(t, lpr, vec, std::true_type{});
    else f(t, lpr, vec, std::false_type{});
  };
  auto by_vec = [&](auto t, auto lpr) {
    if (a.vec) by_norm(t, lpr, std::true_type{});
    else by_norm(t, lpr, std::false_type{});
  };
  auto by_lanes = [&](auto t) {
    const int lanes = (a.hn + 7) / 8;
    if (lanes <= 8) by_vec(t, std::integral_constant<int, 8>{});
    else if (lanes <= 16) by_vec(t, std::integral_constant<int, 16>{});
    else if (lanes <= 32) by_vec(t, std::integral_constant<int, 32>{});
    else if (lanes <= 64) by_vec(t, std::integral_constant<int, 64>{});
    else throw std::runtime_error("qk_norm_rope: head size above 512");
  };
  switch (dt) {
    case kF32: by_lanes(TypeTag<float>{}); break;
    case kF16: by_lanes(TypeTag<f16>{}); break;
    case kBF16: by_lanes(TypeTag<bf16>{}); break;
    default: throw std::runtime_error("qk_norm_rope: fp32 / fp16 / bf16 only");
  }
}
struct Plan {
  int ppw, chunks;  // passes of a wave, wave rows per token
  int64_t gx;
};
// A wave takes all passes of a token when there are tokens enough to fill the card (2048 waves), else the
// token's passes are spread over more waves. persistent (weight gradients: a workgroup has one partial row): the 1024
// workgroups that are resident at once; 16384 tokens, 32 + 8 heads of 128 in bf16: backward 115 + 6 us, with 512 164 + 4,
// with 2048 115 + 11 (the second figure adds the partial rows).
Plan plan(const QkRopeArgs& a, bool persistent) {
  int lpr = 8;
  while (lpr * 8 < a.hn) lpr *= 2;
  const int hpw = kWave / lpr, np = (a.heads[0] + hpw - 1) / hpw + (a.heads[1] + hpw - 1) / hpw;
  const int64_t toks = (int64_t)a.s * a.b;
  Plan p;
  const int64_t want = std::min<int64_t>(np, std::max<int64_t>(1, 2048 / std::max<int64_t>(1, toks)));
  p.ppw = (int)((np + want - 1) / want);
  p.chunks = (np + p.ppw - 1) / p.ppw;
  p.gx = (toks + kWaves - 1) / kWaves;
  if (persistent) p.gx = std::min<int64_t>(p.gx, std::max(1, 1024 / p.chunks));
  return p;
}

}  // namespace

void qk_rope_forward(int dt, const QkRopeArgs& a, hipStream_t st) {
  const Plan p = plan(a, false);
  dispatch(dt, a, [&](auto t, auto lpr, auto vec, auto norm) {
    hipLaunchKernelGGL((k_qk_rope_fwd<typename decltype(t)::type, decltype(lpr)::value, decltype(vec)::value,
                                      decltype(norm)::value>),
                       dim3((unsigned)p.gx, (unsigned)p.chunks), dim3(kThreads), 0, st, a, p.ppw);
  });
  check_launch("qk_norm_rope forward");
}

int64_t qk_rope_partial_rows(const QkRopeArgs& a) {
  if (!a.w[0]) return 0;
  const Plan p = plan(a, true);
  return p.gx * p.chunks;
}

void qk_rope_backward(int dt, const QkRopeArgs& a, float* partials, void* dwq, void* dwk, hipStream_t st) {
  const bool norm = a.w[0] != nullptr;
  const Plan p = plan(a, norm);
  dispatch(dt, a, [&](auto t, auto lpr, auto vec, auto nn) {
    hipLaunchKernelGGL((k_qk_rope_bwd<typename decltype(t)::type, decltype(lpr)::value, decltype(vec)::value,
                                      decltype(nn)::value>),
                       dim3((unsigned)p.gx, (unsigned)p.chunks), dim3(kThreads), 0, st, a, p.ppw, partials);
  });
  if (norm) {
    const dim3 grid((unsigned)((a.hn + 63) / 64), 2);
    const int rows = (int)(p.gx * p.chunks);
    auto sums = [&](auto w) {
      using W = typename decltype(w)::type;
      hipLaunchKernelGGL((k_qk_rope_dw<W>), grid, dim3(1024), 0, st, partials, rows, a.hn, reinterpret_cast<W*>(dwq),
                         reinterpret_cast<W*>(dwk));
    };
    if (a.w_dt == kF16) sums(TypeTag<f16>{});
    else if (a.w_dt == kBF16) sums(TypeTag<bf16>{});
    else sums(TypeTag<float>{});
  }
  check_launch("qk_norm_rope backward");
}

}  // namespace bh
