// Grouped-query attention, forward and recomputing backward (gfx950, MFMA 32x32x16).
//
//   S = scale Q K^T,  P = softmax of S over the keys a query sees,  O = (P * keep / (1 - p)) V
//   dV = Pd^T dO,  dP = (dO V^T) * keep / (1 - p),  delta = rowsum(dO * O),  dS = P (dP - delta),
//   dQ = scale dS K,  dK = scale dS^T Q
//
// The forward keeps one number per query, L = log2 sum 2^(scale log2(e) s); the backward rebuilds
// P = 2^(scale log2(e) s - L). Scores, sums, L, delta and every accumulator are fp32; P and dS are rounded to
// the tensors' 16-bit type where they enter a matrix product (their rounding errors are independent and
// average out over the keys, like the rounding of the inputs).
#include "bh/api.h"
#include "bh/grouped_attn_api.h"
#include "bh/mfma32.h"

#include <algorithm>
#include <type_traits>
#include <stdexcept>
#include <string>

namespace bh {
namespace {

using namespace m32;

constexpr int kThreads = 256;  // 4 waves
constexpr int kTileQ = 128;    // rows of a workgroup: 32 per wave
constexpr int kBlk = 64;       // rows of the streamed operand per step
constexpr float kLog2e = 1.4426950408889634f;

// ---- LDS images ------------------------------------------------------------------------------------------
// Row-major, 2 D bytes a row, 16-byte chunks XOR-swizzled by the row so that both reads are conflict free:
// 16 consecutive rows of one chunk (ds_read_b128) land in 16 different slots, and the 4 consecutive rows x
// 64 bytes of a transposed read (ds_read_b64_tr_b16) in 4 different quarters of the 256-byte bank line.
template <int D> BH_HD constexpr int swz(int row) {
  return D == 64 ? ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) : (((row & 3) << 2) | ((row >> 2) & 3));
}
template <int D> struct Frag {
  static constexpr int RB = 2 * D;
  int r0, lo, hi;  // this lane's byte offsets; the swizzle only mixes chunk bits, so a step is one XOR
  BH_DEVICE explicit Frag(int lane) {
    const int r = lane & 31, h = lane >> 5;
    r0 = r * RB + ((h ^ swz<D>(r)) << 4);
    const int g = (lane >> 4) & 1, q = (lane & 15) >> 2, p = lane & 3;
    const int row = 4 * h + q, ch = 2 * g + (p >> 1), b = (p & 1) << 3;
    lo = row * RB + ((ch ^ swz<D>(row)) << 4) + b;
    hi = (row + 8) * RB + ((ch ^ swz<D>(row + 8)) << 4) + b;
  }
  // rows `row0 ..+31`, columns 16 s ..+15 as a row operand (row0 a multiple of 16)
  BH_DEVICE i4v row(const char* img, int row0, int s) const {
    return *reinterpret_cast<const i4v*>(img + row0 * RB + (r0 ^ (s << 5)));
  }
  // columns 32 dn ..+31 as rows, k = image rows k0 ..+15 in the register order of an accumulator tile
  BH_DEVICE i4v tr(const char* img, int k0, int dn) const {
    const s4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(img + k0 * RB + (lo ^ (dn << 6))));
    const s4v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(img + k0 * RB + (hi ^ (dn << 6))));
    const i2v x = __builtin_bit_cast(i2v, a), y = __builtin_bit_cast(i2v, b);
    return i4v{x[0], x[1], y[0], y[1]};
  }
};

// LDS-DMA of ROWS rows of one operand by NW waves (wave index w of them): rows past the tensor's last and
// columns past the head size land as zeros. Offsets stay below 2^31 for row strides below 2^24 elements
// (checked on the host); the 64-bit part of the address is in the resource's base.
template <int D, int ROWS, int NW> struct Stage {
  static constexpr int RB = 2 * D, CH = RB / 16, NP = ROWS * RB / 1024 / NW;
  int voff[NP];
  BH_DEVICE Stage(int64_t st, int hn, int w, int lane) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int row = (w * NP + i) * (64 / CH) + lane / CH, ch = (lane % CH) ^ swz<D>(row);
      voff[i] = 8 * ch < hn ? row * (int)st * 2 + ch * 16 : kOutOfRange;
    }
  }
  template <typename T>
  BH_DEVICE void issue(const T* base, int64_t st, int hn, int valid, const char* img, int w) const {
    const int n = min(valid, ROWS);
    const i4v rs = make_rsrc(base, n > 0 ? (uint32_t)(((n - 1) * (int)st + hn) * 2) : 0u);
    const unsigned l = __builtin_amdgcn_readfirstlane(lds_addr(img) + w * (NP * 1024));
#pragma unroll
    for (int i = 0; i < NP; ++i) dma16(rs, voff[i], l + i * 1024);
  }
};

// 8 columns of one row straight from memory as a matrix operand; zeros past the head size or the last row
template <typename T> BH_DEVICE i4v load_frag(const T* base, int64_t st, int row, int rows, int col, int hn) {
  if (row < rows && col < hn) return *reinterpret_cast<const i4v*>(base + (int64_t)row * st + col);
  return i4v{0, 0, 0, 0};
}

template <typename T> BH_DEVICE T* at(const GaView& v, int b, int h, void* base) {
  return reinterpret_cast<T*>(base) + (int64_t)b * v.sb + (int64_t)h * v.sh;
}
template <typename T> BH_DEVICE T* at(const GaView& v, int b, int h) { return at<T>(v, b, h, v.p); }
// 4 output values and, for the backward pass, what their rounding left over
template <typename T> BH_DEVICE void store_out(T* out, T* rest, float a, float b, float c, float d) {
  store4<T>(out, a, b, c, d);
  if (rest)
    store4<T>(rest, a - to_f<T>(from_f<T>(a)), b - to_f<T>(from_f<T>(b)), c - to_f<T>(from_f<T>(c)),
              d - to_f<T>(from_f<T>(d)));
}
BH_DEVICE uint64_t eff_seed(const GaArgs& a) {
  return a.seed_dev ? a.seed ^ ((uint64_t)*a.seed_dev * 0x9E3779B97F4A7C15ull) : a.seed;
}
BH_DEVICE int seq_keys(const GaArgs& a, int b) {
  return a.lens ? __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.sk)) : a.sk;
}

// Problem of a workgroup on a 1-D grid of nx tiles x (b * ng) key heads x per heads. Workgroups go round-robin
// to the 8 XCDs, each with an L2 of its own, so the tiles and query heads that read one key head's K / V stay
// on one XCD where the count of key heads allows; an XCD takes neighbouring key heads, whose rows lie on
// different channels of its L2 (2048 x 2500 keys, 16 heads in a fused projection: forward 248 us, 258 with every
// eighth head, both before rows were stored whole). tile_major: all problems' tile 0 first (causal: heaviest tiles
// first, the light ones fill the gaps at the end), else a key head's tiles run together.
struct Problem {
  int tile, unit, j;
};
BH_DEVICE Problem problem(int nx, int units, int per, bool tile_major) {
  const int id = blockIdx.x;
  const int nxcd = (units & 7) == 0 ? 8 : 1;
  const int xcd = id % nxcd, slot = id / nxcd, u = units / nxcd;
  Problem p;
  if (tile_major) {
    p.tile = slot / (u * per);
    const int rem = slot - p.tile * (u * per);
    p.unit = xcd * u + rem / per;
    p.j = rem % per;
  } else {
    p.unit = xcd * u + slot / (nx * per);
    const int rem = slot % (nx * per);
    p.tile = rem / per;
    p.j = rem % per;
  }
  return p;
}

// Writes a wave's accumulators (32 rows on the lanes, dims in the registers) to rows of D values in memory. Straight
// from the registers a store instruction would touch 32 rows with 16 bytes each; through LDS of the wave's own it
// writes whole rows, 16 bytes a lane (forward of 2048 x 2500 keys, 16 heads of 128: 242 -> 197 us; 4096 tokens,
// window 512: 71 -> 64 us). The backward kernels store from the registers: with this they were 1 to 2 % slower at
// D = 128, whose loops have no registers to spare, and no faster at D = 64.
template <typename T, int D> struct RowsOut {
  static constexpr int DN = D / 32, RS = 2 * D + 16, BYTES = 32 * RS;
  static constexpr int CH = D / 8, STEP = 64 / CH;  // chunks of 8 values a row, rows a store
  char* lds;
  int lane;
  // value(dn, i): what goes to dim 32 dn + acc_row(i) + 4 h of this lane's row
  template <typename F> BH_DEVICE void put(F&& value) const {
    char* at = lds + (lane & 31) * RS + 8 * (lane >> 5);
#pragma unroll
    for (int dn = 0; dn < DN; ++dn)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        store4<T>(reinterpret_cast<T*>(at) + 32 * dn + 8 * q, value(dn, 4 * q), value(dn, 4 * q + 1),
                  value(dn, 4 * q + 2), value(dn, 4 * q + 3));
  }
  // rows 0 .. rows - 1 to dst + row * st, their first n values
  BH_DEVICE void flush(T* dst, int64_t st, int rows, int n) const {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // one wave's LDS: its own order is enough
    const int ch = lane % CH;
#pragma unroll
    for (int i = 0; i < 32 / STEP; ++i) {
      const int row = i * STEP + lane / CH;
      const i4v v = *reinterpret_cast<const i4v*>(lds + row * RS + ch * 16);
      if (row < rows && 8 * ch < n) *reinterpret_cast<i4v*>(dst + (int64_t)row * st + 8 * ch) = v;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
};

// Blocks per turn of a loop over a double buffer. At two of them the buffer's index is a constant in the unrolled body,
// so that LDS addresses are registers made once plus immediates (sq = 8192, 32 heads on 8, D = 128, causal: forward
// 558 -> 550 us, backward 1759 -> 1732 us). The 64-channel kernels, whose register limits are tighter, lost more than
// that (forward 36.0 -> 37.6 us, backward 104 -> 122 us at 8 x 1024 x 16 heads).
template <int D> constexpr int kTurn = D == 128 ? 2 : 1;
// buffer of block `block`, the `side`th of its turn
template <int D> BH_DEVICE int buffer_of(int side, int block) { return (kTurn<D> == 2 ? side : block) & 1; }

// dP - delta without a subtraction: dP's products start from -delta (backward of the same case 1790 -> 1759 us). Not
// where dropout scales dP first, nor at 64 channels, where the 16 registers of the start spill.
template <int D, bool DROP> constexpr bool kFromDelta = D == 128 && !DROP;

// masks the scores of one 32-key (32-query) tile whose register i stands for offset acc_row(i): keeps
// lo <= offset <= hi
BH_DEVICE void mask_hi(f16v& s, int hi) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (acc_row(i) > hi) s[i] = -INFINITY;
}
BH_DEVICE void mask_lo(f16v& s, int lo) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (acc_row(i) < lo) s[i] = -INFINITY;
}
BH_DEVICE float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
BH_DEVICE float tile_max(const f16v& s) {
  const float a = max3(s[0], s[1], s[2]), b = max3(s[3], s[4], s[5]), c = max3(s[6], s[7], s[8]);
  const float d = max3(s[9], s[10], s[11]), e = max3(s[12], s[13], s[14]);
  return max3(max3(a, b, c), max3(d, e, s[15]), s[15]);
}

// ---- forward ---------------------------------------------------------------------------------------------
// Workgroup = 4 waves x 32 queries of one head, the query on the lane: S^T = K Q^T puts a query's scores of a
// 64-key block into one lane pair's registers, so the softmax needs one half-wave exchange and P^T feeds
// O^T = V^T P^T from the accumulators. The running maximum is only raised when some query's block maximum
// passes it by more than 2^8 (P <= 256 rounds as well as P <= 1; a wave-uniform vote).
// K / V blocks arrive by LDS-DMA one block ahead: one barrier a block. Two workgroups a CU (D = 128: 64 KiB of LDS and
// 224 registers; four at D = 64) run against each other's matrix and exponential phases.
// 8192 causal bf16 tokens, 32 heads of 128 over 8: 0.55 ms, 1.0 PFLOP/s (a large matrix product reaches 1.3).
// The matrix unit is busy 46 % of the cycles; without the LDS-DMA 20 % less time, without exponentials 10 %,
// without LDS reads 17 % (on zeros, which do not throttle the clock). Measured and not kept, same shape: 8 waves on
// 256 queries 567 us or on two heads of a group 576 us (557 with 4), three buffers 596 us, the scores of the next
// 32 keys issued by hand between the exponentials of this one 547 us (532).
template <typename T, int D, bool DROP>
__global__ __launch_bounds__(kThreads, 2) void k_ga_fwd(GaArgs a, int nx, uint32_t thresh, float kscale) {
  constexpr int RB = 2 * D, IMG = kBlk * RB, KS = D / 16, DN = D / 32;
  __shared__ __attribute__((aligned(16))) char smem[4 * IMG];  // {K, V} x 2 buffers
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int r = a.np / a.ng;
  Problem pr = problem(nx, a.b * a.ng, r, a.causal);
  if (a.causal) pr.tile = nx - 1 - pr.tile;
  const int b = pr.unit / a.ng, g = pr.unit % a.ng, head = g * r + pr.j, bh = b * a.np + head;
  const int nk = seq_keys(a, b), off = a.sk - a.sq;
  const int q0 = pr.tile * kTileQ, q0w = q0 + wave * 32, myq = q0w + r32, pos = myq + off;
  const int qlw = min(q0w + 31, a.sq - 1);  // the wave's last query

  const T* K = at<const T>(a.k, b, g);
  const T* V = at<const T>(a.v, b, g);
  const T* Q = at<const T>(a.q, b, head);
  i4v qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = load_frag<T>(Q, a.q.st, myq, a.sq, 16 * s + 8 * h, a.hn);

  const float c = a.scale * kLog2e;
  const uint32_t rowh = DROP ? row_hash(eff_seed(a), bh, myq) : 0u;
  float m = -INFINITY, l = 0.f;  // running base-2 maximum (both halves agree), this half's sum
  f16v O[DN];                    // O^T: dims 32 dn + acc_row(i) + 4h of query myq
#pragma unroll
  for (int dn = 0; dn < DN; ++dn) O[dn] = zero16();

  int kbeg = 0, kend = nk;
  if (a.causal) {
    kend = min(nk, min(q0 + kTileQ, a.sq) + off);
    kbeg = max(0, q0 + off - a.window + 1) & ~(kBlk - 1);
  }
  const int nb = kend > kbeg ? (kend - kbeg + kBlk - 1) / kBlk : 0;
  const Stage<D, kBlk, 4> sk(a.k.st, a.hn, wave, lane), sv(a.v.st, a.hn, wave, lane);
  const Frag<D> fr(lane);
  auto stage = [&](int kb, char* buf) {
    sk.issue(K + (int64_t)kb * a.k.st, a.k.st, a.hn, nk - kb, buf, wave);
    sv.issue(V + (int64_t)kb * a.v.st, a.v.st, a.hn, nk - kb, buf + IMG, wave);
  };
  if (nb > 0) stage(kbeg, smem);
  for (int turn = 0; turn < nb; turn += kTurn<D>) {
#pragma unroll
    for (int side = 0; side < kTurn<D>; ++side) {
      const int ib = turn + side;
      if (ib >= nb) break;
      const int kb = kbeg + ib * kBlk;
      const char* kimg = smem + buffer_of<D>(side, ib) * 2 * IMG;
      const char* vimg = kimg + IMG;
      wait_vmcnt<0>();
      lds_barrier();  // block ib is in LDS, block ib - 1 is read by every wave
      if (ib + 1 < nb) stage(kb + kBlk, smem + buffer_of<D>(side + 1, ib + 1) * 2 * IMG);
      if (q0w >= a.sq) continue;
      if (a.causal && (kb > qlw + off || kb + kBlk - 1 < q0w + off - a.window + 1)) continue;
      f16v S[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        S[t] = zero16();
#pragma unroll
        for (int s = 0; s < KS; ++s) S[t] = Mfma<T>::run(fr.row(kimg, 32 * t, s), qf[s], S[t]);
      }
      const bool diag = a.causal && kb + kBlk - 1 > q0w + off;
      if (diag || kb + kBlk > nk) {
        const int hi = (a.causal ? min(pos, nk - 1) : nk - 1) - kb - 4 * h;
#pragma unroll
        for (int t = 0; t < 2; ++t) mask_hi(S[t], hi - 32 * t);
      }
      if (a.causal && kb < qlw + off - a.window + 1) {
        const int lo = pos - a.window + 1 - kb - 4 * h;
#pragma unroll
        for (int t = 0; t < 2; ++t) mask_lo(S[t], lo - 32 * t);
      }
      const float mx = half_max(fmaxf(tile_max(S[0]), tile_max(S[1]))) * c;
      if (__any(mx > m + 8.f)) {
        const float mn = fmaxf(m, mx);
        const float corr = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        l *= corr;
#pragma unroll
        for (int dn = 0; dn < DN; ++dn)
#pragma unroll
          for (int i = 0; i < 16; ++i) O[dn][i] *= corr;
        m = mn;
      }
      const float nm = m == -INFINITY ? 0.f : -m;
      float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(S[t][i], c, nm));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(S[t][i + 1], c, nm));
          ls[(i >> 1) & 3] += p0 + p1;
          if (DROP) {
            const uint32_t x = pair_hash(rowh, kb + 32 * t + acc_row(i) + 4 * h);
            S[t][i] = keep_even(x, thresh) ? p0 : 0.f;
            S[t][i + 1] = keep_odd(x, thresh) ? p1 : 0.f;
          } else {
            S[t][i] = p0;
            S[t][i + 1] = p1;
          }
        }
      l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const i4v pb = pack8<T>(S[t], u);
#pragma unroll
          for (int dn = 0; dn < DN; ++dn) O[dn] = Mfma<T>::run(fr.tr(vimg, 32 * t + 16 * u, dn), pb, O[dn]);
        }
    }
  }
  l = half_sum(l);
  if (h == 0 && myq < a.sq) a.lse[(int64_t)bh * a.sq + myq] = l == 0.f ? INFINITY : m + __log2f(l);
  const float inv = l > 0.f ? (DROP ? kscale : 1.f) / l : (l == 0.f ? 0.f : l);  // no key: zeros; NaN stays
  lds_barrier();  // every wave is done with the blocks
  const RowsOut<T, D> out{smem + wave * RowsOut<T, D>::BYTES, lane};
  const int64_t at_o = (int64_t)q0w * a.o.st;
  out.put([&](int dn, int i) { return O[dn][i] * inv; });
  out.flush(at<T>(a.o, b, head) + at_o, a.o.st, a.sq - q0w, a.hn);
  if (a.olo) {
    out.put([&](int dn, int i) {
      const float x = O[dn][i] * inv;
      return x - to_f<T>(from_f<T>(x));
    });
    out.flush(at<T>(a.o, b, head, a.olo) + at_o, a.o.st, a.sq - q0w, a.hn);
  }
}

// ---- forward, keys split over waves and workgroups ---------------------------------------------------------
// For grids that would leave the card empty (few queries: single tokens against a long cache). The 32 lanes of
// a tile are packed rows of one key head (all r query heads of its group x sq queries) so a group's K / V
// are read once. Every wave walks its own 32-key blocks through an LDS buffer of its own (no barrier in the
// loop); eight waves on a CU with one block in flight each keep the memory busy: 8 tokens against 4099 keys, 32
// heads over 8, half the keys there, take 15 + 4 us (34 MB of K / V); four waves that compute one block while the
// next is in flight took 25 + 6 us. The waves join through LDS, the splits through an fp32 workspace. The kernel is
// bound by the latency of its few dependent steps: 256 workgroups of at most 5 blocks a wave. 512 workgroups
// took 31 us where 256 took 27, 128 took 29 (all keys there). Only the blocks that a tile's rows see are walked (8
// tokens, window 512 of 32768 keys: 10 us, 198 over all keys; 4096 causal tokens, 4 heads: 45 us, 57).
constexpr int kSplitWaves = 8, kSplitKeys = 32 * kSplitWaves, kJoinSerial = 8;
template <typename T, int D>
__global__ __launch_bounds__(64 * kSplitWaves, 2) void k_ga_split(GaArgs a, int rtiles, int splits, int chunk, int kbeg,
                                                                  float* __restrict__ ws) {
  constexpr int RB = 2 * D, IMG = 32 * RB, KS = D / 16, DN = D / 32, NP = IMG / 1024, NW = kSplitWaves;
  constexpr int OS = D + 4;  // floats of a joined row: 4 of padding keep the 32 rows off one bank
  constexpr int BYTES = NW * 2 * IMG > NW * 32 * OS * 4 ? NW * 2 * IMG : NW * 32 * OS * 4;
  __shared__ __attribute__((aligned(16))) char smem[BYTES];
  __shared__ float sml[2][NW][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int r = a.np / a.ng, rows = r * a.sq;
  // problems (units x row tiles) fastest: the splits of a unit are spread in time, not over XCDs
  const int units = a.b * a.ng, prob = blockIdx.x % (units * rtiles), split = blockIdx.x / (units * rtiles);
  const int unit = prob % units, rt = prob / units;
  const int b = unit / a.ng, g = unit % a.ng;
  const int nk = seq_keys(a, b), off = a.sk - a.sq;
  const T* K = at<const T>(a.k, b, g);
  const T* V = at<const T>(a.v, b, g);
  // the wave's blocks of the split that some row of the tile sees
  int k1 = min(nk, kbeg + split * chunk + chunk), first = kbeg + split * chunk + wave * 32;
  if (a.causal) {
    const int r0 = rt * 32, r1 = min(r0 + 31, rows - 1), j0 = r0 / a.sq, j1 = r1 / a.sq;
    const int i0 = j0 == j1 ? r0 - j0 * a.sq : 0, i1 = j0 == j1 ? r1 - j1 * a.sq : a.sq - 1;
    const int unseen = i0 + off - a.window + 1 - (first + 31);
    if (unseen > 0) first += (unseen + kSplitKeys - 1) / kSplitKeys * kSplitKeys;
    k1 = min(k1, i1 + off + 1);
  }
  const char* kimg = smem + wave * 2 * IMG;
  const char* vimg = kimg + IMG;
  const Stage<D, 32, 1> sk(a.k.st, a.hn, 0, lane), sv(a.v.st, a.hn, 0, lane);
  auto stage = [&](int kb) {
    sk.issue(K + (int64_t)kb * a.k.st, a.k.st, a.hn, nk - kb, kimg, 0);
    sv.issue(V + (int64_t)kb * a.v.st, a.v.st, a.hn, nk - kb, vimg, 0);
  };
  if (first < k1) stage(first);
  const int myr = rt * 32 + r32, jq = min(myr, rows - 1);
  const int j = jq / a.sq, i_q = jq - j * a.sq, pos = i_q + off;
  const T* Q = at<const T>(a.q, b, g * r) + (int64_t)j * a.q.sh;
  i4v qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = load_frag<T>(Q, a.q.st, i_q, a.sq, 16 * s + 8 * h, a.hn);
  const float c = a.scale * kLog2e;
  const Frag<D> fr(lane);
  float m = -INFINITY, l = 0.f;
  f16v O[DN];
#pragma unroll
  for (int dn = 0; dn < DN; ++dn) O[dn] = zero16();
  for (int kb = first; kb < k1; kb += kSplitKeys) {
    wait_vmcnt<0>();
    f16v S = zero16();
#pragma unroll
    for (int s = 0; s < KS; ++s) S = Mfma<T>::run(fr.row(kimg, 0, s), qf[s], S);
    i4v vf[2 * DN];
#pragma unroll
    for (int x = 0; x < 2 * DN; ++x) vf[x] = fr.tr(vimg, 16 * (x / DN), x % DN);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // both images are in registers: the next block may land
    if (kb + kSplitKeys < k1) stage(kb + kSplitKeys);
    mask_hi(S, (a.causal ? min(pos, nk - 1) : nk - 1) - kb - 4 * h);
    if (a.causal) mask_lo(S, pos - a.window + 1 - kb - 4 * h);
    const float mx = half_max(tile_max(S)) * c;
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx);
      const float corr = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      l *= corr;
#pragma unroll
      for (int dn = 0; dn < DN; ++dn)
#pragma unroll
        for (int i = 0; i < 16; ++i) O[dn][i] *= corr;
      m = mn;
    }
    const float nm = m == -INFINITY ? 0.f : -m;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      S[i] = __builtin_amdgcn_exp2f(fmaf(S[i], c, nm));
      l += S[i];
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const i4v pb = pack8<T>(S, u);
#pragma unroll
      for (int dn = 0; dn < DN; ++dn) O[dn] = Mfma<T>::run(vf[u * DN + dn], pb, O[dn]);
    }
  }
  l = half_sum(l);
  lds_barrier();  // every wave is done with its buffers: the same LDS now joins them
  float* jo = reinterpret_cast<float*>(smem);
  if (h == 0) {
    sml[0][wave][r32] = m;
    sml[1][wave][r32] = l;
  }
#pragma unroll
  for (int dn = 0; dn < DN; ++dn)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f4v*>(jo + (wave * 32 + r32) * OS + 32 * dn + 8 * q + 4 * h) =
          f4v{O[dn][4 * q], O[dn][4 * q + 1], O[dn][4 * q + 2], O[dn][4 * q + 3]};
  __syncthreads();
  constexpr int TPR = 64 * NW / 32, PER = D / TPR;  // threads a row, dims a thread
  const int row = tid / TPR, d0 = (tid % TPR) * PER, grow = rt * 32 + row;
  if (grow >= rows) return;
  float mm = -INFINITY;
#pragma unroll
  for (int w = 0; w < NW; ++w) mm = fmaxf(mm, sml[0][w][row]);
  float lw = 0.f, acc[PER];
#pragma unroll
  for (int d = 0; d < PER; ++d) acc[d] = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const float mw = sml[0][w][row], f = mw == -INFINITY ? (sml[1][w][row] == 0.f ? 0.f : 1.f)
                                                         : __builtin_amdgcn_exp2f(mw - mm);
    lw += f * sml[1][w][row];
#pragma unroll
    for (int d = 0; d < PER; ++d) acc[d] += f * jo[(w * 32 + row) * OS + d0 + d];
  }
  if (splits > 1) {
    const int64_t slot = ((int64_t)prob * splits + split) * 32 + row;
    float* wo = ws + slot * D + d0;
#pragma unroll
    for (int d = 0; d < PER; d += 4) *reinterpret_cast<f4v*>(wo + d) = f4v{acc[d], acc[d + 1], acc[d + 2], acc[d + 3]};
    float* wm = ws + (int64_t)units * rtiles * splits * 32 * D + slot * 2;
    if (d0 == 0) {
      wm[0] = mm;
      wm[1] = lw;
    }
    return;
  }
  const int jj = grow / a.sq, iq = grow - jj * a.sq, head = g * r + jj;
  const float inv = lw > 0.f ? 1.f / lw : (lw == 0.f ? 0.f : lw);
  const int64_t at_o = (int64_t)iq * a.o.st + d0;
  T* out = at<T>(a.o, b, head) + at_o;
  T* rest = a.olo ? at<T>(a.o, b, head, a.olo) + at_o : nullptr;
#pragma unroll
  for (int d = 0; d < PER; d += 4)
    if (d0 + d < a.hn)
      store_out<T>(out + d, rest ? rest + d : nullptr, acc[d] * inv, acc[d + 1] * inv, acc[d + 2] * inv,
                   acc[d + 3] * inv);
  if (d0 == 0) a.lse[((int64_t)b * a.np + head) * a.sq + iq] = lw == 0.f ? INFINITY : mm + __log2f(lw);
}

// Joins the splits: D / 4 threads a row with 4 dims each, GR times over, each group every GR-th split with 4 splits'
// loads in flight; the groups meet in LDS. GR = 1 for up to kJoinSerial splits, else a workgroup a row. One token, 32
// heads over 8, 4099 keys, forward with GR = 1 and GR = 8: 4 splits (8 sequences) 27.1 and 27.9 us, 8 splits 18.0 and
// 17.9 us, 16 splits 13.5 and 12.4 us; 64 splits (1 sequence, 8 heads over 1, 16384 keys) 21.8 and 11.8 us.
template <typename T, int D, int GR>
__global__ __launch_bounds__(kThreads) void k_ga_join(GaArgs a, int rtiles, int splits, const float* __restrict__ ws) {
  constexpr int TPR = D / 4, RPB = kThreads / (TPR * GR);
  static_assert(GR == 1 || RPB == 1, "a workgroup whose row is behind the last leaves before the barrier");
  __shared__ float sm[GR], sl[GR];
  __shared__ f4v so[GR][TPR];
  const int r = a.np / a.ng, rows = r * a.sq, units = a.b * a.ng;
  const int64_t id = (int64_t)blockIdx.x * RPB + (GR == 1 ? threadIdx.x / TPR : 0);
  const int prob = (int)(id / 32), row = (int)(id % 32), grp = GR == 1 ? 0 : threadIdx.x / TPR;
  const int t = threadIdx.x % TPR, d = t * 4;
  if (prob >= units * rtiles) return;
  const int unit = prob % units, grow = prob / units * 32 + row;
  if (grow >= rows) return;
  const float* wo = ws + ((int64_t)prob * splits * 32 + row) * D + d;
  const float* wm = ws + (int64_t)units * rtiles * splits * 32 * D + ((int64_t)prob * splits * 32 + row) * 2;
  // the running maximum rescales what is already there
  float mm = -INFINITY, l = 0.f;
  f4v acc = f4v{0.f, 0.f, 0.f, 0.f};
  auto scale_of = [](float m, float sum, float to) {  // no key: 0; NaN stays
    return m == -INFINITY ? (sum == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - to);
  };
  for (int s0 = grp; s0 < splits; s0 += 4 * GR) {
    float ms[4], ls[4];
    f4v o[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int64_t s = min(s0 + x * GR, splits - 1);
      ms[x] = wm[s * 64];
      ls[x] = s0 + x * GR < splits ? wm[s * 64 + 1] : 0.f;
      o[x] = *reinterpret_cast<const f4v*>(wo + s * 32 * D);
    }
    const float mn = fmaxf(mm, fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])));
    const float corr = scale_of(mm, l, mn);
    mm = mn;
    l *= corr;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= corr;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (s0 + x * GR >= splits) break;
      const float f = scale_of(ms[x], ls[x], mm);
      l += f * ls[x];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += f * o[x][i];
    }
  }
  if constexpr (GR > 1) {
    if (t == 0) {
      sm[grp] = mm;
      sl[grp] = l;
    }
    so[grp][t] = acc;
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int x = 1; x < GR; ++x) mm = fmaxf(mm, sm[x]);
    l = 0.f;
    acc = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < GR; ++x) {
      const float f = scale_of(sm[x], sl[x], mm);
      l += f * sl[x];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += f * so[x][t][i];
    }
  }
  const int b = unit / a.ng, g = unit % a.ng, jj = grow / a.sq, iq = grow - jj * a.sq, head = g * r + jj;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  if (d < a.hn) {
    const int64_t at_o = (int64_t)iq * a.o.st + d;
    store_out<T>(at<T>(a.o, b, head) + at_o, a.olo ? at<T>(a.o, b, head, a.olo) + at_o : nullptr, acc[0] * inv,
                 acc[1] * inv, acc[2] * inv, acc[3] * inv);
  }
  if (d == 0) a.lse[((int64_t)b * a.np + head) * a.sq + iq] = l == 0.f ? INFINITY : mm + __log2f(l);
}

// ---- backward --------------------------------------------------------------------------------------------
// sum of the products of 8 values of two operand fragments
template <typename T> BH_DEVICE float dot8(i4v x, i4v y, float acc) {
  typedef T t8v __attribute__((ext_vector_type(8)));
  const t8v a = __builtin_bit_cast(t8v, x), b = __builtin_bit_cast(t8v, y);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc = fmaf(to_f<T>(a[i]), to_f<T>(b[i]), acc);
  return acc;
}

// dQ: the forward's layout. S^T = K Q^T and dP^T = V dO^T from row fragments, dS^T stays in registers and feeds
// dQ^T = K^T dS^T (K^T by transposed reads of the same image). It runs before the dK / dV kernel and leaves
// delta (and the dropout row hashes) for it: its dO fragments are in registers anyway. delta is taken from O
// with its rounding's rest: where few keys carry a query, dP - delta cancels and the rounding of O alone would
// be a good part of dS (GPT-2-medium's shape: error of dQ 2.5e-3 instead of 2.35e-3, dS rounding included).
template <typename T, int D, bool DROP>
__global__ __launch_bounds__(kThreads, D == 64 ? 4 : 2) void k_ga_dq(GaArgs a, int nx, uint32_t thresh, float kscale) {
  constexpr bool FROM = kFromDelta<D, DROP>;
  constexpr int RB = 2 * D, IMG = kBlk * RB, KS = D / 16, DN = D / 32;
  __shared__ __attribute__((aligned(16))) char smem[4 * IMG];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int r = a.np / a.ng;
  Problem pr = problem(nx, a.b * a.ng, r, a.causal);
  if (a.causal) pr.tile = nx - 1 - pr.tile;
  const int b = pr.unit / a.ng, g = pr.unit % a.ng, head = g * r + pr.j, bh = b * a.np + head;
  const int nk = seq_keys(a, b), off = a.sk - a.sq;
  const int q0 = pr.tile * kTileQ, q0w = q0 + wave * 32, myq = q0w + r32, pos = myq + off;
  const int qlw = min(q0w + 31, a.sq - 1);
  const T* K = at<const T>(a.k, b, g);
  const T* V = at<const T>(a.v, b, g);
  i4v qf[KS], df[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    qf[s] = load_frag<T>(at<const T>(a.q, b, head), a.q.st, myq, a.sq, 16 * s + 8 * h, a.hn);
    df[s] = load_frag<T>(at<const T>(a.dout, b, head), a.dout.st, myq, a.sq, 16 * s + 8 * h, a.hn);
  }
  const float c = a.scale * kLog2e;
  const int64_t row = (int64_t)bh * a.sq + min(myq, a.sq - 1);
  const float nl = -a.lse[row];
  float dl = 0.f;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    dl = dot8<T>(load_frag<T>(at<const T>(a.o, b, head), a.o.st, myq, a.sq, 16 * s + 8 * h, a.hn), df[s], dl);
    dl = dot8<T>(load_frag<T>(at<const T>(a.o, b, head, a.olo), a.o.st, myq, a.sq, 16 * s + 8 * h, a.hn), df[s], dl);
  }
  dl = half_sum(dl);
  const uint32_t rowh = DROP ? row_hash(eff_seed(a), bh, myq) : 0u;
  if (h == 0 && myq < a.sq) {
    a.delta[row] = FROM ? -dl : dl;
    if (DROP) a.rowh[row] = rowh;
  }
  f16v acc[DN];
#pragma unroll
  for (int dn = 0; dn < DN; ++dn) acc[dn] = zero16();
  int kbeg = 0, kend = nk;
  if (a.causal) {
    kend = min(nk, min(q0 + kTileQ, a.sq) + off);
    kbeg = max(0, q0 + off - a.window + 1) & ~(kBlk - 1);
  }
  const int nb = kend > kbeg ? (kend - kbeg + kBlk - 1) / kBlk : 0;
  const Stage<D, kBlk, 4> sk(a.k.st, a.hn, wave, lane), sv(a.v.st, a.hn, wave, lane);
  const Frag<D> fr(lane);
  auto stage = [&](int kb, char* buf) {
    sk.issue(K + (int64_t)kb * a.k.st, a.k.st, a.hn, nk - kb, buf, wave);
    sv.issue(V + (int64_t)kb * a.v.st, a.v.st, a.hn, nk - kb, buf + IMG, wave);
  };
  if (nb > 0) stage(kbeg, smem);
  f16v start;
#pragma unroll
  for (int i = 0; i < 16; ++i) start[i] = FROM ? -dl : 0.f;
  for (int turn = 0; turn < nb; turn += kTurn<D>) {
#pragma unroll
    for (int side = 0; side < kTurn<D>; ++side) {
      const int ib = turn + side;
      if (ib >= nb) break;
      const int kb = kbeg + ib * kBlk;
      const char* kimg = smem + buffer_of<D>(side, ib) * 2 * IMG;
      const char* vimg = kimg + IMG;
      wait_vmcnt<0>();
      lds_barrier();
      if (ib + 1 < nb) stage(kb + kBlk, smem + buffer_of<D>(side + 1, ib + 1) * 2 * IMG);
      if (q0w >= a.sq) continue;
      if (a.causal && (kb > qlw + off || kb + kBlk - 1 < q0w + off - a.window + 1)) continue;
      const bool mh = (a.causal && kb + kBlk - 1 > q0w + off) || kb + kBlk > nk;
      const bool ml = a.causal && kb < qlw + off - a.window + 1;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f16v S = zero16(), P = FROM ? start : zero16();
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          S = Mfma<T>::run(fr.row(kimg, 32 * t, s), qf[s], S);
          P = Mfma<T>::run(fr.row(vimg, 32 * t, s), df[s], P);  // dP^T
        }
        if (mh) mask_hi(S, (a.causal ? min(pos, nk - 1) : nk - 1) - kb - 4 * h - 32 * t);
        if (ml) mask_lo(S, pos - a.window + 1 - kb - 4 * h - 32 * t);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(S[i], c, nl));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(S[i + 1], c, nl));
          if (DROP) {
            const uint32_t x = pair_hash(rowh, kb + 32 * t + acc_row(i) + 4 * h);
            P[i] = p0 * ((keep_even(x, thresh) ? P[i] * kscale : 0.f) - dl);
            P[i + 1] = p1 * ((keep_odd(x, thresh) ? P[i + 1] * kscale : 0.f) - dl);
          } else {
            P[i] = p0 * (FROM ? P[i] : P[i] - dl);
            P[i + 1] = p1 * (FROM ? P[i + 1] : P[i + 1] - dl);
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const i4v sb = pack8<T>(P, u);
#pragma unroll
          for (int dn = 0; dn < DN; ++dn) acc[dn] = Mfma<T>::run(fr.tr(kimg, 32 * t + 16 * u, dn), sb, acc[dn]);
        }
      }
    }
  }
  if (myq < a.sq) {
    T* dq = at<T>(a.dq, b, head) + (int64_t)myq * a.dq.st;
#pragma unroll
    for (int dn = 0; dn < DN; ++dn)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (32 * dn + 8 * q < a.hn)
          store4<T>(dq + 32 * dn + 8 * q + 4 * h, acc[dn][4 * q] * a.scale, acc[dn][4 * q + 1] * a.scale,
                    acc[dn][4 * q + 2] * a.scale, acc[dn][4 * q + 3] * a.scale);
  }
}

// dK / dV: workgroup = 4 waves x 32 keys of one key head, the key on the lane; it walks the query blocks of all
// r query heads of the group, so the gradients of shared heads are summed in the accumulators (no atomics, one
// order). S = Q K^T and dP = dO V^T from row fragments, P and dS feed dV^T = dO^T P and dK^T = Q^T dS from the
// accumulators. L, delta and the row hashes of a block ride along.
// Registers decide the shape: K stays in registers, V is read from LDS again for every block. At D = 128 the
// accumulators take 128 of the 256 registers that two waves a SIMD leave (with V in registers 34 spilled, and
// 8192 causal keys took 2.70 ms instead of 1.05); at D = 64 it makes room for a third wave (GPT-2-medium's shape
// with dropout, dQ + dK / dV: 124 us, 129 with V in registers and two waves). Blocks are 32 queries at D = 128
// (LDS for two workgroups a CU), 64 at D = 64.
// The blocks of a key tile are cut into `splits` runs (few key tiles, or a causal mask that gives the first
// tiles most of the work); their fp32 sums then meet in k_ga_dkdv_join, in order.
template <typename T, int D, bool DROP>
__global__ __launch_bounds__(kThreads, D == 64 ? 3 : 2) void k_ga_dkdv(GaArgs a, int nx, int splits, uint32_t thresh,
                                                                       float kscale, float* __restrict__ ws) {
  constexpr int RB = 2 * D, QB = D == 64 ? 64 : 32, IMG = QB * RB, KS = D / 16, DN = D / 32, BUF = 2 * IMG + 3 * 256;
  __shared__ __attribute__((aligned(16))) char smem[2 * BUF + kTileQ * RB];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int r = a.np / a.ng;
  const Problem pr = problem(nx, a.b * a.ng, splits, a.causal);
  const int b = pr.unit / a.ng, g = pr.unit % a.ng;
  const int nk = seq_keys(a, b), off = a.sk - a.sq;
  const int k0 = pr.tile * kTileQ, k0w = k0 + wave * 32, mykey = k0w + r32;
  const bool odd = mykey & 1;
  const Frag<D> fr(lane);
  char* const vtile = smem + 2 * BUF + wave * 32 * RB;  // this wave's 32 keys
  i4v kf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    kf[s] = load_frag<T>(at<const T>(a.k, b, g), a.k.st, mykey, nk, 16 * s + 8 * h, a.hn);
    *reinterpret_cast<i4v*>(vtile + (fr.r0 ^ (s << 5))) =
        load_frag<T>(at<const T>(a.v, b, g), a.v.st, mykey, nk, 16 * s + 8 * h, a.hn);
  }
  const float c = a.scale * kLog2e;
  f16v dK[DN], dV[DN];
#pragma unroll
  for (int dn = 0; dn < DN; ++dn) dK[dn] = dV[dn] = zero16();
  // queries that see a key of the tile: key - off <= i < key - off + window
  int qbeg = 0, qend = k0 < nk ? a.sq : 0;
  if (a.causal) {
    qbeg = max(0, k0 - off) & ~(QB - 1);
    qend = min(qend, min(k0 + kTileQ, nk) - 1 - off + a.window);
  }
  const int nqb = qend > qbeg ? (qend - qbeg + QB - 1) / QB : 0, total = nqb * r;
  const int it0 = (int)((int64_t)total * pr.j / splits), it1 = (int)((int64_t)total * (pr.j + 1) / splits);
  const Stage<D, QB, 4> sq(a.q.st, a.hn, wave, lane), sd(a.dout.st, a.hn, wave, lane);
  auto stage = [&](int j, int q0, char* buf) {
    const int head = g * r + j;
    sq.issue(at<const T>(a.q, b, head) + (int64_t)q0 * a.q.st, a.q.st, a.hn, a.sq - q0, buf, wave);
    sd.issue(at<const T>(a.dout, b, head) + (int64_t)q0 * a.dout.st, a.dout.st, a.hn, a.sq - q0, buf + IMG, wave);
    // rows past the last query read as zeros: their Q and dO rows are zero too, so P = 1 meets dO = 0
    const int64_t row = ((int64_t)b * a.np + head) * a.sq + q0;
    const uint32_t bytes = 4u * (uint32_t)min(a.sq - q0, QB);
    const unsigned l = __builtin_amdgcn_readfirstlane(lds_addr(buf + 2 * IMG));
    if (wave == 0) dma4(make_rsrc(a.lse + row, bytes), lane * 4, l);
    else if (wave == 1) dma4(make_rsrc(a.delta + row, bytes), lane * 4, l + 256);
    else if (DROP && wave == 2) dma4(make_rsrc(a.rowh + row, bytes), lane * 4, l + 512);
  };
  int j = nqb ? it0 / nqb : 0, q0 = qbeg + (it0 - j * nqb) * QB;  // head of the group and first query of a block
  if (it0 < it1) stage(j, q0, smem);
  constexpr bool FROM = kFromDelta<D, DROP>;
  for (int turn = it0; turn < it1; turn += kTurn<D>) {
#pragma unroll
    for (int side = 0; side < kTurn<D>; ++side) {
      const int it = turn + side;
      if (it >= it1) break;
      const int qb = q0;
      const char* qimg = smem + buffer_of<D>(side, it - it0) * BUF;
      const char* dimg = qimg + IMG;
      const float* lp = reinterpret_cast<const float*>(dimg + IMG);
      wait_vmcnt<0>();
      lds_barrier();
      q0 += QB;
      if (q0 >= qend) {
        q0 = qbeg;
        ++j;
      }
      if (it + 1 < it1) stage(j, q0, smem + buffer_of<D>(side + 1, it - it0 + 1) * BUF);
      if (k0w >= nk) continue;
      if (a.causal && (qb + QB - 1 + off < k0w || qb + off - a.window + 1 > k0w + 31)) continue;
      const bool ml = a.causal && qb + off < k0w + 31;                       // some query precedes some key
      const bool mh = a.causal && qb + QB - 1 + off - a.window + 1 > k0w;    // some key left the window
#pragma unroll
      for (int t = 0; t < QB / 32; ++t) {
        f16v S = zero16(), P = zero16();
        if (FROM) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f4v d4 = *reinterpret_cast<const f4v*>(lp + 64 + 32 * t + 8 * q + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) P[4 * q + e] = d4[e];
          }
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          S = Mfma<T>::run(fr.row(qimg, 32 * t, s), kf[s], S);
          P = Mfma<T>::run(fr.row(dimg, 32 * t, s), fr.row(vtile, 0, s), P);  // dP
        }
        if (ml) mask_lo(S, mykey - off - qb - 4 * h - 32 * t);
        if (mh) mask_hi(S, mykey - off + a.window - 1 - qb - 4 * h - 32 * t);
        // Two neighbouring keys share a hash: the even lane takes the pair's for the first 16 queries, the odd one for
        // the other 16, and they swap.
        uint32_t hash[16];
        if (DROP) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const i4v r4 = *reinterpret_cast<const i4v*>(lp + 128 + 32 * t + 8 * q + 4 * h + (odd ? 16 : 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t mine = pair_hash((uint32_t)r4[e], mykey);
              const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)mine, 0xB1, 0xf, 0xf, true);
              hash[4 * q + e] = odd ? other : mine;
              hash[8 + 4 * q + e] = odd ? mine : other;
            }
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float* at4 = lp + 32 * t + 8 * q + 4 * h;
          const f4v l4 = *reinterpret_cast<const f4v*>(at4);
          f4v d4 = f4v{0.f, 0.f, 0.f, 0.f};
          if (!FROM) d4 = *reinterpret_cast<const f4v*>(at4 + 64);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 4 * q + e;
            const float p = __builtin_amdgcn_exp2f(fmaf(S[i], c, -l4[e]));
            if (DROP) {
              const float kk = keep16(fold16(hash[i]) >> (odd ? 16 : 0), thresh) ? kscale : 0.f;
              S[i] = p * kk;
              P[i] = p * (P[i] * kk - d4[e]);
            } else {
              S[i] = p;
              P[i] = p * (FROM ? P[i] : P[i] - d4[e]);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const i4v pb = pack8<T>(S, u), sb = pack8<T>(P, u);
#pragma unroll
          for (int dn = 0; dn < DN; ++dn) {
            dV[dn] = Mfma<T>::run(fr.tr(dimg, 32 * t + 16 * u, dn), pb, dV[dn]);
            dK[dn] = Mfma<T>::run(fr.tr(qimg, 32 * t + 16 * u, dn), sb, dK[dn]);
          }
        }
      }
    }
  }
  const bool real = mykey < nk;  // keys past the sequence's length take zeros, whatever their lanes held
  if (mykey >= a.sk) return;
  if (splits > 1) {
    float* w = ws + (((int64_t)pr.j * a.b * a.ng + pr.unit) * a.sk + mykey) * (2 * D) + 4 * h;
#pragma unroll
    for (int dn = 0; dn < DN; ++dn)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f4v x, y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = real ? dK[dn][4 * q + e] * a.scale : 0.f;
          y[e] = real ? dV[dn][4 * q + e] : 0.f;
        }
        *reinterpret_cast<f4v*>(w + 32 * dn + 8 * q) = x;
        *reinterpret_cast<f4v*>(w + D + 32 * dn + 8 * q) = y;
      }
    return;
  }
  T* dk = at<T>(a.dk, b, g) + (int64_t)mykey * a.dk.st + 4 * h;
  T* dv = at<T>(a.dv, b, g) + (int64_t)mykey * a.dv.st + 4 * h;
#pragma unroll
  for (int dn = 0; dn < DN; ++dn)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (32 * dn + 8 * q < a.hn) {
        float x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = real ? dK[dn][4 * q + e] * a.scale : 0.f;
          y[e] = real ? dV[dn][4 * q + e] : 0.f;
        }
        store4<T>(dk + 32 * dn + 8 * q, x[0], x[1], x[2], x[3]);
        store4<T>(dv + 32 * dn + 8 * q, y[0], y[1], y[2], y[3]);
      }
}

// dK / dV = sums of the splits' fp32 rows, in order; 2 D / 4 threads a key, 4 values each
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void k_ga_dkdv_join(GaArgs a, int splits, const float* __restrict__ ws) {
  constexpr int TPR = 2 * D / 4;
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x, row = id / TPR, rows = (int64_t)a.b * a.ng * a.sk;
  if (row >= rows) return;
  const int x = (int)(id % TPR) * 4, d = x % D;
  if (d >= a.hn) return;
  f4v acc = f4v{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) {
    const f4v v = *reinterpret_cast<const f4v*>(ws + ((int64_t)s * rows + row) * (2 * D) + x);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += v[i];
  }
  const int unit = (int)(row / a.sk), key = (int)(row - (int64_t)unit * a.sk);
  const GaView& o = x < D ? a.dk : a.dv;
  store4<T>(at<T>(o, unit / a.ng, unit % a.ng) + (int64_t)key * o.st + d, acc[0], acc[1], acc[2], acc[3]);
}

inline void check_launch(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw std::runtime_error(std::string(what) + ": " + hipGetErrorString(e));
}
template <typename T> struct TypeTag { using type = T; };
template <typename F> void dispatch(int dt, int hn, bool drop, F&& f) {
  auto by_d = [&](auto t) {
    auto by_drop = [&](auto d) {
      if (drop) f(t, d, std::true_type{});
      else f(t, d, std::false_type{});
    };
    if (hn <= 64) by_drop(std::integral_constant<int, 64>{});
    else by_drop(std::integral_constant<int, 128>{});
  };
  switch (dt) {
    case kF16: by_d(TypeTag<f16>{}); break;
    case kBF16: by_d(TypeTag<bf16>{}); break;
    default: throw std::runtime_error("grouped attention: fp16 / bf16 only");
  }
}
// keep where a 16-bit hash is below this: floor((1 - p) 2^16)
uint32_t keep_thresh(const GaArgs& a) { return (uint32_t)std::min(65536.0, (1.0 - a.p_drop) * 65536.0); }
// whether any weight is dropped: a threshold of 2^16 keeps all (and would not fit the kernels' 16-bit compare)
bool drops(const GaArgs& a) { return a.p_drop > 0. && keep_thresh(a) < 65536u; }
float keep_scale(const GaArgs& a) { return (float)(1.0 / (1.0 - a.p_drop)); }

struct SplitPlan {
  int rtiles = 0, splits = 0, chunk = 0, kbeg = 0;  // splits == 0: the tiled forward; keys before kbeg: no one's
};
SplitPlan split_plan(const GaArgs& a) {
  SplitPlan p;
  const int64_t tiled = (int64_t)((a.sq + kTileQ - 1) / kTileQ) * a.b * a.np;
  const int64_t rows = (int64_t)(a.np / a.ng) * a.sq, rt = (rows + 31) / 32, probs = rt * a.b * a.ng;
  if (drops(a) || (tiled >= 256 && rows > 64)) return p;
  if (a.causal) p.kbeg = std::max(0, a.sk - a.sq - a.window + 1) & ~31;
  const int64_t keys = a.sk - p.kbeg;
  const int64_t want = std::max<int64_t>(1, 256 / probs), most = (keys + kSplitKeys - 1) / kSplitKeys;
  const int64_t s = std::min(want, most);
  p.rtiles = (int)rt;
  p.chunk = (int)(((keys + s - 1) / s + kSplitKeys - 1) / kSplitKeys * kSplitKeys);
  p.splits = (int)((keys + p.chunk - 1) / p.chunk);
  return p;
}

// Runs of a key tile's query blocks. 512 workgroups fill the card; under a plain causal mask the first key tiles
// have most of the work, and twice as many, heaviest first, level that out (8192 causal keys, 8 key heads of 128:
// backward 1751 us with 2 runs, 2292 with 1, 1767 with 4). Where tiles weigh the same, more than 512 only adds
// partial sums (4096 keys, window 512, 8 key heads: 192 us with 2 runs, 220 with 4, 206 with 1). A run has at
// least 2 blocks of 64 queries.
int dkdv_splits(const GaArgs& a) {
  const int64_t wgs = (int64_t)((a.sk + kTileQ - 1) / kTileQ) * a.b * a.ng;
  const int64_t blocks = ((int64_t)std::min<int64_t>(a.sq, (int64_t)a.window + kTileQ) + 63) / 64 * (a.np / a.ng);
  const int64_t target = a.causal && a.window >= a.sk ? 1024 : 512;
  return (int)std::max<int64_t>(1, std::min(target / wgs, blocks / 2));
}

}  // namespace

int64_t ga_forward_workspace(const GaArgs& a) {
  const SplitPlan p = split_plan(a);
  if (p.splits <= 1) return 0;
  const int64_t d = a.hn <= 64 ? 64 : 128;
  return (int64_t)a.b * a.ng * p.rtiles * p.splits * 32 * (d + 2);
}

void ga_forward(int dt, const GaArgs& a, float* ws, hipStream_t st) {
  const SplitPlan p = split_plan(a);
  dispatch(dt, a.hn, drops(a), [&](auto t, auto dd, auto drop) {
    using T = typename decltype(t)::type;
    constexpr int D = decltype(dd)::value;
    constexpr bool DROP = decltype(drop)::value;
    if (p.splits > 0) {
      if constexpr (!DROP) {
        const int64_t probs = (int64_t)a.b * a.ng * p.rtiles;
        hipLaunchKernelGGL((k_ga_split<T, D>), dim3((unsigned)(probs * p.splits)), dim3(64 * kSplitWaves), 0, st, a,
                           p.rtiles, p.splits, p.chunk, p.kbeg, ws);
        auto join = [&](auto gr) {
          constexpr int GR = decltype(gr)::value, RPB = kThreads / (D / 4 * GR);
          hipLaunchKernelGGL((k_ga_join<T, D, GR>), dim3((unsigned)((probs * 32 + RPB - 1) / RPB)), dim3(kThreads), 0,
                             st, a, p.rtiles, p.splits, ws);
        };
        if (p.splits > kJoinSerial) join(std::integral_constant<int, kThreads / (D / 4)>{});
        else if (p.splits > 1) join(std::integral_constant<int, 1>{});
      }
    } else {
      const int nx = (a.sq + kTileQ - 1) / kTileQ;
      hipLaunchKernelGGL((k_ga_fwd<T, D, DROP>), dim3((unsigned)((int64_t)nx * a.b * a.np)), dim3(kThreads), 0, st, a,
                         nx, keep_thresh(a), keep_scale(a));
    }
  });
  check_launch("ga_forward");
}

int64_t ga_backward_workspace(const GaArgs& a) {
  const int n = dkdv_splits(a);
  return n > 1 ? (int64_t)n * a.b * a.ng * a.sk * 2 * (a.hn <= 64 ? 64 : 128) : 0;
}

void ga_backward(int dt, const GaArgs& a, float* ws, hipStream_t st) {
  const int nq = (a.sq + kTileQ - 1) / kTileQ, nkt = (a.sk + kTileQ - 1) / kTileQ, splits = dkdv_splits(a);
  dispatch(dt, a.hn, drops(a), [&](auto t, auto dd, auto drop) {
    using T = typename decltype(t)::type;
    constexpr int D = decltype(dd)::value;
    constexpr bool DROP = decltype(drop)::value;
    hipLaunchKernelGGL((k_ga_dq<T, D, DROP>), dim3((unsigned)((int64_t)nq * a.b * a.np)), dim3(kThreads), 0, st, a, nq,
                       keep_thresh(a), keep_scale(a));
    if (!a.dk.p) return;
    hipLaunchKernelGGL((k_ga_dkdv<T, D, DROP>), dim3((unsigned)((int64_t)nkt * a.b * a.ng * splits)), dim3(kThreads), 0,
                       st, a, nkt, splits, keep_thresh(a), keep_scale(a), ws);
    if (splits > 1) {
      const int64_t n = (int64_t)a.b * a.ng * a.sk * (2 * D / 4);
      hipLaunchKernelGGL((k_ga_dkdv_join<T, D>), dim3((unsigned)((n + kThreads - 1) / kThreads)), dim3(kThreads), 0, st,
                         a, splits, ws);
    }
  });
  check_launch("ga_backward");
}

}  // namespace bh
