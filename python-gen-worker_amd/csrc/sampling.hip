// Drawing the next tokens from a step's logits: temperature, top-k, top-p, min-p, one given random number a row.
#include <type_traits>

#include "gwa_common.h"

namespace {

constexpr int SM_BINS = 384, SM_DIGITS = 2048, SM_FOUND = 8192;
constexpr int SM_HELD = 8;            // logits a thread holds where a row fits a workgroup's registers
constexpr int SM_PART = 4096, SM_PARTS = 64;  // tokens a part of a longer row at least; parts of a row at most
constexpr int SM_AHEAD = 4;           // 16-byte loads a lane has in flight
constexpr int SM_FEW = 256;           // collected tokens that are ranked all against all
// Measured, bf16 logits: 64 rows of 131072, a top_k of 50: 27 us with SM_FEW at 256, 35 where none are ranked so; up to 512 at
// 512 the squares cost more than sorting does (rows of 300 to 470 collected tokens: 61 against 51).
constexpr int kTableBits = 9;         // of the table of 2^(j / 512)

struct SampleArgs {
  const void* logits;
  int64_t ld;
  const float* uniform;
  gwa_sampling s;
  int64_t* tokens;
  float* logprobs;
  int vocab, shift;   // weights are integers of 2^-shift
  int parts, part;    // of a row, and the tokens of one
  uint64_t* bins;     // [rows][parts][SM_BINS]: a part's tokens (of rows with a top_k) or their weight, up to and with each bin
  float* most;        // [rows][parts]
};

// fp32 values as integers of the same order: -0 counts as 0, NaN below everything
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int DT>
struct Logits;
template <>
struct Logits<GWA_DT_F32> {
  static constexpr int kBytes = 4, kVec = 4;
  static __device__ __forceinline__ float at(const void* p, int64_t i) { return ((const float*)p)[i]; }
  static __device__ __forceinline__ float of(const v4i& w, int e) { return __int_as_float(w[e]); }
};
template <>
struct Logits<GWA_DT_BF16> {
  static constexpr int kBytes = 2, kVec = 8;
  static __device__ __forceinline__ float at(const void* p, int64_t i) { return bf16_to_f32(((const uint16_t*)p)[i]); }
  static __device__ __forceinline__ float of(const v4i& w, int e) {
    return e & 1 ? bf16_hi((uint32_t)w[e / 2]) : bf16_lo((uint32_t)w[e / 2]);
  }
};
template <>
struct Logits<GWA_DT_F16> {
  static constexpr int kBytes = 2, kVec = 8;
  static __device__ __forceinline__ float at(const void* p, int64_t i) { return f16_bits_to_f32(((const uint16_t*)p)[i]); }
  static __device__ __forceinline__ float of(const v4i& w, int e) {
    return f16_bits_to_f32((uint16_t)((uint32_t)w[e / 2] >> (e & 1 ? 16 : 0)));
  }
};

// 2^(j / 16) and 2^(j / 512), rounded to nearest
__device__ const double kPowers16[16] = {
    0x1.0000000000000p+0, 0x1.0b5586cf9890fp+0, 0x1.172b83c7d517bp+0, 0x1.2387a6e756238p+0,
    0x1.306fe0a31b715p+0, 0x1.3dea64c123422p+0, 0x1.4bfdad5362a27p+0, 0x1.5ab07dd485429p+0,
    0x1.6a09e667f3bcdp+0, 0x1.7a11473eb0187p+0, 0x1.8ace5422aa0dbp+0, 0x1.9c49182a3f090p+0,
    0x1.ae89f995ad3adp+0, 0x1.c199bdd85529cp+0, 0x1.d5818dcfba487p+0, 0x1.ea4afa2a490dap+0};
__device__ const double kPowers512[32] = {
    0x1.0000000000000p+0, 0x1.0058c86da1c0ap+0, 0x1.00b1afa5abcbfp+0, 0x1.010ab5b2cbd11p+0,
    0x1.0163da9fb3335p+0, 0x1.01bd1e77170b4p+0, 0x1.02168143b0281p+0, 0x1.027003103b10ep+0,
    0x1.02c9a3e778061p+0, 0x1.032363d42b027p+0, 0x1.037d42e11bbccp+0, 0x1.03d7411915a8ap+0,
    0x1.04315e86e7f85p+0, 0x1.048b9b35659d8p+0, 0x1.04e5f72f654b1p+0, 0x1.0540727fc1762p+0,
    0x1.059b0d3158574p+0, 0x1.05f5c74f0bec2p+0, 0x1.0650a0e3c1f89p+0, 0x1.06ab99fa6407cp+0,
    0x1.0706b29ddf6dep+0, 0x1.0761ead925493p+0, 0x1.07bd42b72a836p+0, 0x1.0818ba42e7d30p+0,
    0x1.0874518759bc8p+0, 0x1.08d0088f8093fp+0, 0x1.092bdf66607e0p+0, 0x1.0987d61701716p+0,
    0x1.09e3ecac6f383p+0, 0x1.0a402331b9715p+0, 0x1.0a9c79b1f3919p+0, 0x1.0af8f03834e52p+0};
// 2^shift 2^(j / 512)
__device__ __forceinline__ void fill_table(double* table, int shift) {
  for (int i = threadIdx.x; i < (1 << kTableBits); i += blockDim.x)
    table[i] = __builtin_amdgcn_ldexp(kPowers16[i >> 5] * kPowers512[i & 31], shift);
}

// A row's tokens by their weight exp((x - m) / temperature) = 2^y, y = (x - m) log2(e) / temperature in 64 bits. The weight
// is an integer of 2^-shift: 2^y = 2^n 2^(j/512) 2^r, |r| <= 1/1024, by a table (which holds the 2^shift) and the series of
// 2^r to r^3 (the rest is below 2^-46), rounded by an addition of 2^52. Bins are an eighth of a unit of y wide; the last is
// for what weighs nothing: y < -47, -inf and NaN. Bins, and the SM_BINS parts of one (`inside`), fall as x grows, never the other
// way. A token's weight and bin have to be the same wherever they are formed, so the compiler may not choose where products and
// sums are fused.
// m = +inf is held as 1e300: +inf is then at y = 0, all else far below.
struct Scale {
  double c, m;
  const double* table;
  double c3, c2, c1;  // of the series, ln(2)^i / i!
  static constexpr double kMagic = 6755399441055744.0 / (1 << kTableBits);  // 1.5 * 2^52: its last bit is 1 / 512
  static constexpr int kPerBin = 6;  // log2 of the 1 / 512 in a bin
  __device__ __forceinline__ bool weighs(float x, double& y) const {
#pragma clang fp contract(off)
    y = ((double)x - m) * c;
    return y >= -47.0;
  }
  static __device__ __forceinline__ int steps_of(double& y, double& r) {
#pragma clang fp contract(off)
    y = fmin(y, 0.0);
    const double t = y + kMagic;
    r = y - (t - kMagic);
    return (int)(uint32_t)__builtin_bit_cast(uint64_t, t);
  }
  __device__ __forceinline__ uint64_t of_steps(int k, double r) const {
#pragma clang fp contract(off)
    double p = __builtin_fma(c3, r, c2);
    p = __builtin_fma(p, r, c1);
    p = __builtin_fma(p, r, 1.0);
    // times 2^(k >> 9), in the exponent: the product lies in 2^shift [0.99, 2), n is -48 at least and shift 38
    const uint64_t u = __builtin_bit_cast(uint64_t, p * table[k & ((1 << kTableBits) - 1)]);
    const uint32_t hi = (uint32_t)(u >> 32) + ((uint32_t)(k & ~((1 << kTableBits) - 1)) << (20 - kTableBits));
    p = __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)u);
    return __builtin_bit_cast(uint64_t, p + 4503599627370496.0) & 0xfffffffffffffull;
  }
  static __device__ __forceinline__ int bin_of_steps(int k) { return -k >> kPerBin; }
  __device__ __forceinline__ uint64_t weight(float x, int& bin) const {
    double y, r;
    bin = SM_BINS - 1;
    if (!weighs(x, y)) return 0;
    const int k = steps_of(y, r);
    bin = bin_of_steps(k);
    return of_steps(k, r);
  }
  __device__ __forceinline__ uint64_t weight(float x) const {
    int bin;
    return weight(x, bin);
  }
  __device__ __forceinline__ int bin(float x) const {
    double y, r;
    return weighs(x, y) ? bin_of_steps(steps_of(y, r)) : SM_BINS - 1;
  }
  // a bin's tokens once more into SM_BINS: by how far -8 y lies past the bin's start, bin - 1 / 128
  __device__ __forceinline__ int inside(float x, int bin) const {
#pragma clang fp contract(off)
    double y;
    if (!weighs(x, y)) return SM_BINS - 1;
    const double f = (fmin(y, 0.0) * -8.0 - ((double)bin - 0.0078125)) * (double)SM_BINS;
    return min(max((int)f, 0), SM_BINS - 1);
  }
  // a range of logits that holds all of bins from to .. (and some more), in fp32
  __device__ __forceinline__ void range(int from, int to, float& lo, float& hi) const {
    const double a = m - ((double)(to + 1) * 0.125 + 0.01) / c, b = m - ((double)from * 0.125 - 0.02) / c;
    lo = (float)(a - fabs(a) * 1e-6 - 1e-37);
    hi = from == 0 ? INFINITY : (float)(b + fabs(b) * 1e-6 + 1e-37);
  }
};

// A token's weight and bin: as they were formed, or to be formed
struct Formed {
  uint64_t w;
  int b;
  __device__ __forceinline__ uint64_t weight() const { return w; }
  __device__ __forceinline__ int bin() const { return b; }
};
struct Unformed {
  const Scale& scale;
  float x;
  __device__ __forceinline__ uint64_t weight() const { return scale.weight(x); }
  __device__ __forceinline__ int bin() const { return scale.bin(x); }
};

__device__ __forceinline__ uint64_t two_words(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }
// lane `lane`'s x (the same lane for the wave)
__device__ __forceinline__ uint64_t lane64(uint64_t x, int lane) {
  return two_words((uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane),
                   (uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane));
}
// x of another lane by a data-parallel move, 0 where there is none
template <int MOVE, int ROWS>
__device__ __forceinline__ uint64_t moved64(uint64_t x) {
  return two_words((uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, MOVE, ROWS, 0xf, false),
                   (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(x >> 32), MOVE, ROWS, 0xf, false));
}
// Sums up to and with each lane: within rows of 16 lanes (shifts by 1, 2, 4, 8), then over the wave (lane 15 of a row to the
// next, lane 31 to the upper half). All lanes take part.
__device__ __forceinline__ uint64_t row_scan64(uint64_t x) {
  x += moved64<0x111, 0xf>(x);
  x += moved64<0x112, 0xf>(x);
  x += moved64<0x114, 0xf>(x);
  x += moved64<0x118, 0xf>(x);
  return x;
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t x) {
  x = row_scan64(x);
  x += moved64<0x142, 0xa>(x);
  x += moved64<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t x) { return lane64(wave_scan64(x), 63); }

// x of lane ^ X
template <int X>
__device__ __forceinline__ uint32_t beside32(uint32_t x) {
  if constexpr (X == 4) return beside32<3>(beside32<7>(x));
  else if constexpr (X >= 16) return (uint32_t)__shfl_xor((int)x, X);
  else {
    // within fours; eights and sixteens mirrored; sixteens turned by 8
    constexpr int kMove = X == 1 ? 0xb1 : X == 2 ? 0x4e : X == 3 ? 0x1b : X == 7 ? 0x141 : X == 15 ? 0x140 : 0x128;
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kMove, 0xf, 0xf, true);
  }
}
// A step of sorting: the larger of a pair to the lower place, the one without the bit LOW
template <int X, int LOW>
__device__ __forceinline__ uint32_t stepped32(uint32_t x) {
  const uint32_t o = beside32<X>(x);
  return threadIdx.x & LOW ? min(x, o) : max(x, o);
}
template <int S>
__device__ __forceinline__ uint32_t settled32(uint32_t x) {
  x = stepped32<S, S>(x);
  if constexpr (S > 1) x = settled32<S / 2>(x);
  return x;
}
// Falling over the first 2^bits threads of a workgroup of NT (bits at least 6; all threads call it, with 0 behind what is
// sorted): runs of twice the length from two, the one against the other reversed, then halved; between waves by LDS, two
// buffers in turn, so that one barrier a step is enough. cells[1] may hold the threads' own values.
template <int NT>
__device__ __forceinline__ uint32_t sorted32(uint32_t x, int bits, uint32_t (&cells)[2][NT]) {
  const int tid = threadIdx.x;
  const bool in = tid < 1 << bits;  // the same for the wave
  if (in) {
    x = stepped32<1, 1>(x);
    x = settled32<1>(stepped32<3, 2>(x));
    x = settled32<2>(stepped32<7, 4>(x));
    x = settled32<4>(stepped32<15, 8>(x));
    x = settled32<8>(stepped32<31, 16>(x));
    x = settled32<16>(stepped32<63, 32>(x));
  }
  int turn = 0;
  for (int size = 128; size <= 1 << bits; size *= 2) {
    for (int low = size / 2, other = size - 1; low >= 64; other = low /= 2) {
      if (in) cells[turn][tid] = x;
      __syncthreads();
      if (in) {
        const uint32_t o = cells[turn][tid ^ other];
        x = tid & low ? min(x, o) : max(x, o);
      }
      turn ^= 1;
    }
    if (in) x = settled32<32>(x);
  }
  return x;
}

// Below this a min_p keeps all: there weights of a few units of 2^-shift (38 at least) would be compared, whose rounding
// tells the least kept one apart from its neighbours no better than a bin does.
constexpr float kLeastMinP = 0x1p-28f;

// One row's settings and how its cuts are found: kCount: the first top_k by the numbers of tokens in the bins; kMass: what
// there are of top_p and min_p by the weights in them; kWhole: by passes over the whole row. 64 rows of 131072 by kCount: 34 us
// for a top_k of 200 and 46 for 4000; by kWhole 73 and 101. Past half of SM_FOUND a wave's own part of the collected tokens
// would often be too short.
enum Way { kGreedy, kCount, kMass, kWhole };
struct Settings {
  float temperature, top_p, min_p, uniform;
  int top_k;  // 0: all
  Way way;
};
__device__ __forceinline__ float held_in(float x, float lo, float hi) { return fminf(fmaxf(x, lo), hi); }
__device__ __forceinline__ Settings settings_of(const SampleArgs& a, int64_t row) {
  Settings s;
  s.temperature = a.s.temperature ? a.s.temperature[row] : a.s.all_temperature;
  if (s.temperature > 3.0e38f) s.temperature = 3.0e38f;  // (not a NaN)
  s.top_k = a.s.top_k ? a.s.top_k[row] : a.s.all_top_k;
  s.top_p = held_in(a.s.top_p ? a.s.top_p[row] : a.s.all_top_p, 0.0f, 1.0f);
  s.min_p = held_in(a.s.min_p ? a.s.min_p[row] : a.s.all_min_p, 0.0f, 1.0f);
  s.uniform = held_in(a.uniform[row], 0.0f, 1.0f);
  if (s.top_k <= 0 || s.top_k >= a.vocab) s.top_k = 0;
  if (s.min_p < kLeastMinP) s.min_p = 0.0f;
  s.way = !(s.temperature > 0.0f) ? kGreedy : s.top_k == 0 ? kMass : s.top_k <= SM_FOUND / 2 ? kCount : kWhole;
  return s;
}

__device__ __forceinline__ Scale scale_of(const SampleArgs& a, const Settings& s, float m, const double* table) {
  double c3 = 5.5504108664821580e-2, c2 = 2.4022650695910072e-1, c1 = 6.9314718055994531e-1;
  asm("" : "+v"(c3), "+v"(c2), "+v"(c1));  // in registers: as constants they are moved for every weight (1.6 us of 37.5)
  return {1.4426950408889634 / (double)s.temperature, m == INFINITY ? 1e300 : (double)m, table, c3, c2, c1};
}

// f(N, index of the first, N neighbouring logits) over tokens [lo, hi) of the row at base, by threads `id` of n, in 16-byte
// pieces where they are whole
template <int DT, class F>
__device__ __forceinline__ void each_vector(const uint8_t* base, int lo, int hi, int id, int n, F f) {
  using L = Logits<DT>;
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, L::kVec> many;
  const uint8_t* p = base + (int64_t)lo * L::kBytes;
  const int head = min((int)((16 - ((uintptr_t)p & 15)) & 15) / L::kBytes, hi - lo);
  if (id < head) {
    const float x[1] = {L::at(p, id)};
    f(one, lo + id, x);
  }
  const int v0 = lo + head, vecs = (hi - v0) / L::kVec;
  const v4i* body = (const v4i*)(base + (int64_t)v0 * L::kBytes);
  for (int v = id; v < vecs; v += n * SM_AHEAD) {
    v4i w[SM_AHEAD];
#pragma unroll
    for (int u = 0; u < SM_AHEAD; ++u) w[u] = body[min(v + n * u, vecs - 1)];
#pragma unroll
    for (int u = 0; u < SM_AHEAD; ++u)
      if (v + n * u < vecs) {
        float x[L::kVec];
#pragma unroll
        for (int e = 0; e < L::kVec; ++e) x[e] = L::of(w[u], e);
        f(many, v0 + (v + n * u) * L::kVec, x);
      }
  }
  const int tail = v0 + vecs * L::kVec + id;
  if (tail < hi) {
    const float x[1] = {L::at(base, tail)};
    f(one, tail, x);
  }
}

// the same with f(index, logit)
template <int DT, class F>
__device__ __forceinline__ void each_token(const uint8_t* base, int lo, int hi, int id, int n, F f) {
  each_vector<DT>(base, lo, hi, id, n, [&](auto n_c, int i, const float (&x)[decltype(n_c)::value]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < decltype(n_c)::value; ++e) f(i + e, x[e]);
  });
}

// What a cut keeps: the tokens ordered above `key`, and of those equal to it the first `ties` by index. `equal`: how many
// those are.
struct Cut {
  uint32_t key, ties, equal;
};

// A workgroup of NW waves on one row
template <int NW>
struct Drawer {
  static constexpr int NT = 64 * NW;
  struct Lds {
    double table[1 << kTableBits];
    uint64_t mass[SM_DIGITS];
    uint32_t count[SM_DIGITS];
    uint32_t list[2][NT];
    uint64_t cells[2][NW];
    uint64_t found[4];
    uint32_t n;
  };
  Lds& l;
  const SampleArgs& a;
  const Settings& s;
  int64_t row;
  Scale scale;
  float m;
  double low;  // the least weight that min_p keeps

  __device__ __forceinline__ Drawer(Lds& l, const SampleArgs& a, const Settings& s, int64_t row, float m)
      : l(l), a(a), s(s), row(row), scale(scale_of(a, s, m, l.table)), m(m),
        low((double)s.min_p * (double)(1ull << a.shift)) {}
  __device__ __forceinline__ uint64_t weight(float x) const { return scale.weight(x); }

  // The sum of x over the threads before this one, in the threads' order, and over all
  __device__ __forceinline__ void scan(uint64_t x, uint64_t& before, uint64_t& all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t p = wave_scan64(x);
    __syncthreads();
    if (lane == 63) l.cells[0][wave] = p;
    __syncthreads();
    // the waves' sums, one a lane (16 at most)
    const uint64_t c = lane < NW ? l.cells[0][lane] : 0, upto = row_scan64(c);
    before = p - x + lane64(upto - c, wave), all = lane64(upto, NW - 1);
  }
  // Sums of x and y over the threads before this one, in the threads' order, and over all
  __device__ __forceinline__ void scan(uint64_t x, uint64_t y, uint64_t& x_before, uint64_t& y_before, uint64_t& x_all,
                                       uint64_t& y_all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t p = wave_scan64(x), q = wave_scan64(y);
    __syncthreads();
    if (lane == 63) l.cells[0][wave] = p, l.cells[1][wave] = q;
    __syncthreads();
    const uint64_t cx = lane < NW ? l.cells[0][lane] : 0, cy = lane < NW ? l.cells[1][lane] : 0;
    const uint64_t sx = row_scan64(cx), sy = row_scan64(cy);
    x_before = p - x + lane64(sx - cx, wave), y_before = q - y + lane64(sy - cy, wave);
    x_all = lane64(sx, NW - 1), y_all = lane64(sy, NW - 1);
  }

  // Where a sum over bins of counts n and weights w (SM_BINS / NT bins or fewer a thread, from bin `first` on) reaches what
  // is wanted: MASS: the weight `target`, else the number `want`, both counted from n0, w0 on
  struct Place {
    int bin;
    uint32_t inside;
    uint64_t before, above;  // tokens, or weight, ahead of it
  };
  template <bool MASS, int PER, class Target>
  __device__ __forceinline__ Place reach(const uint64_t (&n)[PER], const uint64_t (&w)[PER], int first, uint64_t n0,
                                         uint64_t w0, uint64_t want, Target target_of) {
    uint64_t sum = 0, upto, all;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += MASS ? w[i] : n[i];
    scan(sum, upto, all);
    upto += MASS ? w0 : n0;
    const double target = MASS ? target_of(all) : 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint64_t before = upto;
      upto += MASS ? w[i] : n[i];
      if (MASS ? (double)before < target && (double)upto >= target : before < want && upto >= want)
        l.found[0] = first + i, l.found[1] = before, l.found[2] = n[i];
    }
    __syncthreads();
    const uint64_t before = l.found[1];
    const Place p = {(int)l.found[0], (uint32_t)l.found[2], MASS ? 0 : before, MASS ? before : 0};
    __syncthreads();
    return p;
  }

  // the ties that are kept of `equal` weights w each behind a weight of `from`: as few as reach the target
  static __device__ __forceinline__ uint32_t ties_to(double target, uint64_t from, uint64_t w, uint32_t equal) {
    uint32_t e = w ? (uint32_t)fmin(fmax(ceil((target - (double)from) / (double)w), 1.0), (double)equal) : 1;
    while (e > 1 && (double)(from + (e - 1) * w) >= target) --e;
    while (e < equal && (double)(from + e * w) < target) ++e;
    return e;
  }

  // a histogram by bin_of of the tokens that `each` passes on (their index, logit, and weight and bin) and `take` accepts,
  // and the place in it
  static constexpr int kPer = (SM_BINS + NT - 1) / NT;
  template <bool MASS, class Each, class Take, class Of, class Target>
  __device__ __forceinline__ Place locate(Each each, Take take, Of bin_of, uint64_t n0, uint64_t w0, uint64_t want,
                                          Target target_of) {
    __syncthreads();
    for (int i = threadIdx.x; i < SM_BINS; i += NT) l.count[i] = 0, l.mass[i] = 0;
    __syncthreads();
    each([&](int, float x, auto of) __attribute__((always_inline)) {
      if (take(x, of)) {
        const int b = bin_of(x, of);
        atomicAdd(&l.count[b], 1u);
        if (MASS) atomicAdd((unsigned long long*)&l.mass[b], (unsigned long long)of.weight());
      }
    });
    __syncthreads();
    uint64_t n[kPer], w[kPer];
    const int first = kPer * threadIdx.x;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool in = first + i < SM_BINS;
      n[i] = in ? l.count[first + i] : 0, w[i] = in ? l.mass[first + i] : 0;
    }
    return reach<MASS>(n, w, first, n0, w0, want, target_of);
  }

  // The cut inside bin `p.bin` of p.inside tokens (or fewer), from the tokens that `each` passes on and `take` accepts, which
  // hold all of the bin's
  template <bool MASS, class Each, class Take>
  __device__ __forceinline__ Cut resolve(Each each, Take take, Place p, uint64_t want, double target) {
    const int bin = p.bin;
    auto in_bin = [&](float x, auto of) __attribute__((always_inline)) { return take(x, of) && of.bin() == bin; };
    int sub = -1;
    if (p.inside > NT) {  // once more into bins
      p = locate<MASS>(each, in_bin, [&](float x, auto) { return scale.inside(x, bin); }, p.before, p.above, want,
                       [&](uint64_t) { return target; });
      sub = p.bin;
    }
    auto here = [&](float x, auto of) __attribute__((always_inline)) {
      return in_bin(x, of) && (sub < 0 || scale.inside(x, bin) == sub);
    };
    if (p.inside <= NT) {  // sorted, one a thread
      const int tid = threadIdx.x;
      if (tid == 0) l.n = 0;
      __syncthreads();
      each([&](int, float x, auto of) __attribute__((always_inline)) {
        if (here(x, of)) {
          const uint32_t i = atomicAdd(&l.n, 1u);
          if (i < NT) l.list[1][i] = order_of(x);  // (more only of logits that are written meanwhile)
        }
      });
      __syncthreads();
      const int n = min((int)l.n, NT);
      const uint32_t key = sorted32<NT>(tid < n ? l.list[1][tid] : 0, n <= 64 ? 6 : 32 - __clz(n - 1), l.list);
      const uint64_t w = MASS && tid < n ? weight(value_of(key)) : 0;
      uint64_t before = 0, all;
      if (MASS) scan(w, before, all);
      else __syncthreads();
      if (tid < n) l.list[0][tid] = key;
      __syncthreads();
      before += p.above;
      if (tid < n && (MASS ? (double)before < target && (double)(before + w) >= target : p.before + tid + 1 == want))
        l.found[0] = key, l.found[1] = tid;
      __syncthreads();
      // the first place of that value, and the one behind its last
      const uint32_t at = (uint32_t)l.found[0], place = (uint32_t)l.found[1];
      if (tid < n && key == at) {
        if (tid == 0 || l.list[0][tid - 1] != at) l.found[2] = tid;
        if (tid == n - 1 || l.list[0][tid + 1] != at) l.found[3] = tid + 1;
      }
      __syncthreads();
      const uint32_t first = (uint32_t)l.found[2], behind = (uint32_t)l.found[3];
      __syncthreads();
      return {at, place + 1 - first, behind - first};
    }
    // digit by digit of the ordered values: 11 + 11 + 10 bits
    uint32_t prefix = 0;
    int shift = 21;
    uint64_t digit_w = 0;
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass == 2 ? 10 : 11;
      for (int i = threadIdx.x; i < SM_DIGITS; i += NT) l.count[i] = 0, l.mass[i] = 0;
      __syncthreads();
      each([&](int, float x, auto of) __attribute__((always_inline)) {
        const uint32_t key = order_of(x);
        if (here(x, of) && (pass == 0 || key >> (shift + bits) == prefix)) {
          const uint32_t d = SM_DIGITS - 1 - (key >> shift & ((1u << bits) - 1));  // falling
          atomicAdd(&l.count[d], 1u);
          if (MASS) atomicAdd((unsigned long long*)&l.mass[d], (unsigned long long)of.weight());
        }
      });
      __syncthreads();
      constexpr int PER = SM_DIGITS / NT;
      uint64_t n[PER], w[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) n[i] = l.count[PER * threadIdx.x + i], w[i] = l.mass[PER * threadIdx.x + i];
      p = reach<MASS>(n, w, PER * threadIdx.x, p.before, p.above, want, [&](uint64_t) { return target; });
      digit_w = l.mass[p.bin];
      prefix = prefix << bits | (uint32_t)(SM_DIGITS - 1 - p.bin);
      shift = pass == 0 ? 10 : 0;
      __syncthreads();
    }
    const uint32_t equal = min(max(p.inside, 1u), (uint32_t)a.vocab);
    return {prefix, MASS ? ties_to(target, p.above, digit_w / equal, equal) : (uint32_t)(want - p.before), equal};
  }

  static __device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
  }
  __device__ __forceinline__ double target_of(uint64_t all) const {
    return fmax((double)s.top_p * (double)all, 0.5);  // the first token reaches 0.5 alone
  }

  // top_k's cut among the tokens of `each`
  template <class Each>
  __device__ __forceinline__ Cut cut_by_count(Each each) {
    auto any = [](float, auto) { return true; };
    const Place p = locate<false>(each, any, [&](float, auto of) { return of.bin(); }, 0, 0, (uint64_t)s.top_k,
                                  [](uint64_t) { return 0.0; });
    return resolve<false>(each, any, p, (uint64_t)s.top_k, 0.0);
  }
  // top_p's among those that `top` (of top_k, or of all) keeps
  template <class Each>
  __device__ __forceinline__ Cut cut_by_mass(Each each, const Cut& top) {
    auto take = [&](float x, auto) __attribute__((always_inline)) { return order_of(x) >= top.key; };
    const uint32_t dropped = top.equal - top.ties;
    const uint64_t off = dropped ? dropped * weight(value_of(top.key)) : 0;
    double target = 0.0;
    const Place p = locate<true>(each, take, [&](float, auto of) { return of.bin(); }, 0, 0, 0,
                                 [&](uint64_t all) { return target = target_of(all - off); });
    return resolve<true>(each, take, p, 0, target);
  }

  __device__ __forceinline__ uint64_t kept(uint64_t w) const { return (double)w >= low ? w : 0; }
  __device__ __forceinline__ uint64_t tie_weight(const Cut& cut) const { return cut.key ? kept(weight(value_of(cut.key))) : 0; }
  static __device__ __forceinline__ uint64_t ties_in(const Cut& cut, uint64_t before, uint64_t n) {  // kept, of n behind `before`
    return before >= cut.ties ? 0 : min(n, (uint64_t)cut.ties - before);
  }
  // cum > u total: for integers, cum > floor(u total)
  __device__ __forceinline__ uint64_t drawn(uint64_t total) const {
    return min((uint64_t)((double)s.uniform * (double)total), total - 1);
  }

  __device__ __forceinline__ void draw(int index, float x, uint64_t total) const {
    a.tokens[row] = index;
    const double y = x == m ? 0.0 : ((double)x - (double)m) / (double)s.temperature;
    a.logprobs[row] = (float)(y - log((double)total / (double)(1ull << a.shift)));
  }
  // The token at which the kept weights, `cum` of them and `upto` ties before this thread's tokens, pass r: one of its n
  // neighbouring ones from `index` on
  template <int N>
  __device__ __forceinline__ void pick(const Cut& cut, uint64_t tie_w, uint64_t cum, uint64_t upto, uint64_t r, uint64_t total,
                                       int index, int n, const float (&x)[N], const uint64_t (&w)[N]) const {
    int at = -1;
    float x_at = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t key = order_of(x[i]);
      if (i < n && key > cut.key) cum += kept(w[i]);
      else if (i < n && key == cut.key) cum += upto++ < cut.ties ? tie_w : 0;
      if (at < 0 && cum > r) at = i, x_at = x[i];
    }
    draw(index + at, x_at, total);
  }
};

__device__ __forceinline__ const uint8_t* row_at(const SampleArgs& a, int64_t row, int bytes) {
  return (const uint8_t*)a.logits + row * a.ld * bytes;
}
// n of N neighbouring logits from i0 on, NaN behind them
template <int DT, int N>
__device__ __forceinline__ void run_of(const uint8_t* base, int i0, int n, float (&x)[N]) {
  using L = Logits<DT>;
  const uint8_t* at = base + (int64_t)i0 * L::kBytes;
  if (N % L::kVec == 0 && n == N && ((uintptr_t)at & 15) == 0) {
#pragma unroll
    for (int v = 0; v < N / L::kVec; ++v) {
      const v4i w = ((const v4i*)at)[v];
#pragma unroll
      for (int e = 0; e < L::kVec; ++e) x[v * L::kVec + e] = L::of(w, e);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i < n ? L::at(at, i) : NAN;
  }
}
__device__ __forceinline__ float wave_max(float m) {
#pragma unroll
  for (int w = 32; w; w >>= 1) m = fmaxf(m, __shfl_xor(m, w));
  return m;
}

// Rows that fit a workgroup's registers: SM_HELD neighbouring tokens a thread, read once. Bound by its chain of barriers and
// scans: one row of 2048 with a top_p 8.8 us, 1024 such rows 20. With 16 waves for such rows as well, 41 (one of them with a
// top_k too: 13 where four waves take 11.5); rows of 8192 by the three kernels below: 64 of them 20 us instead of 15, 1024 62 instead of 55.
template <int DT, int NW>
__global__ __launch_bounds__(64 * NW) void sample_held_kernel(SampleArgs a) {
  using D = Drawer<NW>;
  using L = Logits<DT>;
  __shared__ typename D::Lds l;
  __shared__ uint32_t least;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const uint8_t* base = row_at(a, row, L::kBytes);
  const Settings s = settings_of(a, row);
  const int i0 = SM_HELD * tid, n = min(max(a.vocab - i0, 0), SM_HELD);
  float x[SM_HELD];
  run_of<DT>(base, i0, n, x);
  fill_table(l.table, a.shift);
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < SM_HELD; ++i) m = fmaxf(m, x[i]);
  m = wave_max(m);
  if (lane == 0) l.cells[0][wave] = __float_as_uint(m);
  if (tid == 0) least = 0xffffffffu;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) m = fmaxf(m, __uint_as_float((uint32_t)l.cells[0][i]));
  if (m == -INFINITY) {
    if (tid == 0) a.tokens[row] = -1, a.logprobs[row] = NAN;
    return;
  }
  if (s.way == kGreedy) {
    uint32_t first = 0xffffffffu;
#pragma unroll
    for (int i = SM_HELD - 1; i >= 0; --i) first = x[i] == m ? (uint32_t)(i0 + i) : first;
    if (first != 0xffffffffu) atomicMin(&least, first);
    __syncthreads();
    if (tid == 0) a.tokens[row] = least, a.logprobs[row] = 0.0f;
    return;
  }
  D d(l, a, s, row, m);
  uint64_t w[SM_HELD];
  int bin[SM_HELD];
#pragma unroll
  for (int i = 0; i < SM_HELD; ++i) w[i] = d.scale.weight(x[i], bin[i]);
  auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < SM_HELD; ++i)
      if (i < n) f(i0 + i, x[i], Formed{w[i], bin[i]});
  };
  Cut cut = {0, (uint32_t)a.vocab, (uint32_t)a.vocab};
  if (s.top_k) cut = d.cut_by_count(each);
  if (s.top_p < 1.0f) cut = d.cut_by_mass(each, cut);
  const uint64_t tie_w = d.tie_weight(cut);
  uint64_t sum = 0, ties = 0, sum_before, ties_before, sum_all, ties_all;
  each([&](int, float x, auto of) __attribute__((always_inline)) {
    const uint32_t key = order_of(x);
    if (key > cut.key) sum += d.kept(of.weight());
    ties += key == cut.key;
  });
  d.scan(sum, ties, sum_before, ties_before, sum_all, ties_all);
  const uint64_t total = sum_all + D::ties_in(cut, 0, ties_all) * tie_w, r = d.drawn(total);
  const uint64_t cum = sum_before + D::ties_in(cut, 0, ties_before) * tie_w;
  if (cum <= r && cum + sum + D::ties_in(cut, ties_before, ties) * tie_w > r) {
    d.pick(cut, tie_w, cum, ties_before, r, total, i0, n, x, w);
  }
}

// Longer rows, first: the largest logit of every part. Bound by memory: 256 rows of 131072, fp32: 23 us, 5.8 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void sample_max_kernel(SampleArgs a) {
  __shared__ float cells[4];
  const int64_t row = blockIdx.x / a.parts;
  const int g = blockIdx.x - (int)row * a.parts, lo = g * a.part, hi = min(lo + a.part, a.vocab);
  float m = -INFINITY;
  each_token<DT>(row_at(a, row, Logits<DT>::kBytes), lo, hi, threadIdx.x, 256,
                 [&](int, float x) __attribute__((always_inline)) { m = fmaxf(m, x); });
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) cells[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) a.most[blockIdx.x] = fmaxf(fmaxf(cells[0], cells[1]), fmaxf(cells[2], cells[3]));
}
__device__ __forceinline__ float row_max(const SampleArgs& a, int64_t row) {
  const int lane = threadIdx.x & 63;
  return wave_max(lane < a.parts ? a.most[row * a.parts + lane] : -INFINITY);  // SM_PARTS at most
}

// second: every part's histogram, of tokens or of their weight, as sums up to each bin. Bound by the weights' arithmetic in
// 64 bits, 31 vector instructions a logit (the logits come from the last-level cache): 256 rows of 131072 35 us, 3.8 TB/s; 64
// of bf16 10 us. All of a load's weights formed ahead of the branches: 35 to 36.5 and 11.
template <int DT>
__global__ __launch_bounds__(256) void sample_bins_kernel(SampleArgs a) {
  __shared__ uint64_t bin[SM_BINS];
  __shared__ double table[1 << kTableBits];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.parts;
  const int g = blockIdx.x - (int)row * a.parts, lo = g * a.part, hi = min(lo + a.part, a.vocab);
  const Settings s = settings_of(a, row);
  if (s.way == kGreedy || s.way == kWhole) return;
  const float m = row_max(a, row);
  if (m == -INFINITY) return;
  fill_table(table, a.shift);
  for (int i = tid; i < SM_BINS; i += 256) bin[i] = 0;
  __syncthreads();
  const Scale scale = scale_of(a, s, m, table);
  const uint8_t* base = row_at(a, row, Logits<DT>::kBytes);
  if (s.way == kCount) {
    each_token<DT>(base, lo, hi, tid, 256, [&](int, float x) __attribute__((always_inline)) {
      double y, r;
      if (scale.weighs(x, y)) atomicAdd((uint32_t*)&bin[Scale::bin_of_steps(Scale::steps_of(y, r))], 1u);
    });
  } else {
    each_token<DT>(base, lo, hi, tid, 256, [&](int, float x) __attribute__((always_inline)) {
      double y, r;
      if (scale.weighs(x, y)) {
        const int k = Scale::steps_of(y, r);
        atomicAdd((unsigned long long*)&bin[Scale::bin_of_steps(k)], (unsigned long long)scale.of_steps(k, r));
      }
    });
  }
  __syncthreads();
  if (tid < 64) {
    constexpr int PER = SM_BINS / 64;
    uint64_t* out = a.bins + (int64_t)blockIdx.x * SM_BINS + PER * tid;
    uint64_t upto[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) upto[i] = sum += bin[PER * tid + i];
    const uint64_t before = wave_scan64(sum) - sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) out[i] = before + upto[i];
  }
}

// third: a workgroup a row. From the parts' histograms the bin that the cut falls into; the tokens that may be kept (kCount)
// or that lie where the cuts fall (kMass) are collected in one pass of comparisons and the cut found among them; the kept
// weight of every part; and the tokens of the part that the random number falls into. Where the collected ones are too
// many (thousands of nearly equal logits, a very large top_k) all is done by passes over the row.
// 256 rows of 131072, fp32, a top_p: 41 us, of which 20 read the row once more (6.7 TB/s), 7 find the cut among some 800
// tokens, 5 the drawn token in its part; 64 rows of bf16, each with settings of its own: 27, the slowest row's. Bound by
// what one workgroup does in turn.
template <int DT>
__global__ __launch_bounds__(1024) void sample_draw_kernel(SampleArgs a) {
  constexpr int NW = 16, NT = 1024;
  using D = Drawer<NW>;
  using L = Logits<DT>;
  __shared__ typename D::Lds l;
  constexpr int SEG = SM_FOUND / NW;  // a wave's own part of the collected tokens
  __shared__ float found_x[SM_FOUND];
  __shared__ int found_i[SM_FOUND];
  __shared__ int found_n[NW];
  __shared__ ulonglong2 few[SM_FEW];  // weight, and order
  __shared__ uint64_t few_sum[2][SM_FEW];
  __shared__ uint32_t few_rank[SM_FEW], few_equal[SM_FEW];
  __shared__ float few_x[SM_FEW];
  __shared__ int few_i[SM_FEW];
  __shared__ uint64_t part_w[SM_PARTS];
  __shared__ uint32_t part_ties[SM_PARTS], least;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const uint8_t* base = row_at(a, row, L::kBytes);
  const Settings s = settings_of(a, row);
  const float m = row_max(a, row);
  if (m == -INFINITY) {
    if (tid == 0) a.tokens[row] = -1, a.logprobs[row] = NAN;
    return;
  }
  if (s.way == kGreedy) {
    // the first part that holds the largest
    const uint64_t with = __ballot(lane < a.parts && a.most[row * a.parts + min(lane, a.parts - 1)] == m);
    const int g = __ffsll((unsigned long long)with) - 1, lo = g * a.part, hi = min(lo + a.part, a.vocab);
    if (tid == 0) least = 0xffffffffu;
    __syncthreads();
    uint32_t first = 0xffffffffu;
    each_token<DT>(base, lo, hi, tid, NT,
                   [&](int i, float x) __attribute__((always_inline)) { first = x == m ? min(first, (uint32_t)i) : first; });
    if (first != 0xffffffffu) atomicMin(&least, first);
    __syncthreads();
    if (tid == 0) a.tokens[row] = least, a.logprobs[row] = 0.0f;
    return;
  }
  fill_table(l.table, a.shift);
  if (tid < SM_PARTS) part_w[tid] = 0, part_ties[tid] = 0;
  D d(l, a, s, row, m);
  const uint64_t* bins = a.bins + row * a.parts * SM_BINS;
  Cut cut = {0, (uint32_t)a.vocab, (uint32_t)a.vocab};
  bool whole = s.way == kWhole;
  int from = 0, to = SM_BINS - 1;  // bins whose tokens are collected
  typename D::Place p = {SM_BINS, 0, 0, 0};
  double target = 0.0;
  uint64_t ahead_of = 0, part_ahead = 0;
  if (!whole) {
    // the row's sums up to each bin: two threads a bin, each half of the parts, joined in LDS
    uint64_t mine = 0;
    const int b = tid & 511;
    if (b < SM_BINS) {
#pragma unroll 8
      for (int g = tid / 512; g < a.parts; g += 2) mine += bins[g * SM_BINS + b];
    }
    if (tid >= 512 && b < SM_BINS) l.mass[b] = mine;
    if (tid == 0) l.found[0] = SM_BINS;
    __syncthreads();
    if (tid < SM_BINS) l.mass[tid] = mine += l.mass[tid];
    __syncthreads();
    const uint64_t before = tid > 0 && tid < SM_BINS ? l.mass[tid - 1] : 0;
    if (s.way == kMass) target = d.target_of(l.mass[SM_BINS - 1]);
    if (tid < SM_BINS && (s.way == kCount ? before < (uint64_t)s.top_k && mine >= (uint64_t)s.top_k
                                          : (double)before < target && (double)mine >= target))
      l.found[0] = tid, l.found[1] = before, l.found[2] = mine - before;
    __syncthreads();
    if (s.way == kCount) {
      // where fewer tokens weigh anything all of them are kept
      p = {(int)l.found[0], (uint32_t)l.found[2], l.found[1], 0};
      to = min(p.bin, SM_BINS - 2);
      whole = p.bin < SM_BINS && p.before + p.inside > SM_FOUND;
    } else {
      from = SM_BINS, to = SM_BINS - 2;  // the last bin's weights are 0
      if (s.top_p < 1.0f) {
        p = {(int)l.found[0], 0, 0, l.found[1]};  // its tokens are counted below
        from = to = p.bin;
      }
      if (s.min_p > 0.0f) {
        // the bin of the least weight that stays (-8 y + 1 / 128 of it; fp32 finds it to 2^-12), and the one beside it where
        // their border is near
        const float at = -log2f(s.min_p) * 8.0f + 0.0078125f;
        from = min(from, (int)fminf(fmaxf(at - 0.01f, 0.0f), (float)SM_BINS));
        to = min(to, (int)fminf(at + 0.01f, (float)SM_BINS));
      }
      // what lies ahead of the collected bins is kept whole: in the row, and in the lane's part
      if (from > 0) {
        ahead_of = l.mass[from - 1];
        if (lane < a.parts) part_ahead = bins[lane * SM_BINS + from - 1];
      }
    }
  }
  float* const my_x = found_x + wave * SEG;
  int* const my_i = found_i + wave * SEG;
  int mine_n = 0;
  if (!whole && from < SM_BINS) {
    // by comparisons in fp32, of a range that holds the bins; then what is not of them goes
    float lo, hi;
    d.scale.range(from, to, lo, hi);
    auto below = [](uint64_t m) __attribute__((always_inline)) {
      return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
    };
    // the lane's N neighbouring tokens from i on
    auto take = [&](auto n_c, int i, const float (&x)[decltype(n_c)::value]) __attribute__((always_inline)) {
      constexpr int N = decltype(n_c)::value;
      uint64_t hits[N], any = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) any |= hits[e] = __ballot(__builtin_amdgcn_fmed3f(x[e], lo, hi) == x[e]);
      if (any == 0) return;
      // the first lane takes part whenever any of its wave does, so its count is the wave's
      int at = __builtin_amdgcn_readfirstlane(mine_n);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (hits[e]) {  // the same for the wave
          const int to = at + below(hits[e]);
          if (__builtin_amdgcn_fmed3f(x[e], lo, hi) == x[e] && to < SEG) my_x[to] = x[e], my_i[to] = i + e;
          at += __popcll(hits[e]);
        }
      mine_n = at;
    };
    each_vector<DT>(base, 0, a.vocab, tid, NT, take);
    mine_n = __shfl(mine_n, 0);
    whole = mine_n > SEG;
    int left = 0;
    for (int i = 0; i < min(mine_n, SEG); i += 64) {
      const bool in = i + lane < min(mine_n, SEG);
      const float x = in ? my_x[i + lane] : NAN;
      const int index = in ? my_i[i + lane] : 0, b = d.scale.bin(x);
      const bool stays = in && b >= from && b <= to;
      const uint64_t those = __ballot(stays);
      if (stays) my_x[left + below(those)] = x, my_i[left + below(those)] = index;
      left += __popcll(those);
    }
    mine_n = left;
  }
  if (lane == 0) found_n[wave] = whole ? -1 : mine_n;
  __syncthreads();
  const int of_wave = found_n[lane & (NW - 1)];
  whole = __ballot(of_wave < 0) != 0;
  int upto_wave = lane < NW ? of_wave : 0;
#pragma unroll
  for (int w = 1; w < NW; w <<= 1) {
    const int u = __shfl_up(upto_wave, w);
    if (lane >= w) upto_wave += u;
  }
  const int n = __shfl(upto_wave, NW - 1), my_first = __shfl(upto_wave, wave) - mine_n;
  const bool cuts = s.way == kCount || p.bin <= to;  // whether what is collected is cut by its order
  if (s.way == kMass) p.inside = (uint32_t)n;
  const bool few_found = !whole && cuts && n <= SM_FEW;
  if (few_found) {
    // each against all, by as many threads a token as there are (four at least). `order`: larger for what comes first (equal
    // logits: the lowest index)
    const int bits = n <= 64 ? 6 : 32 - __clz(n - 1), share = NT >> bits;
    const int j = tid & ((1 << bits) - 1), i0 = tid >> bits;
    const bool mine = tid < n;
    for (int i = lane; i < mine_n; i += 64) few_x[my_first + i] = my_x[i], few_i[my_first + i] = my_i[i];
    if (tid < SM_FEW) few_sum[0][tid] = few_sum[1][tid] = 0, few_rank[tid] = few_equal[tid] = 0;
    __syncthreads();
    uint64_t w = 0, order = 0;
    if (mine) {
      w = d.weight(few_x[tid]);
      order = (uint64_t)order_of(few_x[tid]) << 32 | (uint32_t)~few_i[tid];
      few[tid] = make_ulonglong2(w, order);
    }
    __syncthreads();
    if (j < n) {
      const uint64_t my_order = few[j].y;
      uint64_t ahead = 0;
      uint32_t rank = 0, equal = 0;
#pragma unroll 4
      for (int i = i0; i < n; i += share) {
        const ulonglong2 o = few[i];
        const bool first = o.y > my_order;
        rank += first, ahead += first ? o.x : 0, equal += first && (o.y ^ my_order) >> 32 == 0;
      }
      atomicAdd(&few_rank[j], rank);
      atomicAdd(&few_equal[j], equal);
      atomicAdd((unsigned long long*)&few_sum[0][j], (unsigned long long)ahead);
    }
    __syncthreads();
    const uint32_t rank = mine ? few_rank[tid] : 0, equal = mine ? few_equal[tid] : 0;
    const uint64_t ahead = ahead_of + (mine ? few_sum[0][tid] : 0);
    if (s.way == kCount) {
      const bool among = mine && rank < (uint32_t)s.top_k;
      if (tid < SM_FEW) {
        const uint64_t sum = wave_sum64(among ? w : 0);
        if (lane == 0) l.cells[0][wave] = sum;
      }
      __syncthreads();
      uint64_t all = 0;
#pragma unroll
      for (int i = 0; i < SM_FEW / 64; ++i) all += l.cells[0][i];
      // of the run that reaches top_p of the sum, what lies ahead of a token does not
      const bool stays = among && (s.top_p >= 1.0f || (double)ahead < d.target_of(all)) && (double)w >= d.low;
      if (mine) few[tid].x = stays ? w : 0;
      if (tid < SM_FEW) {
        const uint64_t sum = wave_sum64(stays ? w : 0);
        if (lane == 0) l.cells[1][wave] = sum;
      }
      __syncthreads();
      if (j < n && few[j].x) {
        const uint32_t my_place = (uint32_t)few[j].y;  // larger for lower indices
        uint64_t cum = 0;
#pragma unroll 4
        for (int i = i0; i < n; i += share) {
          const ulonglong2 o = few[i];
          cum += (uint32_t)o.y > my_place ? o.x : 0;
        }
        atomicAdd((unsigned long long*)&few_sum[1][j], (unsigned long long)cum);
      }
      __syncthreads();
      if (stays) {
        uint64_t total = 0;
#pragma unroll
        for (int i = 0; i < SM_FEW / 64; ++i) total += l.cells[1][i];
        const uint64_t r = d.drawn(total), cum = few_sum[1][tid];
        if (cum <= r && cum + w > r) d.draw(few_i[tid], few_x[tid], total);
      }
      return;
    }
    if (mine && (double)ahead < target && (double)(ahead + w) >= target) l.found[0] = order >> 32, l.found[1] = equal + 1;
    __syncthreads();
    cut = {(uint32_t)l.found[0], (uint32_t)l.found[1], (uint32_t)l.found[1]};
  }
  auto each_found = [&](auto f) __attribute__((always_inline)) {
    for (int i = lane; i < mine_n; i += 64) f(my_i[i], my_x[i], Unformed{d.scale, my_x[i]});
  };
  auto each = [&](auto f) __attribute__((always_inline)) {
    each_token<DT>(base, 0, a.vocab, tid, NT,
                   [&](int i, float x) __attribute__((always_inline)) { f(i, x, Unformed{d.scale, x}); });
  };
  if (whole) {
    if (s.top_k) cut = d.cut_by_count(each);
    if (s.top_p < 1.0f) cut = d.cut_by_mass(each, cut);
  } else if (s.way == kCount) {
    auto any = [](float, auto) { return true; };
    if (p.bin < SM_BINS) cut = d.template resolve<false>(each_found, any, p, (uint64_t)s.top_k, 0.0);
    if (s.top_p < 1.0f) cut = d.cut_by_mass(each_found, cut);
  } else if (cuts && !few_found) {
    auto any = [](float, auto) { return true; };
    cut = d.template resolve<true>(each_found, any, p, 0, target);
  }
  const uint64_t tie_w = d.tie_weight(cut);

  // the parts' kept weights and their ties
  if (whole || s.way == kCount || from < SM_BINS) {
    auto add = [&](int g, float x) __attribute__((always_inline)) {
      const uint32_t key = order_of(x);
      if (key > cut.key) {
        const uint64_t w = d.kept(d.weight(x));
        if (w) atomicAdd((unsigned long long*)&part_w[g], (unsigned long long)w);
      } else if (key == cut.key) {
        atomicAdd(&part_ties[g], 1u);
      }
    };
    if (whole) {
      for (int g = wave; g < a.parts; g += NW) {
        uint64_t sum = 0;
        uint32_t ties = 0;
        each_token<DT>(base, g * a.part, min((g + 1) * a.part, a.vocab), lane, 64,
                       [&](int, float x) __attribute__((always_inline)) {
                         const uint32_t key = order_of(x);
                         if (key > cut.key) sum += d.kept(d.weight(x));
                         ties += key == cut.key;
                       });
        sum = wave_sum64(sum);
        const uint64_t t = wave_sum64(ties);
        if (lane == 0) part_w[g] = sum, part_ties[g] = (uint32_t)t;
      }
    } else {
      for (int i = lane; i < mine_n; i += 64) add(my_i[i] / a.part, my_x[i]);
    }
  }
  __syncthreads();
  // the parts, one a lane of every wave: the weight and the ties before each; the first at whose end the kept weights pass r
  const uint64_t pw = part_w[lane] + (whole ? 0 : part_ahead), pt = part_ties[lane];
  const uint64_t pw_end = wave_scan64(pw), pt_end = wave_scan64(pt);
  const uint64_t end = pw_end + D::ties_in(cut, 0, pt_end) * tie_w, total = lane64(end, 63), r = d.drawn(total);
  const int at = max(__ffsll((unsigned long long)__ballot(end > r)) - 1, 0);
  uint64_t upto = lane64(pt_end - pt, at), cum = lane64(pw_end - pw, at) + D::ties_in(cut, 0, upto) * tie_w;
  // that part's tokens, PER neighbouring ones a thread at a time
  const int end_at = min((at + 1) * a.part, a.vocab);
  auto search = [&](auto per_c) __attribute__((always_inline)) {
    constexpr int PER = decltype(per_c)::value;
    for (int p0 = at * a.part; p0 < end_at; p0 += NT * PER) {
      const int i0 = p0 + PER * tid, n_here = min(max(end_at - i0, 0), PER);
      float x[PER];
      uint64_t w[PER], sum = 0, ties = 0, sum_before, ties_before, sum_all, ties_all;
      run_of<DT>(base, i0, n_here, x);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t key = order_of(x[i]);
        w[i] = d.weight(x[i]);
        if (key > cut.key) sum += d.kept(w[i]);
        ties += i < n_here && key == cut.key;
      }
      d.scan(sum, ties, sum_before, ties_before, sum_all, ties_all);
      const uint64_t first = cum + sum_before + D::ties_in(cut, upto, ties_before) * tie_w;
      if (first <= r && first + sum + D::ties_in(cut, upto + ties_before, ties) * tie_w > r)
        d.pick(cut, tie_w, first, upto + ties_before, r, total, i0, n_here, x, w);
      cum += sum_all + D::ties_in(cut, upto, ties_all) * tie_w;
      upto += ties_all;
      if (cum > r) break;
    }
  };
  // (a larger part in half as many turns: 256 rows of 131072 41.0 us, 42.1 with four tokens a thread)
  if (a.part == SM_PART) search(std::integral_constant<int, SM_PART / NT>{});
  else search(std::integral_constant<int, 2 * SM_PART / NT>{});
}

// tokens a part of a row of `vocab`, of `rows`: SM_PART, more where that gives more than SM_PARTS parts, or more workgroups
// than keep the chip busy (a part costs 3 KB of bins, written and read): 256 rows of 131072 with a top_k of 40 take 49 us with
// parts of 8192 and 55 with 4096; 64 rows 38 with either, 33 against 28 (top_k) with 2048.
int part_of(int64_t rows, int64_t vocab) {
  int64_t part = SM_PART;
  while (part * SM_PARTS < vocab || (part < 2 * SM_PART && rows * (vocab / part) > 4096)) part *= 2;
  return (int)part;
}
bool row_is_held(int64_t vocab) { return vocab <= 1024 * SM_HELD; }

template <int DT>
void launch_sample(const SampleArgs& a, int64_t rows, hipStream_t st) {
  const dim3 grid((unsigned)rows), parts((unsigned)(rows * a.parts));
  if (a.vocab <= 256 * SM_HELD) {
    hipLaunchKernelGGL((sample_held_kernel<DT, 4>), grid, dim3(256), 0, st, a);
  } else if (row_is_held(a.vocab)) {
    hipLaunchKernelGGL((sample_held_kernel<DT, 16>), grid, dim3(1024), 0, st, a);
  } else {
    hipLaunchKernelGGL((sample_max_kernel<DT>), parts, dim3(256), 0, st, a);
    hipLaunchKernelGGL((sample_bins_kernel<DT>), parts, dim3(256), 0, st, a);
    hipLaunchKernelGGL((sample_draw_kernel<DT>), grid, dim3(1024), 0, st, a);
  }
}

}  // namespace

extern "C" int64_t gwa_sample_tokens_workspace(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0 || vocab > (1 << 24) || row_is_held(vocab)) return 0;
  const int64_t part = part_of(rows, vocab);
  return rows * ((vocab + part - 1) / part) * (SM_BINS * 8 + 4);
}

extern "C" int gwa_sample_tokens(const void* logits, int64_t ld, int dtype, const float* uniform,
                                 const gwa_sampling* settings, int64_t* tokens, float* logprobs, int64_t rows,
                                 int64_t vocab, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "sample_tokens";
  GWA_REQUIRE(settings, "%s: null settings", what);
  GWA_REQUIRE(dtype >= GWA_DT_BF16 && dtype <= GWA_DT_F32, "%s: dtype %d", what, dtype);
  GWA_REQUIRE(vocab > 0 && vocab <= (1 << 24) && rows >= 0 && rows < (1ll << 31), "%s: %lld rows of %lld tokens (1 to 2^24)",
              what, (long long)rows, (long long)vocab);
  const gwa_sampling& s = *settings;
  GWA_REQUIRE(s.temperature || (s.all_temperature >= 0.0f && s.all_temperature < INFINITY),
              "%s: a temperature of %g", what, (double)s.all_temperature);
  GWA_REQUIRE(s.top_k || s.all_top_k >= 0, "%s: top_k %d", what, s.all_top_k);
  GWA_REQUIRE(s.top_p || (s.all_top_p >= 0.0f && s.all_top_p <= 1.0f), "%s: top_p %g", what, (double)s.all_top_p);
  GWA_REQUIRE(s.min_p || (s.all_min_p >= 0.0f && s.all_min_p <= 1.0f), "%s: min_p %g", what, (double)s.all_min_p);
  if (rows == 0) return GWA_OK;
  GWA_REQUIRE(logits && uniform && tokens && logprobs, "%s: null pointer", what);
  const int elem = dtype == GWA_DT_F32 ? 4 : 2;
  GWA_REQUIRE(ld >= vocab && ld < (1ll << 40), "%s: a row stride of %lld", what, (long long)ld);
  GWA_REQUIRE(GWA_ALIGNED(logits, elem) && GWA_ALIGNED(uniform, 4) && GWA_ALIGNED(tokens, 8) && GWA_ALIGNED(logprobs, 4) &&
                  GWA_ALIGNED(s.temperature, 4) && GWA_ALIGNED(s.top_k, 4) && GWA_ALIGNED(s.top_p, 4) &&
                  GWA_ALIGNED(s.min_p, 4),
              "%s: misaligned pointer", what);
  int bits = 0;  // sums of `vocab` weights stay below 2^62
  while ((1ll << bits) < vocab) ++bits;
  const int64_t need = gwa_sample_tokens_workspace(rows, vocab), part = part_of(rows, vocab);
  const int64_t parts = (vocab + part - 1) / part;
  GWA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && GWA_ALIGNED(workspace, 16)),
              "%s: a workspace of %lld bytes, %lld are needed (16-byte aligned)", what, (long long)workspace_bytes,
              (long long)need);
  GWA_REQUIRE(rows * max((int64_t)1024, 256 * parts) < (1ll << 32), "%s: %lld rows of %lld tokens are too many", what,
              (long long)rows, (long long)vocab);
  uint64_t* bins = (uint64_t*)workspace;
  const SampleArgs a = {logits, ld, uniform, s, tokens, logprobs, (int)vocab, bits <= 17 ? 45 : 62 - bits, (int)parts,
                        (int)part, bins, need ? (float*)(bins + rows * parts * SM_BINS) : nullptr};
  if (dtype == GWA_DT_BF16) launch_sample<GWA_DT_BF16>(a, rows, (hipStream_t)stream);
  else if (dtype == GWA_DT_F16) launch_sample<GWA_DT_F16>(a, rows, (hipStream_t)stream);
  else launch_sample<GWA_DT_F32>(a, rows, (hipStream_t)stream);
  return gwa_check_launch(what);
}
