// Drawing the next tokens from a step's logits: temperature, top-k, top-p, min-p, one given random number a row.
#include <type_traits>

#include "gwa_common.h"

namespace {

constexpr int SM_THREADS = 1024, SM_WAVES = SM_THREADS / 64, SM_BINS = 1024, SM_DIGITS = 2048, SM_LIST = 1024;
constexpr int SM_AHEAD = 4;       // 16-byte loads a lane has in flight
constexpr float SM_PER_UNIT = 32.0f;  // bins a unit of (m - x) / temperature
constexpr int kTableBits = 5;     // of the table of 2^(j / 32)

struct SampleArgs {
  const void* logits;
  int64_t ld;
  const float* uniform;
  gwa_sampling s;
  int64_t* tokens;
  float* logprobs;
  int vocab, shift;  // weights are integers of 2^-shift
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

// A row's weights: w = exp((x - m) / temperature) as an integer of 2^-shift. With y = (x - m) log2(e) / temperature in
// 64 bits, 2^y = 2^n 2^(j/32) 2^r, |r| <= 1/64: a table and the series of 2^r to r^5 (the rest is below 2^-48), rounded to
// an integer by an addition of 2^52.
struct Weigher {
  double c;  // log2(e) / temperature
  float m;
  int shift;
  const double* table;
  __device__ __forceinline__ uint64_t operator()(float x) const {
    const double y = ((double)x - (double)m) * c;
    uint64_t w = 0;
    if (y >= -47.0) {  // not for -inf and NaN
      constexpr double kMagic = 6755399441055744.0 / (1 << kTableBits);  // 1.5 * 2^52: its last bit is 1 / 32
      const double t = y + kMagic;
      const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, t);
      const double r = y - (t - kMagic);
      // ln(2)^i / i!
      double p = 1.3333558146428441e-3;
      p = __builtin_fma(p, r, 9.6181291076284772e-3);
      p = __builtin_fma(p, r, 5.5504108664821580e-2);
      p = __builtin_fma(p, r, 2.4022650695910072e-1);
      p = __builtin_fma(p, r, 6.9314718055994531e-1);
      p = __builtin_fma(p, r, 1.0);
      p = __builtin_amdgcn_ldexp(p * table[k & ((1 << kTableBits) - 1)], shift + (k >> kTableBits));
      w = __builtin_bit_cast(uint64_t, p + 4503599627370496.0) & 0xfffffffffffffull;
    }
    return x == m ? 1ull << shift : w;
  }
};

__device__ __forceinline__ uint64_t shfl64(uint64_t x, int lane) {
  const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)x, lane), hi = (uint32_t)__shfl((int)(x >> 32), lane);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t shfl64_up(uint64_t x, int by) {
  const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)x, by), hi = (uint32_t)__shfl_up((int)(x >> 32), by);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t x) {
  for (int w = 32; w; w >>= 1) x += shfl64(x, (threadIdx.x & 63) ^ w);
  return x;
}

struct SampleLds {
  double table[1 << kTableBits];
  uint64_t mass[SM_DIGITS];
  uint32_t count[SM_DIGITS];
  uint64_t list_w[SM_LIST];
  uint32_t list_key[SM_LIST];
  uint64_t cells[2][SM_WAVES];
  uint64_t found[4];
  uint32_t n;
};

// Sums of a and b over the threads before this one, in the threads' order, and over all
__device__ __forceinline__ void block_scan(SampleLds& l, uint64_t a, uint64_t b, uint64_t& a_before, uint64_t& b_before,
                                           uint64_t& a_all, uint64_t& b_all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t x = a, y = b;
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) {
    const uint64_t p = shfl64_up(x, w), q = shfl64_up(y, w);
    if (lane >= w) x += p, y += q;
  }
  __syncthreads();
  if (lane == 63) l.cells[0][wave] = x, l.cells[1][wave] = y;
  __syncthreads();
  a_before = x - a, b_before = y - b, a_all = b_all = 0;
  for (int i = 0; i < SM_WAVES; ++i) {
    if (i < wave) a_before += l.cells[0][i], b_before += l.cells[1][i];
    a_all += l.cells[0][i], b_all += l.cells[1][i];
  }
}

// What a cut keeps: the tokens ordered above `key`, and of those equal to it the first `ties` by index. `equal`: how many
// those are, `above`: the weight of the ones before them (where weights were asked for).
struct Cut {
  uint32_t key;
  uint32_t ties, equal;
  uint64_t above;
};

// One workgroup a row, several passes over its logits (from the caches after the first): the largest; for a cut a histogram
// of the tokens by their distance from it, then the tokens of the one bin that the cut falls into, ranked by counting; the
// kept weights of 16 parts of the vocabulary; and the tokens of the part that the random number falls into.
template <int DT>
__global__ __launch_bounds__(SM_THREADS) void sample_rows_kernel(SampleArgs a) {
  using L = Logits<DT>;
  __shared__ SampleLds l;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const uint8_t* base = (const uint8_t*)a.logits + row * a.ld * L::kBytes;
  const int vocab = a.vocab;
  auto held = [](float x, float lo, float hi) { return fminf(fmaxf(x, lo), hi); };
  const float temperature = a.s.temperature ? a.s.temperature[row] : a.s.all_temperature;
  const int top_k = a.s.top_k ? a.s.top_k[row] : a.s.all_top_k;
  const float top_p = held(a.s.top_p ? a.s.top_p[row] : a.s.all_top_p, 0.0f, 1.0f);
  const float min_p = held(a.s.min_p ? a.s.min_p[row] : a.s.all_min_p, 0.0f, 1.0f);

  // The waves' parts of the row, [part(i), part(i + 1)): tokens before the first 16-byte boundary, whole 16-byte pieces,
  // and the rest, so that loads are wide whatever the row's alignment is
  const int head = min((int)((16 - ((uintptr_t)base & 15)) & 15) / L::kBytes, vocab);
  const int vecs = (vocab - head) / L::kVec;
  const int per = (vecs + SM_WAVES - 1) / SM_WAVES;
  auto vec_of = [&](int w) { return min(w * per, vecs); };
  auto part = [&](int w) { return w == 0 ? 0 : w == SM_WAVES ? vocab : head + vec_of(w) * L::kVec; };
  const v4i* body = (const v4i*)(base + head * L::kBytes);
  // f(index, logit) over this wave's part
  auto each = [&](auto f) __attribute__((always_inline)) {
    if (wave == 0 && lane < head) f(lane, L::at(base, lane));
    const int v1 = vec_of(wave + 1);
    for (int v = vec_of(wave) + lane; v < v1; v += 64 * SM_AHEAD) {
      v4i x[SM_AHEAD];
#pragma unroll
      for (int u = 0; u < SM_AHEAD; ++u) x[u] = body[min(v + 64 * u, v1 - 1)];
#pragma unroll
      for (int u = 0; u < SM_AHEAD; ++u)
        if (v + 64 * u < v1) {
#pragma unroll
          for (int e = 0; e < L::kVec; ++e) f(head + (v + 64 * u) * L::kVec + e, L::of(x[u], e));
        }
    }
    const int tail = head + vecs * L::kVec + lane;
    if (wave == SM_WAVES - 1 && tail < vocab) f(tail, L::at(base, tail));
  };

  if (tid < (1 << kTableBits)) l.table[tid] = exp2((double)tid / (1 << kTableBits));
  float m = -INFINITY;
  each([&](int, float x) __attribute__((always_inline)) { m = fmaxf(m, x); });
#pragma unroll
  for (int w = 32; w; w >>= 1) m = fmaxf(m, __shfl_xor(m, w));
  if (lane == 0) l.cells[0][wave] = __float_as_uint(m);
  __syncthreads();
  for (int i = 0; i < SM_WAVES; ++i) m = fmaxf(m, __uint_as_float((uint32_t)l.cells[0][i]));
  if (m == -INFINITY) {
    if (tid == 0) a.tokens[row] = -1, a.logprobs[row] = NAN;
    return;
  }
  if (!(temperature > 0.0f)) {
    if (tid == 0) l.n = 0xffffffffu;
    __syncthreads();
    uint32_t first = 0xffffffffu;
    each([&](int i, float x) __attribute__((always_inline)) { first = x == m ? min(first, (uint32_t)i) : first; });
    if (first != 0xffffffffu) atomicMin(&l.n, first);
    __syncthreads();
    if (tid == 0) a.tokens[row] = l.n, a.logprobs[row] = 0.0f;
    return;
  }
  const Weigher weight = {1.4426950408889634 / (double)temperature, m, a.shift, l.table};
  const float per_unit = SM_PER_UNIT / temperature;
  // bins of falling logits; the last takes all from SM_BINS - 1 on, whose weights are 0
  auto bin_of = [&](float x) __attribute__((always_inline)) {
    const float d = (m - x) * per_unit;
    return x == m ? 0 : d < (float)(SM_BINS - 1) ? (int)d : SM_BINS - 1;
  };

  // The cut at the want-th token (MASS: at which the weight reaches `target`) among those ordered at or above `least`
  auto cut_at = [&](auto mass_c, uint32_t least, uint64_t want, auto target_of) __attribute__((always_inline)) {
    constexpr bool MASS = decltype(mass_c)::value;
    __syncthreads();
    l.count[tid] = 0, l.mass[tid] = 0;
    if (tid == 0) l.n = 0;
    __syncthreads();
    each([&](int, float x) __attribute__((always_inline)) {
      const int b = bin_of(x);
      if (b < SM_BINS - 1 && (!MASS || order_of(x) >= least)) {
        atomicAdd(&l.count[b], 1u);
        if (MASS) atomicAdd((unsigned long long*)&l.mass[b], (unsigned long long)weight(x));
      }
    });
    __syncthreads();
    uint64_t n = l.count[tid], w = l.mass[tid], n_before, w_before, n_all, w_all;
    block_scan(l, n, w, n_before, w_before, n_all, w_all);
    const double target = MASS ? target_of(w_all) : 0.0;
    if (!MASS && tid == SM_BINS - 1) n = vocab - n_all;  // the last bin's
    const bool here = MASS ? (double)w_before < target && (double)(w_before + w) >= target
                           : n_before < want && n_before + n >= want;
    if (here) l.found[0] = tid, l.found[1] = n_before, l.found[2] = w_before, l.found[3] = n;
    __syncthreads();
    const int bin = (int)l.found[0];
    uint64_t before = l.found[1], above = l.found[2];
    const uint32_t inside = (uint32_t)l.found[3];
    __syncthreads();
    Cut cut;
    // the ties that are kept of `equal` weights w each behind a weight of `above`: as few as reach the target
    auto ties_to = [&](uint64_t from, uint64_t w, uint32_t equal) __attribute__((always_inline)) {
      uint32_t e = w ? (uint32_t)fmin(fmax(ceil((target - (double)from) / (double)w), 1.0), (double)equal) : 1;
      while (e > 1 && (double)(from + (e - 1) * w) >= target) --e;
      while (e < equal && (double)(from + e * w) < target) ++e;
      return e;
    };
    if (inside <= SM_LIST) {
      each([&](int, float x) __attribute__((always_inline)) {
        if (bin_of(x) == bin && (!MASS || order_of(x) >= least)) {
          const uint32_t i = atomicAdd(&l.n, 1u);
          l.list_key[i] = order_of(x);
          if (MASS) l.list_w[i] = weight(x);
        }
      });
      __syncthreads();
      if (tid < (int)inside) {
        const uint32_t key = l.list_key[tid];
        uint32_t over = 0, equal = 0;
        uint64_t heavier = 0;
        for (uint32_t i = 0; i < inside; ++i) {
          const uint32_t k = l.list_key[i];
          over += k > key, equal += k == key;
          if (MASS) heavier += k > key ? l.list_w[i] : 0;
        }
        const uint64_t from = above + heavier;
        const uint64_t mine = MASS ? l.list_w[tid] : 0;
        const bool at = MASS ? (double)from < target && (double)(from + equal * mine) >= target
                             : before + over < want && before + over + equal >= want;
        if (at) {  // equal ones all write the same
          l.found[0] = key, l.found[1] = equal, l.found[2] = from;
          l.found[3] = MASS ? ties_to(from, mine, equal) : want - before - over;
        }
      }
      __syncthreads();
      cut = {(uint32_t)l.found[0], (uint32_t)l.found[3], (uint32_t)l.found[1], l.found[2]};
    } else {
      // digit by digit of the ordered values: 11 + 11 + 10 bits
      uint32_t prefix = 0, in_digit = 0;
      uint64_t digit_w = 0;
      int shift = 21;
      for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < SM_DIGITS; i += SM_THREADS) l.count[i] = 0, l.mass[i] = 0;
        __syncthreads();
        each([&](int, float x) __attribute__((always_inline)) {
          const uint32_t key = order_of(x);
          if (bin_of(x) == bin && (!MASS || key >= least) && (pass == 0 || key >> (shift + bits) == prefix)) {
            const uint32_t d = key >> shift & ((1u << bits) - 1);
            atomicAdd(&l.count[d], 1u);
            if (MASS) atomicAdd((unsigned long long*)&l.mass[d], (unsigned long long)weight(x));
          }
        });
        __syncthreads();
        // digits from the top, two a thread
        const int d1 = SM_DIGITS - 1 - 2 * tid, d0 = d1 - 1;
        const uint32_t n1 = l.count[d1], n0 = l.count[d0];
        const uint64_t w1 = l.mass[d1], w0 = l.mass[d0];
        uint64_t n_up, w_up, na, wa;
        block_scan(l, n1 + n0, w1 + w0, n_up, w_up, na, wa);
        n_up += before, w_up += above;
        auto check = [&](int d, uint64_t nb, uint64_t wb, uint32_t n, uint64_t w) __attribute__((always_inline)) {
          const bool at = MASS ? (double)wb < target && (double)(wb + w) >= target : nb < want && nb + n >= want;
          if (at) l.found[0] = (uint64_t)d << 32 | n, l.found[1] = nb, l.found[2] = wb, l.found[3] = w;
        };
        check(d1, n_up, w_up, n1, w1);
        check(d0, n_up + n1, w_up + w1, n0, w0);
        __syncthreads();
        prefix = prefix << bits | (uint32_t)(l.found[0] >> 32);
        in_digit = (uint32_t)l.found[0];
        before = l.found[1], above = l.found[2], digit_w = l.found[3];
        shift = pass == 0 ? 10 : 0;
        __syncthreads();
      }
      cut = {prefix, MASS ? ties_to(above, digit_w / in_digit, in_digit) : (uint32_t)(want - before), in_digit, above};
    }
    __syncthreads();
    return cut;
  };

  Cut cut = {0, (uint32_t)vocab, (uint32_t)vocab, 0};
  uint32_t least = 0, dropped = 0;  // of the tokens at `least`, the last `dropped` are not among the first top_k
  if (top_k > 0 && top_k < vocab) {
    cut = cut_at(std::false_type{}, 0, (uint64_t)top_k, [](uint64_t) { return 0.0; });
    least = cut.key, dropped = cut.equal - cut.ties;
  }
  auto value_of = [](uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); };
  if (top_p < 1.0f) {
    const uint64_t off = dropped ? dropped * weight(value_of(least)) : 0;
    cut = cut_at(std::true_type{}, least, 0, [&](uint64_t all) {
      return fmax((double)top_p * (double)(all - off), 0.5);  // the first token reaches 0.5 alone
    });
  }

  // the kept weights of the waves' parts, and the ties in them
  const double low = (double)min_p * (double)(1ull << a.shift);
  auto kept = [&](float x) __attribute__((always_inline)) {
    const uint64_t w = weight(x);
    return (double)w >= low ? w : 0;
  };
  const uint64_t tie_w = cut.key ? kept(value_of(cut.key)) : 0;
  uint64_t sum = 0, ties = 0;
  each([&](int, float x) __attribute__((always_inline)) {
    const uint32_t key = order_of(x);
    if (key > cut.key) sum += kept(x);
    ties += key == cut.key;
  });
  sum = wave_sum64(sum), ties = wave_sum64(ties);
  __syncthreads();
  if (lane == 0) l.cells[0][wave] = sum, l.cells[1][wave] = ties;
  __syncthreads();
  uint64_t total = 0, n_ties = 0;
  auto ties_in = [&](uint64_t upto, uint64_t n) {  // those kept of n ties behind `upto` others
    return upto >= cut.ties ? 0 : min(n, (uint64_t)cut.ties - upto);
  };
  for (int i = 0; i < SM_WAVES; ++i) {
    total += l.cells[0][i] + ties_in(n_ties, l.cells[1][i]) * tie_w;
    n_ties += l.cells[1][i];
  }
  // cum > u total: for integers, cum > floor(u total)
  const uint64_t r = min((uint64_t)((double)held(a.uniform[row], 0.0f, 1.0f) * (double)total), total - 1);
  uint64_t cum = 0, upto = 0;
  int at = 0;
  for (; at < SM_WAVES - 1; ++at) {
    const uint64_t next = cum + l.cells[0][at] + ties_in(upto, l.cells[1][at]) * tie_w;
    if (next > r) break;
    cum = next, upto += l.cells[1][at];
  }
  // that part's tokens, neighbouring ones a thread
  const int p0 = part(at), len = part(at + 1) - p0, each_n = (len + SM_THREADS - 1) / SM_THREADS;
  const int i0 = min(tid * each_n, len), i1 = min(i0 + each_n, len);
  sum = ties = 0;
  for (int i = i0; i < i1; ++i) {
    const float x = L::at(base, p0 + i);
    const uint32_t key = order_of(x);
    if (key > cut.key) sum += kept(x);
    ties += key == cut.key;
  }
  uint64_t sum_before, ties_before, sa, ta;
  block_scan(l, sum, ties, sum_before, ties_before, sa, ta);
  upto += ties_before;
  // kept ties before this thread's tokens, less those before the part
  const uint64_t first_tie = upto - ties_before;
  uint64_t c = cum + sum_before + ties_in(first_tie, ties_before) * tie_w;
  if (c <= r && c + sum + ties_in(upto, ties) * tie_w > r) {
    for (int i = i0; i < i1; ++i) {
      const float x = L::at(base, p0 + i);
      const uint32_t key = order_of(x);
      uint64_t w = 0;
      if (key > cut.key) w = kept(x);
      else if (key == cut.key) w = upto++ < cut.ties ? tie_w : 0;
      c += w;
      if (c > r) {
        a.tokens[row] = p0 + i;
        const double y = x == m ? 0.0 : ((double)x - (double)m) / (double)temperature;
        a.logprobs[row] = (float)(y - log((double)total / (double)(1ull << a.shift)));
        break;
      }
    }
  }
}

}  // namespace

extern "C" int gwa_sample_tokens(const void* logits, int64_t ld, int dtype, const float* uniform,
                                 const gwa_sampling* settings, int64_t* tokens, float* logprobs, int64_t rows,
                                 int64_t vocab, void* stream) {
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
  const SampleArgs a = {logits, ld, uniform, s, tokens, logprobs, (int)vocab, bits <= 17 ? 45 : 62 - bits};
  const dim3 grid((unsigned)rows), block(SM_THREADS);
  if (dtype == GWA_DT_BF16) hipLaunchKernelGGL((sample_rows_kernel<GWA_DT_BF16>), grid, block, 0, (hipStream_t)stream, a);
  else if (dtype == GWA_DT_F16) hipLaunchKernelGGL((sample_rows_kernel<GWA_DT_F16>), grid, block, 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL((sample_rows_kernel<GWA_DT_F32>), grid, block, 0, (hipStream_t)stream, a);
  return gwa_check_launch(what);
}
