// Drawing a token per logits row: temperature, top-k, top-p and min-p from given random numbers.
//
// The mathematics. Tokens of a row stand in order of their logit, the largest first, the lower index first among equals. With
// w(l) = exp((l - max) / T) each filter keeps the first so many of them: top-k the first k; top-p the fewest whose weights reach
// top_p of what top-k left; min-p those of w >= min_p. What all of them keep is the first n, of mass m, and the token drawn is the
// first one whose running sum of weights exceeds u m.
//
// Weights and sums are in 64 bits: a running sum over a vocabulary in 32 bits moves the borders between tokens by up to 1e-6 of
// the mass, so that one draw in a hundred of a flat row would be another token's. What makes 64 bits cheap is that a row of bf16 has
// few values: the kernel counts how often each occurs and takes one exponential a value, 1000 to 2000 of them instead of 128256,
// and the order of tokens is the order of values. Counts are whole numbers, so that no order of atomics changes a bit; masses are
// summed in a fixed tree over the values, whatever the number of CTAs a row has.
//
// Counting: a bin a value, of the magnitudes [2^-25, 2^7) of either sign (the home window), 32 KB of shared memory. A row with
// other magnitudes (but for -inf, and one smaller value of either sign, as a row in five hundred has) takes another pass over
// itself for each of the eight other windows of 32 binary orders that it has values in, so that any row is exact; zeros are
// counted apart. The counts and masses of the binades lie in shared memory of every CTA of the row's cluster, which then all look
// for the same borders. A bin also adds up where its values stand, so that a value that a CTA has once is found without
// another pass: 512 rows of 256000 took 159 -> 141 us.
//
// What bounds it. Few rows: launch, three cluster barriers and the search's chains of latencies, 2200 cycles a border: one row of
// 128256 11.6 us, seven of 50001 13.1. Many: the counting, at 0.7 of what shared memory's atomics take (3.6 wavefronts for a warp's 32
// places), and behind it the accounts and the search, 17000 cycles that only the SM's other CTAs can fill: 128 rows of 128256
// 24.5 us, 192 31.9 (384 CTAs in 444 places; 7.5 us at a copy's rate), 512 of 256000 102 (40). One CTA a row 47 at 192. Masked tokens
// all meet in one bin, whose atomics come one after the other, and a finite mask's window takes passes of its own: 192 rows of
// 128256 with 99 % of -inf take 115 us, of the type's lowest value 240 (30 without).
#include "kc_fused.cuh"
#include "kc_umma.cuh"

namespace kc {

namespace {

// Threads of a CTA, by the CTAs of a row and of an SM: half as many where a row has many, whose barriers then take less (one row of 128256 12.8 ->
// 11.5 us), and where an SM has three.
constexpr int draw_threads(int ctas, int resident) { return ctas > 2 || resident > 2 ? 256 : 512; }
constexpr int DRAW_WINDOW = 4096;                 // magnitudes (bf16 without the sign) of a window, 32 binades
constexpr int DRAW_LOW = 4, DRAW_SIDE = 4128;     // of a sign's bins: the window's first one; all of them (next to the window's: what lies below, above)
constexpr int DRAW_HOME = 4;                      // the window that holds a language model's logits: magnitudes 2^-25 to 2^7
constexpr int DRAW_BASE0 = 102 * 128 - DRAW_HOME * DRAW_WINDOW;   // first magnitude of window 0 (below zero: it is a short one)
constexpr int DRAW_WINDOWS = 9;
// A bin counts in its low bits and adds up the indices of the vectors in the high ones, which is the place of a value that occurs once.
constexpr int DRAW_AT = 18;
// Binades in falling order of value: a run of 32 for each window, the positive ones' from the last window to the first, a run
// that holds zero alone, the negative ones'.
constexpr int DRAW_ZERO = DRAW_WINDOWS, DRAW_RUNS = 2 * DRAW_WINDOWS + 1;
constexpr uint32_t BF16_INF = 0x7F80u;
static_assert(DRAW_BASE0 % 128 == 0 && DRAW_BASE0 + DRAW_WINDOWS * DRAW_WINDOW > 0x7F80, "windows cover all magnitudes in whole binades");

// C: CTAs of a row's cluster. Every C-th binade of the resident window is a CTA's own, to add up over the cluster's parts of the row.
template <int C, int RESIDENT>
struct DrawShared {
  uint32_t bins[2 * DRAW_SIDE];                   // [sign][magnitude]: how often the value occurs in this CTA's part of the row, and where (DRAW_AT)
  double lane_weight[64 / C][32];                 // own binades, four values a lane: the weight of the lane's first one,
  double lane_mass[64 / C][32];                   // mass and
  uint32_t lane_count[64 / C][32];                // tokens of the binade up to the lane's last one
  uint4 lane_counts[C > 2 ? 64 / C : 1][32];      // C > 2: how often each value occurs in the row, in falling order
  double mass[DRAW_RUNS][32];                     // of a binade; later of its run up to it
  uint32_t count[DRAW_RUNS][32];
  uint32_t peer_top[8], peer_out[8], peer_lone[8], peer_seen[8], peer_zeros[8], peer_match[8];   // what each CTA of the cluster found
  uint32_t warp_a[draw_threads(C, RESIDENT) / 32], warp_b[draw_threads(C, RESIDENT) / 32];
  uint32_t far;                                   // whether a finite value lies below the window's negative ones
  uint32_t above;                                 // tokens of w >= min_p, over the cluster
  double ratio[32];                               // of the weights of neighbouring values, by binade of the resident window
  int window;                                     // the one that the search wants resident; -1: it is done
  uint32_t bits, taken; double weight, mass_kept;   // its result
};

__device__ __forceinline__ void peer_put(uint32_t* p, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(cluster_addr(smem_u32(p), rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void peer_put(double* p, uint32_t rank, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(cluster_addr(smem_u32(p), rank)), "d"(v) : "memory");
}
__device__ __forceinline__ void peer_add(uint32_t* p, uint32_t rank, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(cluster_addr(smem_u32(p), rank)), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t peer_get(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ double peer_get(const double* p, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(cluster_addr(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint4 peer_get4(const uint32_t* p, uint32_t rank) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(cluster_addr(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ float value_of(uint32_t bits) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ uint32_t top_bf162(uint32_t a, uint32_t b) {   // a NaN gives way to a number
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t low_bf162(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// 0xFFFF in the halves that are equal as numbers (-0 is +0, NaN is nothing).
__device__ __forceinline__ uint32_t equal_bf162(uint32_t a, uint32_t b) {
  return __heq2_mask(*reinterpret_cast<const bf162*>(&a), *reinterpret_cast<const bf162*>(&b));
}

// A row as vectors of eight values on 16-byte boundaries: the first and the last one may hang over, and have -inf there.
struct DrawRow {
  const bf16* row;
  const uint4* base;                              // vector 0
  int vocab, shift, whole0, whole1;               // the row starts at value `shift` of vector 0; vectors that don't hang over
  __device__ __forceinline__ DrawRow(const bf16* r, int n) : row(r), vocab(n) {
    shift = (int)(reinterpret_cast<uintptr_t>(r) & 15) / 2;
    base = reinterpret_cast<const uint4*>(r - shift);
    whole0 = shift ? 1 : 0;
    whole1 = (shift + n) / 8;
  }
  __device__ __forceinline__ int vecs() const { return (shift + vocab + 7) / 8; }
  __device__ __forceinline__ uint4 vec(int v) const {
    if (v >= whole0 && v < whole1) return base[v];
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = 8 * v - shift + 2 * k;
      const uint32_t a = i >= 0 && i < vocab ? reinterpret_cast<const unsigned short*>(row)[i] : 0xFF80u;
      const uint32_t b = i + 1 >= 0 && i + 1 < vocab ? reinterpret_cast<const unsigned short*>(row)[i + 1] : 0xFF80u;
      w[k] = a | b << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // f of the vectors [from, to) and their indices in any order, `at` of WIDTH threads taking every WIDTH-th: four loads are on their way under the
  // four vectors before.
  template <int WIDTH, typename F>
  __device__ __forceinline__ void each(int from, int to, int at, F&& f) const {
    constexpr int UNROLL = 4;
    if (at == 0) {
      if (from < min(to, whole0)) f(vec(from), from);
      if (to > max(max(from, whole0), whole1)) f(vec(to - 1), to - 1);
    }
    const int begin = max(from, whole0);
    int left = min(to, whole1) - begin - at, v = begin + at;
    const uint4* p = base + begin + at;
    uint4 u[UNROLL], next[UNROLL];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k)
      if (k * WIDTH < left) u[k] = p[k * WIDTH];
#pragma unroll 1
    for (; left > 0; left -= WIDTH * UNROLL) {
      p += WIDTH * UNROLL;
#pragma unroll
      for (int k = 0; k < UNROLL; ++k)
        if ((k + UNROLL) * WIDTH < left) next[k] = p[k * WIDTH];
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) {
        if (k * WIDTH < left) f(u[k], v + k * WIDTH);
        u[k] = next[k];
      }
      v += WIDTH * UNROLL;
    }
  }
};

template <int C, int RESIDENT>
__global__ void __launch_bounds__(draw_threads(C, RESIDENT), RESIDENT)
draw_rows_kernel(const bf16* __restrict__ logits, long long ld, int vocab, const DrawSetting* __restrict__ settings,
                 const float* __restrict__ uniform, uint32_t* __restrict__ tokens, float* __restrict__ logprobs,
                 uint32_t* __restrict__ tokens_host, float* __restrict__ logprobs_host, int skip_greedy) {
  constexpr int DRAW_THREADS = draw_threads(C, RESIDENT), DRAW_WARPS = DRAW_THREADS / 32;
  extern __shared__ __align__(16) uint8_t draw_smem[];
  DrawShared<C, RESIDENT>& s = *reinterpret_cast<DrawShared<C, RESIDENT>*>(draw_smem);
  pdl_launch_dependents();
  cluster_arrive();                      // waited for before the first access to another CTA's shared memory: it has started by then
  const int row_index = blockIdx.x / C, rank = blockIdx.x % C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto clear_bins = [&]() {
    for (int i = tid; i < 2 * DRAW_SIDE / 4; i += DRAW_THREADS) reinterpret_cast<uint4*>(s.bins)[i] = make_uint4(0, 0, 0, 0);
  };
  clear_bins();
  for (int i = tid; i < DRAW_RUNS * 32; i += DRAW_THREADS) { s.mass[0][i] = 0.0; s.count[0][i] = 0; }
  if (tid == 0) s.above = s.far = 0;
  __syncthreads();                       // the bins are clear before any thread counts: the arrival above says nothing about them
  cluster_wait();
  pdl_wait();
  const DrawSetting set = settings[row_index];
  const float u01 = uniform[row_index];
  const bool greedy = !(set.temperature > 0.f);
  const double inv_t = 1.0 / (double)set.temperature;
  // Distance of neighbouring values of a binade, over the temperature; subnormal ones lie like those of the first normal binade.
  auto step_of = [&](int binade) { return inv_t * __hiloint2double((max(binade, 1) - 127 - 7 + 1023) << 20, 0); };
  auto ratios = [&](int window) {
    if (tid < 32) s.ratio[tid] = exp(-step_of((DRAW_BASE0 + window * DRAW_WINDOW) / 128 + tid));
  };
  if (!greedy) ratios(DRAW_HOME);
  const bool skip = greedy && skip_greedy;

  const DrawRow x(logits + (size_t)row_index * ld, vocab);
  const int vecs = x.vecs(), per = (vecs + C - 1) / C;
  const int v0 = min(vecs, rank * per), v1 = skip ? v0 : min(vecs, v0 + per);
  const bool places_fit = per <= 1 << (32 - DRAW_AT);   // 8 values a vector: their counts fit below then too
  const uint32_t at_step = places_fit ? 1u << DRAW_AT : 0u, count_mask = places_fit ? (1u << DRAW_AT) - 1 : ~0u;
  static_assert(8 << (32 - DRAW_AT) < 1 << DRAW_AT, "counts");

  const bool lone_places = vocab <= 262000;   // whatever the cluster's size: a row's bits do not hang on it
  static_assert((262000 + 14) / 8 / 2 + 1 <= 1 << (32 - DRAW_AT), "places");
  // ---- pass over the row: bins of the home window, and the maximum. Two values at a time as halves of a register: their
  // magnitudes, held between the window's neighbours on either side, become places of bins by whole-number arithmetic that
  // neither half carries out of ----
  uint32_t top = 0xFF80FF80u, far = 0;   // far: of -inf 0, of a finite negative value its bits and 0x80: largest where the magnitude is
  constexpr uint32_t FIRST = DRAW_BASE0 + DRAW_HOME * DRAW_WINDOW;
  uint8_t* const bin_bytes = reinterpret_cast<uint8_t*>(s.bins);
  if (greedy) {
    x.each<DRAW_THREADS>(v0, v1, tid, [&](const uint4& u, int) { top = top_bf162(top, top_bf162(top_bf162(u.x, u.y), top_bf162(u.z, u.w))); });
  } else {
    x.each<DRAW_THREADS>(v0, v1, tid, [&](const uint4& u, int v) {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w}, one = 1u + (uint32_t)(v - v0) * at_step;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        top = top_bf162(top, w[j]);
        far = __viaddmax_u16x2(w[j], 0x00800080u, far);
        const uint32_t mag = low_bf162(top_bf162(w[j] & 0x7FFF7FFFu, (FIRST - 1) * 0x10001u), (FIRST + DRAW_WINDOW) * 0x10001u);
        const uint32_t at = mag * 4 + ((w[j] >> 15) & 0x00010001u) * (DRAW_SIDE * 4) - (FIRST - DRAW_LOW) * 4 * 0x10001u;   // bytes: 32912 at the most
        atomicAdd(reinterpret_cast<uint32_t*>(bin_bytes + (at & 0xFFFFu)), one);
        atomicAdd(reinterpret_cast<uint32_t*>(bin_bytes + (at >> 16)), one);
      }
    });
  }
  {
    const float2 two = unpack_bf162(top);
    const float m = warp_max(fmaxf(two.x, two.y));
    if (lane == 0) s.warp_a[warp] = __float_as_uint(m);
    constexpr uint32_t FAR = 0x8000u + FIRST + DRAW_WINDOW + 0x80u;
    if ((far & 0xFFFFu) >= FAR || (far >> 16) >= FAR) s.far = 1;
  }
  __syncthreads();
  const float m_cta = warp_max(__uint_as_float(s.warp_a[lane & (DRAW_WARPS - 1)]));
  // Values outside the home window, masked ones apart: how many lie below it (zeros and NaN among them; 2: more than one) of either sign,
  // whether any lies above. In a vocabulary's normal rows there is one below now and then, which its bin's place finds.
  constexpr int HIGH = DRAW_LOW + DRAW_WINDOW;
  if (tid < C) {
    uint32_t out = (s.bins[HIGH] | s.far) ? 16u : 0u, lone = 0;
#pragma unroll
    for (int sign = 0; sign < 2; ++sign) {
      const uint32_t bin = s.bins[sign * DRAW_SIDE + DRAW_LOW - 1], n = min(bin & count_mask, 2u);
      out |= n << (2 * sign);
      if (n == 1 && lone_places) {
        const uint4 u = x.vec(v0 + (int)(bin >> DRAW_AT));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t b = (w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu, mag = b & 0x7FFFu;
          if ((int)(b >> 15) == sign && (mag < FIRST || mag > BF16_INF)) lone |= mag << (16 * sign);
        }
      }
    }
    peer_put(&s.peer_top[rank], tid, __float_as_uint(m_cta));
    peer_put(&s.peer_out[rank], tid, out);
    peer_put(&s.peer_lone[rank], tid, lone);
  }
  cluster_sync();
  float largest = -INFINITY;
  uint32_t seen = 0, zeros = 0, lone = 0, above_window = 0, below[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < C; ++k) {
    largest = fmaxf(largest, __uint_as_float(s.peer_top[k]));
    const uint32_t out = s.peer_out[k];
    above_window |= out >> 4; below[0] += out & 3; below[1] += out >> 2 & 3;
    lone |= s.peer_lone[k];
  }
  // From here on every branch that holds a barrier is taken by the whole cluster: what it hangs on is the same in all its CTAs.
  if (above_window || max(below[0], below[1]) > (lone_places ? 1u : 0u)) {
    // A pass over the row: zeros are counted, of the others what windows they are in.
    below[0] = below[1] = 0;
    x.each<DRAW_THREADS>(v0, v1, tid, [&](const uint4& u, int) {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t b = (w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu, mag = b & 0x7FFFu;
        if (mag == 0) ++zeros;
        else if (mag < BF16_INF || b == BF16_INF) seen |= 1u << ((mag - (uint32_t)DRAW_BASE0) / DRAW_WINDOW);
      }
    });
    seen = __reduce_or_sync(0xffffffffu, seen) & ~(1u << DRAW_HOME);
    zeros = __reduce_add_sync(0xffffffffu, zeros);
    if (lane == 0) { s.warp_a[warp] = seen; s.warp_b[warp] = zeros; }   // the warps' maxima have been read
    __syncthreads();
    seen = zeros = 0;
    if (tid < C) {
      for (int w = 0; w < DRAW_WARPS; ++w) { seen |= s.warp_a[w]; zeros += s.warp_b[w]; }
      peer_put(&s.peer_seen[rank], tid, seen);
      peer_put(&s.peer_zeros[rank], tid, zeros);
    }
    cluster_sync();
    seen = zeros = 0;
#pragma unroll
    for (int k = 0; k < C; ++k) { seen |= s.peer_seen[k]; zeros += s.peer_zeros[k]; }
  } else {
    zeros = (below[0] && (lone & 0xFFFFu) == 0) + (below[1] && lone >> 16 == 0);
  }
  largest += 0.f;                        // -0 is +0
  const bool empty = largest == -INFINITY;   // nothing but masked tokens and NaN: token 0
  uint32_t bits = __float_as_uint(largest) >> 16, taken = 1;
  int resident = DRAW_HOME;              // window of the bins

  if (!greedy && !empty) {
    const double top_value = largest, min_p = set.min_p;
    auto weight_of = [&](uint32_t b) {
      const float l = value_of(b);
      return l == largest ? 1.0 : largest == INFINITY ? 0.0 : exp(((double)l - top_value) * inv_t);
    };
    // A binade's 128 values are four a lane, in falling order: of the k-th binade of the resident window (negative ones from 32 on) the place of
    // this lane's bins, and whether they lie in falling order of value as they are.
    auto place = [&](int k, int of_lane) { return (k >> 5) * DRAW_SIDE + DRAW_LOW + (k & 31) * 128 + 4 * ((k >> 5) ? of_lane : 31 - of_lane); };
    auto in_order = [](int k, uint4 v) { return (k >> 5) ? v : make_uint4(v.w, v.z, v.y, v.x); };
    auto first_bits = [&](int k, int of_lane) -> int {   // of the lane's largest value
      const int mag = DRAW_BASE0 + resident * DRAW_WINDOW + (k & 31) * 128;
      return (k >> 5) ? 0x8000 | (mag + 4 * of_lane) : mag + 127 - 4 * of_lane;
    };
    // The weights of a lane's values: the first one's by an exponential, the others by the ratio of neighbours (three
    // multiplications: 4e-16 of them), where that is no smaller than 1 / e, so that the first one is finite also where it lies past
    // the largest value.
    auto near = [&](int k) { return largest != INFINITY && step_of((DRAW_BASE0 + resident * DRAW_WINDOW) / 128 + (k & 31)) <= 1.0; };
    auto weights = [&](int k, int b, const uint32_t (&c)[4], double first, double (&w)[4]) {
      const int d = (k >> 5) ? 1 : -1;
      const bool chained = near(k);
      const double q = s.ratio[k & 31];
#pragma unroll
      for (int i = 0; i < 4; ++i, first *= q) {
        w[i] = 0.0;
        if (c[i]) w[i] = chained && value_of(b + i * d) != largest ? first : weight_of(b + i * d);
      }
    };
    // The cluster's counts of this lane's values.
    auto counts = [&](int k) {
      uint4 o[C], v = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < C; ++r) o[r] = peer_get4(&s.bins[place(k, lane)], (rank + r) & (C - 1));
#pragma unroll
      for (int r = 0; r < C; ++r) { v.x += o[r].x & count_mask; v.y += o[r].y & count_mask; v.z += o[r].z & count_mask; v.w += o[r].w & count_mask; }
      return v;
    };
    // Adds the cluster's bins of the resident window and what lanes hold of each binade; `enters`: its totals into every CTA's.
    auto account = [&](bool enters) {
      for (int i = rank + C * warp; i < 64; i += C * DRAW_WARPS) {
        const int k = i < 32 ? i : 32 + ((i + 16) & 31);   // a row's values lie in the same ten or so binades of either sign: one of them a warp
        uint4 v = counts(k);
        if (!__any_sync(0xffffffffu, (v.x | v.y | v.z | v.w) != 0)) continue;
        v = in_order(k, v);
        const uint32_t c[4] = {v.x, v.y, v.z, v.w};
        const int b = first_bits(k, lane);
        const double first = near(k) ? exp(((double)value_of(b) - top_value) * inv_t) : 0.0;
        double w[4], m = 0.0;
        weights(k, b, c, first, w);
        uint32_t above = 0, n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          m += c[i] * w[i]; n += c[i];
          if (w[i] >= min_p) above += c[i];
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t nu = __shfl_up_sync(0xffffffffu, n, o);
          const double mu = __shfl_up_sync(0xffffffffu, m, o);
          if (lane >= o) { n += nu; m += mu; }
        }
        if (C > 2) s.lane_counts[k / C][lane] = v;
        s.lane_weight[k / C][lane] = first; s.lane_mass[k / C][lane] = m; s.lane_count[k / C][lane] = n;
        if (!enters) continue;
        above = __reduce_add_sync(0xffffffffu, above);
        n = __shfl_sync(0xffffffffu, n, 31); m = __shfl_sync(0xffffffffu, m, 31);
        const int run = (k >> 5) ? DRAW_ZERO + 1 + resident : DRAW_ZERO - 1 - resident, e = (k >> 5) ? k & 31 : 31 - k;
        if (lane < C) {
          peer_put(&s.count[run][e], lane, n); peer_put(&s.mass[run][e], lane, m);
          if (above) peer_add(&s.above, lane, above);
        }
      }
    };
    // Makes another window the resident one: a pass over the row for its bins.
    auto enter = [&](int window, bool enters) {
      cluster_sync();                            // the bins have been read
      clear_bins();
      ratios(window);
      __syncthreads();
      resident = window;
      const uint32_t base = DRAW_BASE0 + window * DRAW_WINDOW;
      x.each<DRAW_THREADS>(v0, v1, tid, [&](const uint4& u, int v) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w}, one = 1u + (uint32_t)(v - v0) * at_step;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t b = (w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu, mag = b & 0x7FFFu;
          if (mag - base < DRAW_WINDOW && mag != 0 && (mag < BF16_INF || b == BF16_INF)) atomicAdd(&s.bins[(b >> 15) * DRAW_SIDE + DRAW_LOW + mag - base], one);
        }
      });
      cluster_sync();
      account(enters);
    };
    account(true);
    if (tid == 0 && zeros) {
      const double w = weight_of(0);
      s.count[DRAW_ZERO][0] = zeros; s.mass[DRAW_ZERO][0] = zeros * w;
      if (w >= min_p) peer_add(&s.above, rank, zeros);   // every CTA for itself
    }
    if (tid < 2 && below[tid]) {           // the one value below the window, positive or negative: the only one of its run
      const uint32_t mag = lone >> (16 * tid) & 0xFFFFu, at = mag - (uint32_t)DRAW_BASE0;
      if (mag != 0 && mag < BF16_INF) {
        const int run = tid ? DRAW_ZERO + 1 + (int)(at / DRAW_WINDOW) : DRAW_ZERO - 1 - (int)(at / DRAW_WINDOW), k = at % DRAW_WINDOW / 128;
        const double w = weight_of(tid << 15 | mag);
        s.count[run][tid ? k : 31 - k] = 1; s.mass[run][tid ? k : 31 - k] = w;
        if (w >= min_p) peer_add(&s.above, rank, 1u);
      }
    }
    for (int w = 0; w < DRAW_WINDOWS; ++w)
      if (seen >> w & 1) enter(w, true);
    cluster_sync();

    // ---- running sums within the runs ----
    for (int r = warp; r < DRAW_RUNS; r += DRAW_WARPS) {
      uint32_t n = s.count[r][lane];
      if (!__any_sync(0xffffffffu, n != 0)) continue;
      double m = s.mass[r][lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t nu = __shfl_up_sync(0xffffffffu, n, o);
        const double mu = __shfl_up_sync(0xffffffffu, m, o);
        if (lane >= o) { n += nu; m += mu; }
      }
      s.count[r][lane] = n; s.mass[r][lane] = m;
    }
    __syncthreads();
    // ---- the borders, by the first warp; the others wait for it to be done, or to want another window ----
    enum { COUNT, REACH, EXCEED };
    uint32_t n_run = 0, n = 0;           // of the runs up to this lane's; tokens kept so far
    double m_run = 0.0, mass = 0.0;      // their masses
    bool has_tokens = false;             // this lane's run
    if (warp == 0) {
      if (lane < DRAW_RUNS) { n_run = s.count[lane][31]; m_run = s.mass[lane][31]; }
      has_tokens = n_run != 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t nu = __shfl_up_sync(0xffffffffu, n_run, o);
        const double mu = __shfl_up_sync(0xffffffffu, m_run, o);
        if (lane >= o) { n_run += nu; m_run += mu; }
      }
      n = __shfl_sync(0xffffffffu, n_run, 31); mass = __shfl_sync(0xffffffffu, m_run, 31);
    }
    struct { uint32_t bits, taken, n; double mass, weight; } at = {0, 0, 0, 0.0, 0.0};   // value, how many of it, tokens and mass up to there
    auto crossed = [](int what, uint32_t count, double m, uint32_t want, double target) { return what == COUNT ? count >= want : what == REACH ? m >= target : m > target; };
    // The border that a number of tokens (COUNT) or a mass reaches (REACH) or exceeds (EXCEED): in `at` with -1 returned, or
    // the window that has to be resident; -2 where nothing reaches it. Run, binade, lane, value: of each the first one with tokens at
    // whose end the border is crossed: the tree adds up each end's masses in an order of its own, so that the sum at the end of an empty part may be
    // a rounding above its neighbours'. A sum may be a rounding apart from its parts' too, and then the last part has the border.
    auto border = [&](int what, uint32_t want, double target) -> int {
      auto first_of = [&](bool holds, bool there) {
        const uint32_t h = __ballot_sync(0xffffffffu, holds), t = __ballot_sync(0xffffffffu, there);
        return h ? __ffs(h) - 1 : 31 - __clz(t);
      };
      auto ahead_of = [&](uint32_t v, int i) { const uint32_t u = __shfl_sync(0xffffffffu, v, (i + 31) & 31); return i ? u : 0u; };
      auto mass_ahead_of = [&](double v, int i) { const double u = __shfl_sync(0xffffffffu, v, (i + 31) & 31); return i ? u : 0.0; };
      const uint32_t runs = __ballot_sync(0xffffffffu, has_tokens && crossed(what, n_run, m_run, want, target));
      if (!runs) return -2;
      const int run = __ffs(runs) - 1;
      uint32_t cn = ahead_of(n_run, run), c[4] = {0, 0, 0, 0};   // tokens and mass ahead of what has been narrowed down to
      double cm = mass_ahead_of(m_run, run), w[4] = {0.0, 0.0, 0.0, 0.0};
      int b = 0, d = 0;
      if (run == DRAW_ZERO) {
        c[0] = zeros; w[0] = weight_of(0);
      } else {
        const int neg = run > DRAW_ZERO, window = neg ? run - DRAW_ZERO - 1 : DRAW_ZERO - 1 - run;
        if (window != resident) return window;
        uint32_t ln = s.count[run][lane];
        double lm = s.mass[run][lane];
        uint32_t own = ln - (lane ? s.count[run][lane - 1] : 0);
        const int e = first_of(own && crossed(what, cn + ln, cm + lm, want, target), own != 0);
        cn += ahead_of(ln, e); cm += mass_ahead_of(lm, e);
        const int k = neg ? 32 + e : 31 - e, owner = k & (C - 1);
        ln = peer_get(&s.lane_count[k / C][lane], owner);
        lm = peer_get(&s.lane_mass[k / C][lane], owner);
        const double lw = peer_get(&s.lane_weight[k / C][lane], owner);
        const uint4 v = C > 2 ? peer_get4(&s.lane_counts[k / C][lane].x, owner) : in_order(k, counts(k));
        const int who = first_of((v.x | v.y | v.z | v.w) && crossed(what, cn + ln, cm + lm, want, target), (v.x | v.y | v.z | v.w) != 0);
        cn += ahead_of(ln, who); cm += mass_ahead_of(lm, who);
        c[0] = __shfl_sync(0xffffffffu, v.x, who); c[1] = __shfl_sync(0xffffffffu, v.y, who);
        c[2] = __shfl_sync(0xffffffffu, v.z, who); c[3] = __shfl_sync(0xffffffffu, v.w, who);
        b = first_bits(k, who); d = neg ? 1 : -1;
        weights(k, b, c, __shfl_sync(0xffffffffu, lw, who), w);
      }
      // the same in all lanes from here on
      uint32_t r, c_at = 0;
      double w_at = 0.0;
      int i_at = -1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (c[i] == 0) continue;
        if (i_at >= 0) {
          if (crossed(what, cn + c_at, cm + c_at * w_at, want, target)) continue;
          cn += c_at; cm += c_at * w_at;
        }
        i_at = i; c_at = c[i]; w_at = w[i];
      }
      if (what == COUNT) r = want - cn;
      else if (c_at == 1) r = 1;
      else {
        const double q = (target - cm) / w_at;   // how many of it, to a rounding (a weight of 0 has no border but by rounding)
        r = q >= 1.0 ? q < (double)c_at ? (uint32_t)q : c_at : 1;
        while (r > 1 && crossed(what, 0, cm + (r - 1) * w_at, 0, target)) --r;
        while (r < c_at && !crossed(what, 0, cm + r * w_at, 0, target)) ++r;
      }
      at.bits = b + i_at * d; at.taken = r; at.n = cn + r; at.mass = cm + r * w_at; at.weight = w_at;
      return -1;
    };
    const double unit = u01 < 0.f ? 0.0 : (double)u01;
    for (int stage = 0;;) {
      if (warp == 0) {
        int window = -1;
        for (; stage < 5; ++stage) {
          int what = COUNT;
          uint32_t want = 0;
          double target = 0.0;
          if (stage == 0) {              // top-k
            if (!(set.top_k > 0 && (uint32_t)set.top_k < n)) continue;
            want = set.top_k;
          } else if (stage == 1) {       // top-p of what top-k left
            if (!(set.top_p < 1.f)) continue;
            target = (double)set.top_p * mass;
            if (target > 0.0) what = REACH; else want = 1;
          } else if (stage == 2) {       // min-p
            want = max(s.above, 1u);
            if (!(set.min_p > 0.f && want < n)) continue;
          } else if (stage == 3) {
            if (!(unit < 1.0)) continue; // 1 and more, NaN: a rounding of a sum is not to decide
            what = EXCEED; target = unit * mass;
          } else {                       // the last one kept, also where no sum exceeds the target
            want = n;
          }
          window = border(what, want, target);
          if (window >= 0) break;        // this stage again, with that window
          if (stage < 3) { if (window == -1 && at.n < n) { n = at.n; mass = at.mass; } }
          else if (window == -1 && at.n <= n) break;
        }
        if (lane == 0) {
          s.window = window < 0 ? -1 : window;
          s.bits = at.bits; s.taken = at.taken; s.weight = at.weight; s.mass_kept = mass;
        }
      }
      __syncthreads();
      if (s.window < 0) break;
      enter(s.window, false);
      cluster_sync();
    }
    bits = s.bits; taken = s.taken;
  }

  // ---- the token: occurrence `taken` of the value, in order of index ----
  auto write = [&](uint32_t token) {
    const float logprob = empty ? -INFINITY : greedy ? 0.f : (float)log(s.weight / s.mass_kept);
    tokens[row_index] = token;
    if (logprobs) logprobs[row_index] = logprob;
    if (tokens_host) tokens_host[row_index] = token;
    if (logprobs_host) logprobs_host[row_index] = logprob;
  };
  const uint32_t key = bits * 0x10001u;
  auto matches = [&](const uint4& u, uint32_t (&m)[4]) {        // whether there are any
    m[0] = equal_bf162(u.x, key); m[1] = equal_bf162(u.y, key); m[2] = equal_bf162(u.z, key); m[3] = equal_bf162(u.w, key);
    return (m[0] | m[1] | m[2] | m[3]) != 0;
  };
  auto places = [](const uint32_t (&m)[4]) {                    // bit j: value j of the vector
    uint32_t mask = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) mask |= (m[j] & 1u) << (2 * j) | (m[j] >> 31) << (2 * j + 1);
    return mask;
  };
  // A drawn value's bins say which CTA has the occurrence, and where, if that CTA has no other one.
  const uint32_t place = (bits & 0x7FFFu) - (uint32_t)(DRAW_BASE0 + resident * DRAW_WINDOW);
  const bool binned = !greedy && !empty && bits != 0 && place < DRAW_WINDOW;
  uint32_t ahead = 0, mine = 0, m[4];
  if (binned) {
    const uint32_t* bin = &s.bins[(bits >> 15) * DRAW_SIDE + DRAW_LOW + place];
    const uint32_t own = *bin & count_mask;
    ahead = __reduce_add_sync(0xffffffffu, lane < rank ? peer_get(bin, lane) & count_mask : 0u);
    cluster_arrive();
    const bool here = taken > ahead && taken <= ahead + own, known = own == 1 && places_fit;
    if (here && known && tid == 0) {
      const int v = v0 + (int)(*bin >> DRAW_AT);
      matches(x.vec(v), m);
      write((uint32_t)(8 * v - x.shift + __ffs(places(m)) - 1));
    }
    if (!here || known) { cluster_wait(); return; }   // the last access to another CTA's shared memory lies ahead of its arrival
  }
  const int each = ((v1 - v0) + DRAW_WARPS - 1) / DRAW_WARPS;   // vectors of a warp, one after the other
  const int w0 = min(v1, v0 + warp * each), w1 = min(v1, w0 + each);
  if (!empty) x.each<32>(w0, w1, lane, [&](const uint4& u, int) { if (matches(u, m)) mine += __popc(places(m)); });
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) s.warp_a[warp] = mine;
  __syncthreads();
  if (binned) {
    cluster_wait();
  } else {
    if (tid < C) {
      uint32_t all = 0;
      for (int w = 0; w < DRAW_WARPS; ++w) all += s.warp_a[w];
      peer_put(&s.peer_match[rank], tid, all);
    }
    cluster_sync();                                              // and the last access to another CTA's shared memory lies ahead of it
    if (skip) return;
    if (empty) {
      if (rank == 0 && tid == 0) write(0);
      return;
    }
    for (int k = 0; k < rank; ++k) ahead += s.peer_match[k];
  }
  // The warp whose vectors have it, and then all threads on those, one each.
  if (taken <= ahead) return;            // another CTA's
  int owner = 0;
  while (owner < DRAW_WARPS && taken > ahead + s.warp_a[owner]) ahead += s.warp_a[owner++];
  if (owner == DRAW_WARPS) return;
  const int from = min(v1, v0 + owner * each), to = min(v1, from + each);
  uint32_t left = taken - ahead;                         // of the warp's
  for (int first = from; first < to; first += DRAW_THREADS) {
    const int v = first + tid;
    uint32_t mask = 0;
    if (v < to && matches(x.vec(v), m)) mask = places(m);
    const uint32_t own = __popc(mask);
    uint32_t upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    __syncthreads();                     // the last turn's sums have been read
    if (lane == 31) s.warp_b[warp] = upto;
    __syncthreads();
    uint32_t all = 0;
    for (int w = 0; w < DRAW_WARPS; ++w) {
      if (w == warp) upto += all;
      all += s.warp_b[w];
    }
    if (left <= upto && left > upto - own) {
      for (uint32_t k = left - (upto - own); k > 1; --k) mask &= mask - 1;
      write((uint32_t)(8 * v - x.shift + __ffs(mask) - 1));
    }
    if (left <= all) break;
    left -= all;
  }
}

template <int C, int RESIDENT>
cudaError_t draw_as(const bf16* logits, long long ld, int rows, int vocab, const DrawSetting* settings, const float* uniform, uint32_t* tokens,
                    float* logprobs, cudaStream_t s, uint32_t* tokens_host, float* logprobs_host, int skip_greedy) {
  static DeviceOnce configured;   // the attribute belongs to the device's copy of the kernel
  if (configured.first_on_current_device()) {
    cudaError_t e = cudaFuncSetAttribute(draw_rows_kernel<C, RESIDENT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(DrawShared<C, RESIDENT>));
    if (e != cudaSuccess) { configured.forget_current_device(); return e; }
  }
  return launch_k_cluster(C, draw_rows_kernel<C, RESIDENT>, dim3(rows * C), dim3(draw_threads(C, RESIDENT)), sizeof(DrawShared<C, RESIDENT>), s, logits, ld, vocab, settings, uniform,
                          tokens, logprobs, tokens_host, logprobs_host, skip_greedy);
}

}  // namespace

cudaError_t launch_draw_rows(const bf16* logits, long long ld, int rows, int vocab, const DrawSetting* settings, const float* uniform,
                             uint32_t* tokens, float* logprobs, int sm_count, cudaStream_t s, uint32_t* tokens_host, float* logprobs_host,
                             int skip_greedy) {
  if (rows <= 0) return cudaSuccess;
  // As many CTAs a row as the SMs hold at once, two on each, and two where the rows are more: then three CTAs an SM. Rows of 128256 with 2, 4 and
  // 8 CTAs each: one row 17.6, 13.9 and 11.5 us; 192 rows 36.7, 49 and 95. Two and three CTAs an SM: 128 rows 24.5 and 26.4, 192 36.7 and 31.7, 300
  // of 50001 39.6 and 34.2, 512 of 256000 107 and 102.
  const int room = 2 * sm_count / rows;
  auto as = room >= 8 ? draw_as<8, 2> : room >= 4 ? draw_as<4, 2> : room >= 2 ? draw_as<2, 2> : draw_as<2, 3>;
  return as(logits, ld, rows, vocab, settings, uniform, tokens, logprobs, s, tokens_host, logprobs_host, skip_greedy);
}

}  // namespace kc
