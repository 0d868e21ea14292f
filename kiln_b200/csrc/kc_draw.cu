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
// Counting: a bin a value, of the magnitudes [2^-24, 2^8) of either sign (the home window), 32 KB of shared memory. A row with
// other magnitudes takes another pass over itself for each of the eight other windows of 32 binary orders that it has values in, so that
// any row is exact; zeros are counted apart. 32 neighbouring values are a group; the groups' counts and masses lie in
// shared memory of every CTA of the row's cluster, which then all look for the same borders.
#include "kc_fused.cuh"
#include "kc_umma.cuh"

namespace kc {

namespace {

constexpr int DRAW_THREADS = 512, DRAW_WARPS = DRAW_THREADS / 32;
constexpr int DRAW_WINDOW = 4096;                 // magnitudes (bf16 without the sign) of a window, one bin each and sign
constexpr int DRAW_HOME = 4;                      // the window that holds a language model's logits: magnitudes 2^-24 to 2^8
constexpr int DRAW_BASE0 = 103 * 128 - DRAW_HOME * DRAW_WINDOW;   // first magnitude of window 0 (below zero: it is a short one)
constexpr int DRAW_WINDOWS = 9;
constexpr int DRAW_GROUPS = 2048;                 // of 32 values in falling order: 1024 positive, zero, 1020 negative
constexpr int DRAW_ZERO = 1024;                   // the group of zero, which is one value
constexpr uint32_t BF16_INF = 0x7F80u;
static_assert(DRAW_BASE0 % 32 == 0 && DRAW_BASE0 + DRAW_WINDOWS * DRAW_WINDOW > 0x7F80, "windows cover all magnitudes in whole groups");

struct DrawShared {
  uint32_t bins[2 * DRAW_WINDOW];                 // [sign][magnitude]: how often the value occurs in this CTA's part of the row
  double mass[DRAW_GROUPS];
  uint32_t count[DRAW_GROUPS], above[DRAW_GROUPS];   // above: of those of w >= min_p
  uint32_t peer_top[8], peer_seen[8], peer_zeros[8], peer_match[8];   // what each CTA of the cluster found
  uint32_t warp_a[DRAW_WARPS], warp_b[DRAW_WARPS], warp_c[DRAW_WARPS];
  double warp_m[DRAW_WARPS];
  int found;                                      // group that holds a border
  uint32_t before; double mass_before;            // ahead of it
  uint32_t bits, taken, n; double border_mass, weight;   // a border: value, how many of it, tokens and mass up to there
};

__device__ __forceinline__ void peer_put(uint32_t* p, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(cluster_addr(smem_u32(p), rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void peer_put(double* p, uint32_t rank, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(cluster_addr(smem_u32(p), rank)), "d"(v) : "memory");
}
__device__ __forceinline__ uint32_t peer_get(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ float value_of(uint32_t bits) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ uint32_t top_bf162(uint32_t a, uint32_t b) {   // a NaN gives way to a number
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// A row as vectors of eight values on 16-byte boundaries: the first and the last one may hang over, and have -inf there.
struct DrawRow {
  const bf16* row;
  int vocab, shift;                               // the row starts at value `shift` of vector 0
  __device__ __forceinline__ uint4 vec(int v) const {
    const int e = 8 * v - shift;
    if (e >= 0 && e + 8 <= vocab) return *reinterpret_cast<const uint4*>(row + e);
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = e + 2 * k;
      const uint32_t a = i >= 0 && i < vocab ? reinterpret_cast<const unsigned short*>(row)[i] : 0xFF80u;
      const uint32_t b = i + 1 >= 0 && i + 1 < vocab ? reinterpret_cast<const unsigned short*>(row)[i + 1] : 0xFF80u;
      w[k] = a | b << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// C: CTAs of a row's cluster.
template <int C>
__global__ void __launch_bounds__(DRAW_THREADS, 2)
draw_rows_kernel(const bf16* __restrict__ logits, long long ld, int vocab, const DrawSetting* __restrict__ settings,
                 const float* __restrict__ uniform, uint32_t* __restrict__ tokens, float* __restrict__ logprobs,
                 uint32_t* __restrict__ tokens_host, float* __restrict__ logprobs_host, int skip_greedy) {
  extern __shared__ __align__(16) uint8_t draw_smem[];
  DrawShared& s = *reinterpret_cast<DrawShared*>(draw_smem);
  pdl_launch_dependents();
  if (C > 1) cluster_arrive();           // waited for before the first access to another CTA's shared memory: it has started by then
  const int row_index = blockIdx.x / C, rank = blockIdx.x % C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto meet = [&]() { if (C > 1) cluster_sync(); else __syncthreads(); };
  for (int i = tid; i < 2 * DRAW_WINDOW / 4; i += DRAW_THREADS) reinterpret_cast<uint4*>(s.bins)[i] = make_uint4(0, 0, 0, 0);
  for (int i = tid; i < DRAW_GROUPS; i += DRAW_THREADS) { s.mass[i] = 0.0; s.count[i] = 0; s.above[i] = 0; }
  if (C > 1) cluster_wait(); else __syncthreads();
  pdl_wait();
  const DrawSetting set = settings[row_index];
  const float u01 = uniform[row_index];
  const bool greedy = !(set.temperature > 0.f);
  const bool skip = greedy && skip_greedy;

  DrawRow x;
  x.row = logits + (size_t)row_index * ld;
  x.vocab = vocab;
  x.shift = (int)(reinterpret_cast<uintptr_t>(x.row) & 15) / 2;
  const int vecs = (x.shift + vocab + 7) / 8, per = (vecs + C - 1) / C;
  const int v0 = min(vecs, rank * per), v1 = skip ? v0 : min(vecs, v0 + per);

  // ---- pass over the row: bins of the home window, the maximum, which other windows it has values in ----
  uint32_t top = 0xFF80FF80u, seen = 0, zeros = 0;
  auto tally = [&](uint32_t b) {
    const uint32_t mag = b & 0x7FFFu, off = mag - (DRAW_BASE0 + DRAW_HOME * DRAW_WINDOW);
    if (off < DRAW_WINDOW) atomicAdd(&s.bins[off + ((b & 0x8000u) >> 3)], 1u);
    else if (mag == 0) ++zeros;
    else if (mag < BF16_INF || b == BF16_INF) seen |= 1u << ((mag - DRAW_BASE0) / DRAW_WINDOW);
  };
  constexpr int UNROLL = 4;
  for (int v = v0 + tid; v < v1; v += DRAW_THREADS * UNROLL) {
    uint4 u[UNROLL];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k)
      if (v + k * DRAW_THREADS < v1) u[k] = x.vec(v + k * DRAW_THREADS);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k)
      if (v + k * DRAW_THREADS < v1) {
        const uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          top = top_bf162(top, w[j]);
          if (!greedy) { tally(w[j] & 0xFFFFu); tally(w[j] >> 16); }
        }
      }
  }
  {
    const float2 two = unpack_bf162(top);
    const float m = warp_max(fmaxf(two.x, two.y));
    seen = __reduce_or_sync(0xffffffffu, seen);
    zeros = __reduce_add_sync(0xffffffffu, zeros);
    if (lane == 0) { s.warp_a[warp] = __float_as_uint(m); s.warp_b[warp] = seen; s.warp_c[warp] = zeros; }
  }
  __syncthreads();
  if (tid < C) {
    float m = -INFINITY;
    seen = zeros = 0;
    for (int w = 0; w < DRAW_WARPS; ++w) { m = fmaxf(m, __uint_as_float(s.warp_a[w])); seen |= s.warp_b[w]; zeros += s.warp_c[w]; }
    peer_put(&s.peer_top[rank], tid, __float_as_uint(m));
    peer_put(&s.peer_seen[rank], tid, seen);
    peer_put(&s.peer_zeros[rank], tid, zeros);
  }
  meet();
  float largest = -INFINITY;
  seen = zeros = 0;
#pragma unroll
  for (int k = 0; k < C; ++k) { largest = fmaxf(largest, __uint_as_float(s.peer_top[k])); seen |= s.peer_seen[k]; zeros += s.peer_zeros[k]; }
  largest += 0.f;                        // -0 is +0
  // From here on every branch that holds a barrier is taken by the whole cluster: what it hangs on is the same in all its CTAs.
  const bool empty = largest == -INFINITY;   // nothing but masked tokens and NaN: token 0
  uint32_t bits = __float_as_uint(largest) >> 16, taken = 1;
  double weight = 1.0, mass = 1.0;

  if (!greedy && !empty) {
    const double inv_t = 1.0 / (double)set.temperature, top_value = largest, min_p = set.min_p;
    auto weight_of = [&](uint32_t b) {
      const float l = value_of(b);
      return l == largest ? 1.0 : largest == INFINITY ? 0.0 : exp(((double)l - top_value) * inv_t);
    };
    constexpr int OWN = 256 / C;         // groups of a window that this CTA adds up
    int resident = DRAW_HOME;
    // Adds the cluster's bins of the resident window and enters its groups into every CTA's totals.
    auto account = [&]() {
      const int base = DRAW_BASE0 + resident * DRAW_WINDOW;
      for (int q = rank * OWN + warp; q < (rank + 1) * OWN; q += DRAW_WARPS) {
        const int neg = q >> 7, off = (q & 127) * 32 + (neg ? lane : 31 - lane), bin = neg * DRAW_WINDOW + off;
        uint32_t c = 0;
        if (C == 1) c = s.bins[bin];
        else
#pragma unroll
          for (int k = 0; k < C; ++k) c += peer_get(&s.bins[bin], k);
        if (!__any_sync(0xffffffffu, c != 0)) continue;
        if (C > 1) s.bins[bin] = c;      // no other CTA reads these bins of this one before the next barrier
        const int mag = base + off;
        const double w = c ? weight_of((uint32_t)mag | neg << 15) : 0.0;
        double m = c * w;
        const uint32_t above = __reduce_add_sync(0xffffffffu, c && w >= min_p ? c : 0);
        c = __reduce_add_sync(0xffffffffu, c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
        const int g = neg ? DRAW_ZERO + 1 + (mag >> 5) : DRAW_ZERO - 1 - (mag >> 5);
        if (lane < C) { peer_put(&s.count[g], lane, c); peer_put(&s.above[g], lane, above); peer_put(&s.mass[g], lane, m); }
      }
    };
    // Makes another window the resident one: a pass over the row for its bins.
    auto enter = [&](int window) {
      meet();                            // the bins have been read
      for (int i = tid; i < 2 * DRAW_WINDOW / 4; i += DRAW_THREADS) reinterpret_cast<uint4*>(s.bins)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      resident = window;
      const uint32_t base = DRAW_BASE0 + window * DRAW_WINDOW;
      for (int v = v0 + tid; v < v1; v += DRAW_THREADS) {
        const uint4 u = x.vec(v);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t b = (w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu, mag = b & 0x7FFFu;
          if (mag - base < DRAW_WINDOW && mag != 0 && (mag < BF16_INF || b == BF16_INF)) atomicAdd(&s.bins[mag - base + ((b & 0x8000u) >> 3)], 1u);
        }
      }
      meet();
      account();
    };
    account();
    if (tid == 0 && zeros) {
      const double w = weight_of(0);
      s.count[DRAW_ZERO] = zeros; s.above[DRAW_ZERO] = w >= min_p ? zeros : 0; s.mass[DRAW_ZERO] = zeros * w;
    }
    for (int w = 0; w < DRAW_WINDOWS; ++w)
      if (seen >> w & 1) enter(w);
    meet();

    // ---- running sums over the groups: this thread's are the four from 4 tid on ----
    uint32_t n_before = 0, above_all = 0, tokens_all;
    double m_before = 0.0, mass_all;
    {
      uint32_t c = 0, a = 0;
      double m = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) { c += s.count[4 * tid + i]; a += s.above[4 * tid + i]; m += s.mass[4 * tid + i]; }
      uint32_t ci = c;
      double mi = m;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t cu = __shfl_up_sync(0xffffffffu, ci, o);
        const double mu = __shfl_up_sync(0xffffffffu, mi, o);
        if (lane >= o) { ci += cu; mi += mu; }
      }
      a = __reduce_add_sync(0xffffffffu, a);
      if (lane == 31) { s.warp_a[warp] = ci; s.warp_b[warp] = a; s.warp_m[warp] = mi; }
      __syncthreads();
      tokens_all = 0; mass_all = 0.0;
      for (int w = 0; w < DRAW_WARPS; ++w) {
        if (w == warp) { n_before = tokens_all; m_before = mass_all; }
        tokens_all += s.warp_a[w]; above_all += s.warp_b[w]; mass_all += s.warp_m[w];
      }
      const uint32_t cu = __shfl_up_sync(0xffffffffu, ci, 1);
      const double mu = __shfl_up_sync(0xffffffffu, mi, 1);
      if (lane > 0) { n_before += cu; m_before += mu; }
    }

    // The border that a number of tokens (COUNT) or a mass reaches (REACH) or exceeds (EXCEED): left in s; false where none does.
    enum { COUNT, REACH, EXCEED };
    auto crossed = [](int what, uint32_t n, double m, uint32_t want, double target) { return what == COUNT ? n >= want : what == REACH ? m >= target : m > target; };
    auto border = [&](int what, uint32_t want, double target) {
      __syncthreads();                   // the last border has been read
      if (tid == 0) s.found = DRAW_GROUPS;
      __syncthreads();
      uint32_t n = n_before;
      double m = m_before;
      int mine = DRAW_GROUPS;
      uint32_t mine_n = 0;
      double mine_m = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t c = s.count[4 * tid + i];
        const double g = s.mass[4 * tid + i];
        if (mine == DRAW_GROUPS && c && crossed(what, n + c, m + g, want, target)) { mine = 4 * tid + i; mine_n = n; mine_m = m; }
        n += c; m += g;
      }
      const int first = __reduce_min_sync(0xffffffffu, mine);
      if (lane == 0 && first < DRAW_GROUPS) atomicMin(&s.found, first);
      __syncthreads();
      const int g = s.found;
      if (g == DRAW_GROUPS) return false;
      if (mine == g) { s.before = mine_n; s.mass_before = mine_m; }
      const int neg = g > DRAW_ZERO, mag0 = neg ? (g - DRAW_ZERO - 1) * 32 : (DRAW_ZERO - 1 - g) * 32;
      if (g != DRAW_ZERO && (mag0 - DRAW_BASE0) / DRAW_WINDOW != resident) { enter((mag0 - DRAW_BASE0) / DRAW_WINDOW); meet(); }
      __syncthreads();
      if (warp == 0) {
        uint32_t c, b;                   // of this lane's value
        if (g == DRAW_ZERO) {
          c = lane == 0 ? zeros : 0;
          b = 0;
        } else {
          const int off0 = mag0 - (DRAW_BASE0 + resident * DRAW_WINDOW), q = neg * 128 + off0 / 32, in = neg ? lane : 31 - lane;
          c = C == 1 ? s.bins[neg * DRAW_WINDOW + off0 + in] : peer_get(&s.bins[neg * DRAW_WINDOW + off0 + in], q / OWN);
          b = (uint32_t)(mag0 + in) | neg << 15;
        }
        const double w = c ? weight_of(b) : 0.0;
        uint32_t ci = c;
        double mi = c * w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t cu = __shfl_up_sync(0xffffffffu, ci, o);
          const double mu = __shfl_up_sync(0xffffffffu, mi, o);
          if (lane >= o) { ci += cu; mi += mu; }
        }
        double m_ex = __shfl_up_sync(0xffffffffu, mi, 1);
        if (lane == 0) m_ex = 0.0;
        const uint32_t cn = s.before + ci - c;            // tokens and mass ahead of this lane's value
        const double cm = s.mass_before + m_ex;
        // The group's sum may be a rounding apart from its values': then the last one has the border.
        const uint32_t holds = __ballot_sync(0xffffffffu, c && crossed(what, cn + c, cm + c * w, want, target));
        const uint32_t there = __ballot_sync(0xffffffffu, c != 0);
        if (lane == (holds ? __ffs(holds) - 1 : 31 - __clz(there))) {
          uint32_t r;
          if (what == COUNT) r = want - cn;
          else {
            const double d = (target - cm) / w;           // how many of it, to a rounding (w = 0 has no border but by rounding)
            r = d >= 1.0 ? d < (double)c ? (uint32_t)d : c : 1;
            while (r > 1 && crossed(what, 0, cm + (r - 1) * w, 0, target)) --r;
            while (r < c && !crossed(what, 0, cm + r * w, 0, target)) ++r;
          }
          s.bits = b; s.taken = r; s.n = cn + r; s.border_mass = cm + r * w; s.weight = w;
        }
      }
      __syncthreads();
      return true;
    };

    uint32_t n = tokens_all;
    mass = mass_all;
    if (set.top_k > 0 && (uint32_t)set.top_k < n) {
      n = set.top_k;
      border(COUNT, n, 0.0);
      mass = s.border_mass;
    }
    if (set.top_p < 1.f && border(REACH, 0, (double)set.top_p * mass) && s.n < n) { n = s.n; mass = s.border_mass; }
    if (set.min_p > 0.f && max(above_all, 1u) < n) {
      n = max(above_all, 1u);
      border(COUNT, n, 0.0);
      mass = s.border_mass;
    }
    if (!border(EXCEED, 0, (double)u01 * mass) || s.n > n) border(COUNT, n, 0.0);   // u of 1 and more, NaN: the last one kept
    bits = s.bits; taken = s.taken; weight = s.weight;
  }

  // ---- the token: occurrence `taken` of the value, in order of index ----
  const int each = ((v1 - v0) + DRAW_WARPS - 1) / DRAW_WARPS;   // vectors of a warp, one after the other
  const int w0 = min(v1, v0 + warp * each), w1 = min(v1, w0 + each);
  auto matches = [&](int v) -> uint32_t {                // bit j: value j of the vector
    const uint4 u = x.vec(v);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t mask = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = (w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu;
      if (bits == 0 ? (b & 0x7FFFu) == 0 : b == bits) mask |= 1u << j;
    }
    return mask;
  };
  uint32_t mine = 0;
  if (!empty)
    for (int v = w0 + lane; v < w1; v += 32) mine += __popc(matches(v));
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) s.warp_a[warp] = mine;
  __syncthreads();
  if (tid < C) {
    uint32_t all = 0;
    for (int w = 0; w < DRAW_WARPS; ++w) all += s.warp_a[w];
    peer_put(&s.peer_match[rank], tid, all);
  }
  meet();                                                // and the last access to another CTA's shared memory lies ahead of it
  uint32_t ahead = 0;
  for (int k = 0; k < rank; ++k) ahead += s.peer_match[k];
  for (int w = 0; w < warp; ++w) ahead += s.warp_a[w];
  const float logprob = empty ? -INFINITY : greedy ? 0.f : (float)log(weight / mass);
  auto write = [&](uint32_t token) {
    tokens[row_index] = token;
    if (logprobs) logprobs[row_index] = logprob;
    if (tokens_host) tokens_host[row_index] = token;
    if (logprobs_host) logprobs_host[row_index] = logprob;
  };
  if (skip) return;
  if (empty) {
    if (rank == 0 && tid == 0) write(0);
  } else if (taken > ahead && taken <= ahead + mine) {
    uint32_t left = taken - ahead;                       // of the warp's
    for (int v = w0; v < w1; v += 32) {
      const uint32_t mask = v + lane < w1 ? matches(v + lane) : 0, own = __popc(mask);
      uint32_t upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      if (left <= upto && left > upto - own) {
        uint32_t m = mask;
        for (uint32_t k = left - (upto - own); k > 1; --k) m &= m - 1;
        write((uint32_t)(8 * (v + lane) - x.shift + __ffs(m) - 1));
      }
      const uint32_t all = __shfl_sync(0xffffffffu, upto, 31);
      if (left <= all) break;
      left -= all;
    }
  }
}

template <int C>
cudaError_t draw_as(const bf16* logits, long long ld, int rows, int vocab, const DrawSetting* settings, const float* uniform, uint32_t* tokens,
                    float* logprobs, cudaStream_t s, uint32_t* tokens_host, float* logprobs_host, int skip_greedy) {
  static DeviceOnce configured;   // the attribute belongs to the device's copy of the kernel
  if (configured.first_on_current_device()) {
    cudaError_t e = cudaFuncSetAttribute(draw_rows_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(DrawShared));
    if (e != cudaSuccess) { configured.forget_current_device(); return e; }
  }
  return launch_k_cluster(C, draw_rows_kernel<C>, dim3(rows * C), dim3(DRAW_THREADS), sizeof(DrawShared), s, logits, ld, vocab, settings, uniform,
                          tokens, logprobs, tokens_host, logprobs_host, skip_greedy);
}

}  // namespace

cudaError_t launch_draw_rows(const bf16* logits, long long ld, int rows, int vocab, const DrawSetting* settings, const float* uniform,
                             uint32_t* tokens, float* logprobs, int sm_count, cudaStream_t s, uint32_t* tokens_host, float* logprobs_host,
                             int skip_greedy) {
  if (rows <= 0) return cudaSuccess;
  // As many CTAs a row as the SMs hold at once, two on each.
  const int room = 2 * sm_count / rows;
  auto as = room >= 8 ? draw_as<8> : room >= 4 ? draw_as<4> : room >= 2 ? draw_as<2> : draw_as<1>;
  return as(logits, ld, rows, vocab, settings, uniform, tokens, logprobs, s, tokens_host, logprobs_host, skip_greedy);
}

}  // namespace kc
