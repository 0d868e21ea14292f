// What low-rank adapters add to a projection's rows: out_i = y_i + s_a B_a (A_a x_i), a the adapter of row i.
//
// One launch. Rows are grouped by adapter on the host (kc_adapter_rows_create) into tiles of at most 16, and a tile is a cluster's
// of two to eight CTAs: each multiplies its share of the features of x with A's columns, the partial t = A x [rows, rank] meet
// in the cluster's shared memory, and each CTA takes its share of the projection's features through B and adds them to y. So t
// never goes through memory, and no workspace or order of atomics is involved.
//
// Both products are mma.sync m16n8k16, which takes its operands from registers as they come from memory. The contraction's order is
// free, so a lane's elements of an operand are neighbours: 16-byte loads of x and A, 8 to 32 bytes of B; and the columns of B
// are dealt so that a lane has eight neighbouring features of y.
//
// t is summed in fp32, multiplied by s and rounded to bf16 for the second product, as a model's activations are between two
// projections: with what that leaves as a second bf16 number the result was 0.1 of its own rounding nearer, for twice the instructions
// of the product (2048 rows of rank 64: 118 -> 94 us without). y is added in fp32 and the result rounded once.
//
// What bounds it. Few rows: launch, two latencies of memory and two exchanges, 4.8 us; 32 rows of an adapter each into 28672 features
// read 29 MB of B in 12.5 us, of which 5.7 are memory's. Many rows: the 16 rows of a tile share what they read of B, so that
// L1 sees four times y; 2048 rows of rank 64 into 28672 features take 88 us, 44 at a copy's rate. Tiles of 32 and 64 rows with B and y
// through a ring of shared memory took 74 and 110 us there, but the smaller of them 61 for 46 from 14336 to 4096 features, 58 for 49 at
// 1024 rows and 37 for 24 at 256: how many clusters the SMs hold at once weighs more than what is read of B. Every slot costs
// the ranks of the bank's stride: rank 8 or 16 into 28672 features for 32 adapters 9.4 us from L2, 27 in a bank of rank 64.
#include "kc_lora.cuh"

#include "kc_umma.cuh"

namespace kc {

namespace {

constexpr int LORA_THREADS = 256, LORA_WARPS = 8;

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float peer_float(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ void peer_put(bf16* p, uint32_t rank, bf16 v) {
  asm volatile("st.shared::cluster.b16 [%0], %1;" ::"r"(cluster_addr(smem_u32(p), rank)), "h"(__bfloat16_as_ushort(v)) : "memory");
}

// N registers (2, 4 or 8) from memory on a boundary of their size.
template <int N>
__device__ __forceinline__ void load_regs(uint32_t* r, const void* from) {
  if constexpr (N == 8) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "l"(from) : "memory");
  } else if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(from);
    r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(from);
    r[0] = v.x; r[1] = v.y;
  }
}

// A kernel's shape: CTAs of a cluster, and R, the ranks as they are stored.
template <int CTAS_, int R_>
struct LoraShape {
  static constexpr int CTAS = CTAS_, R = R_, ROWS = LORA_TILE;
  static constexpr int PARTS = (7 + CTAS) / CTAS;  // eighths of the features of x that a CTA has, at the most
  static constexpr int RS = R < 64 ? R : 64;       // ranks of a step of the first product
  static constexpr int PAD = R + 8;                // of a row of t: 16-byte pieces of neighbouring rows lie in different banks
  static constexpr int PART = RS + 4;
  static constexpr int W = R / 8;                  // registers of a lane's quarter of the ranks
  // Rounds (32 features a warp) that a warp has B and y of, and as many on their way; CTAs of an SM: what 65536 registers hold.
  static constexpr int U = R <= 32 ? 2 : 1;
  static constexpr int RESIDENT = R <= 64 ? 2 : 1;
  // Shared memory of a CTA: partial sums of its warps for a step [8][ROWS][PART], its parts' t [PARTS][ROWS][R], the cluster's t [ROWS][PAD].
  static constexpr size_t SMEM = ((size_t)LORA_WARPS * ROWS * PART + (size_t)PARTS * ROWS * R) * 4 + (size_t)ROWS * PAD * 2;
  static_assert(SMEM <= 227 * 1024 / RESIDENT - 1024, "shared memory");
};

// VEC: rows of y and out start on 16-byte boundaries.
template <typename S, bool VEC>
__global__ void __launch_bounds__(LORA_THREADS, S::RESIDENT)
lora_kernel(const LoraParams p) {
  constexpr int R = S::R, RS = S::RS, NB = RS / 8, PAD = S::PAD, PART = S::PART, W = S::W, U = S::U, ROWS = S::ROWS, CTAS = S::CTAS, PARTS = S::PARTS;
  extern __shared__ __align__(16) uint8_t lora_smem[];
  float* part = reinterpret_cast<float*>(lora_smem);
  float* sum = part + LORA_WARPS * ROWS * PART;
  bf16* ts = reinterpret_cast<bf16*>(sum + PARTS * ROWS * R);
  __shared__ int rows[ROWS];
  pdl_launch_dependents();
  cluster_arrive();                    // waited for before the first access to another CTA's shared memory: it has started by then
  const int rank = blockIdx.x % CTAS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();
  const LoraTile tile = p.tiles[blockIdx.x / CTAS];
  const LoraSlot slot = tile.slot >= 0 ? p.slots[tile.slot] : LoraSlot{0, 0.f};
  if (threadIdx.x < ROWS) rows[threadIdx.x] = p.rows[tile.first + min((int)threadIdx.x, tile.n - 1)];
  __syncthreads();
  cluster_wait();
  const int blocks = (p.n_out + 31) / 32, b0 = (int)((long long)blocks * rank / CTAS), b1 = (int)((long long)blocks * (rank + 1) / CTAS);

  if (slot.rank == 0) {                // no adapter: the rows as they are
    if (p.out != p.y) {
      const int f0 = b0 * 32, f1 = min(p.n_out, b1 * 32);
      for (int r = warp; r < tile.n; r += LORA_WARPS) {
        const size_t at = (size_t)rows[r] * p.n_out;
        if (VEC) for (int f = f0 + lane * 8; f < f1; f += 256) *reinterpret_cast<uint4*>(p.out + at + f) = *reinterpret_cast<const uint4*>(p.y + at + f);
        else for (int f = f0 + lane; f < f1; f += 32) p.out[at + f] = p.y[at + f];
      }
    }
    return;                            // all CTAs of the cluster
  }

  // ---- what a warp needs of B and y for 32 features. Column 2 t' + e of column block j is feature 8 t' + 2 j + e, so that a lane's
  // columns are eight neighbours; its ranks are a quarter of them, the t-th ----
  const size_t y_at[2] = {(size_t)rows[g] * p.n_out + t * 8, (size_t)rows[g + 8] * p.n_out + t * 8};
  const bf16* bank = p.b + (size_t)tile.slot * p.n_out * R + t * (R / 4);
  struct Block { uint32_t w[4][W], y[2][4]; };
  auto load = [&](Block& b, int blk) {
    if (blk >= b1) return;
    if constexpr (VEC) {
      if (blk * 32 + t * 8 < p.n_out) {
        if (g < tile.n) load_regs<4>(b.y[0], p.y + y_at[0] + blk * 32);
        if (g + 8 < tile.n) load_regs<4>(b.y[1], p.y + y_at[1] + blk * 32);
      }
    }
    const int feature = blk * 32 + (g >> 1) * 8 + (g & 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16* from = bank + (size_t)min(feature + 2 * j, p.n_out - 1) * R;
      if constexpr (W == 16) { load_regs<8>(b.w[j], from); load_regs<8>(b.w[j] + 8, from + 16); }
      else load_regs<W>(b.w[j], from);
    }
  };
  Block cur[U];
  auto load_first = [&]() {
#pragma unroll
    for (int i = 0; i < U; ++i) load(cur[i], b0 + warp + i * LORA_WARPS);
  };
  constexpr bool EARLY = R == 16;      // under the first product already, where the registers are there
  if (EARLY) load_first();

  // ---- t = A x over this CTA's parts of the features, an eighth of a part a warp. The parts are the same for every size of cluster,
  // so that a row's bits do not hang on it ----
  {
    const int chunks = p.n_in / 32, used = (slot.rank + RS - 1) / RS;   // steps of ranks in use
    const bf16 *x0 = p.x + (size_t)rows[g] * p.n_in + t * 8, *x1 = p.x + (size_t)rows[g + 8] * p.n_in + t * 8;
    const int part0 = rank * 8 / CTAS, part1 = (rank + 1) * 8 / CTAS;
    for (int i = 0; i < part1 - part0; ++i) {
      const int me = (part0 + i) * LORA_WARPS + warp;
      const int c0 = (int)((long long)chunks * me / (8 * LORA_WARPS)), c1 = (int)((long long)chunks * (me + 1) / (8 * LORA_WARPS));
      for (int s = 0; s < used; ++s) {
        const bf16* a = p.a + ((size_t)tile.slot * R + s * RS + g) * p.n_in + t * 8;
        float acc[NB][4] = {};
#pragma unroll 2
        for (int c = c0; c < c1; ++c) {
          uint4 w[NB];
#pragma unroll
          for (int j = 0; j < NB; ++j) w[j] = *reinterpret_cast<const uint4*>(a + (size_t)j * 8 * p.n_in + (size_t)c * 32);
          const uint4 u0 = *reinterpret_cast<const uint4*>(x0 + (size_t)c * 32), u1 = *reinterpret_cast<const uint4*>(x1 + (size_t)c * 32);
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            mma_bf16(acc[j], u0.x, u1.x, u0.y, u1.y, w[j].x, w[j].y);
            mma_bf16(acc[j], u0.z, u1.z, u0.w, u1.w, w[j].z, w[j].w);
          }
        }
        if (i + s > 0) __syncthreads();   // the last partial sums have been read
        float* to = part + (warp * ROWS + g) * PART + t * 2;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          *reinterpret_cast<float2*>(to + j * 8) = make_float2(acc[j][0], acc[j][1]);
          *reinterpret_cast<float2*>(to + 8 * PART + j * 8) = make_float2(acc[j][2], acc[j][3]);
        }
        __syncthreads();
        for (int k = threadIdx.x; k < tile.n * RS; k += LORA_THREADS) {
          const int row = k / RS, r = k % RS;
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < LORA_WARPS; ++w) v += part[(w * ROWS + row) * PART + r];
          sum[(i * ROWS + row) * R + s * RS + r] = v;
        }
      }
    }
  }
  cluster_sync();
  if (!EARLY) load_first();            // they arrive under the exchange
  // ---- the cluster's t, in the order of its parts, rounded to bf16; ranks past the adapter's own are zero, whatever x holds. Of
  // many values each CTA adds up its share and hands it to all, of few every CTA all of them ----
  {
    const int items = tile.n * R;
    const bool shared = items > 1024;
    const int from = shared ? items * rank / CTAS : 0, to = shared ? items * (rank + 1) / CTAS : items;
    for (int i = from + threadIdx.x; i < to; i += LORA_THREADS) {
      const int row = i / R, r = i % R;
      float v = 0.f;
      if (r < slot.rank) {
        float q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int owner = ((k + 1) * CTAS - 1) / 8;
          q[k] = peer_float(&sum[((k - owner * 8 / CTAS) * ROWS + row) * R + r], owner);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) v += q[k];
        v *= slot.scale;
      }
      const bf16 b = __float2bfloat16_rn(v);
      if (!shared) { ts[row * PAD + r] = b; continue; }
#pragma unroll
      for (int k = 0; k < CTAS; ++k) peer_put(&ts[row * PAD + r], k, b);
    }
  }
  cluster_sync();                      // also: no CTA leaves while another one reads its sums

  // ---- out = y + B t: t stays in registers ----
  uint32_t v[2][W];                    // [row][ranks]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bf16* from = ts + (h * 8 + g) * PAD + t * (R / 4);
#pragma unroll
    for (int k = 0; k < W; k += 2) {
      const uint2 q = *reinterpret_cast<const uint2*>(from + 2 * k);
      v[h][k] = q.x; v[h][k + 1] = q.y;
    }
  }
#pragma unroll 1
  for (int blk = b0 + warp; blk < b1; blk += LORA_WARPS * U) {
    Block next[U];
#pragma unroll
    for (int i = 0; i < U; ++i) load(next[i], blk + (U + i) * LORA_WARPS);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int at = blk + i * LORA_WARPS, mine = at * 32 + t * 8;
      if (at < b1) {
        float acc[4][4] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < W; k += 2) mma_bf16(acc[j], v[0][k], v[1][k], v[0][k + 1], v[1][k + 1], cur[i].w[j][k], cur[i].w[j][k + 1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h * 8 + g >= tile.n || mine >= p.n_out) continue;
          bf16* to = p.out + y_at[h] + (size_t)at * 32;
          if constexpr (VEC) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = unpack_bf162(cur[i].y[h][j]);
              o[j] = pack_bf162(f.x + acc[j][2 * h], f.y + acc[j][2 * h + 1]);
            }
            *reinterpret_cast<uint4*>(to) = make_uint4(o[0], o[1], o[2], o[3]);
          } else {
            const bf16* from = p.y + y_at[h] + (size_t)at * 32;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (mine + e < p.n_out) to[e] = __float2bfloat16_rn(__bfloat162float(from[e]) + acc[e >> 1][2 * h + (e & 1)]);
          }
        }
      }
      cur[i] = next[i];
    }
  }
}

template <typename S>
cudaError_t launch(const LoraParams& p, cudaStream_t s) {
  const bool vec = p.n_out % 8 == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  auto as = [&](auto kernel, DeviceOnce& configured) {   // the attribute belongs to the device's copy of the kernel
    if (configured.first_on_current_device()) {
      cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
      if (e != cudaSuccess) { configured.forget_current_device(); return e; }
    }
    return launch_k_cluster(S::CTAS, kernel, dim3(p.n_tiles * S::CTAS), dim3(LORA_THREADS), S::SMEM, s, p);
  };
  static DeviceOnce with_vec, without;
  return vec ? as(lora_kernel<S, true>, with_vec) : as(lora_kernel<S, false>, without);
}

// The largest clusters of which the SMs hold all at once (a cluster lies in one group of SMs: of 296 places for CTAs clusters of eight
// take 256, of seven and six 252, of four 284, of three 270), else two CTAs a tile, whose fixed part weighs least. 4096 -> 28672 features,
// rank 16, the kernel's us by itself with 8, 7, 6, 4, 3 and 2 CTAs: 32 tiles 11.7, 13.1, 13.9, -, -, -; 34 17.6, 14.0, 14.7; 38 20.3, 21.7, 15.2, 18.3; 46 -, 26.8, 27.1, 21.3; 72
// -, -, -, 44.6, 34.7, 41; 94 -, -, -, -, 57.6, 44.9. Clusters of five gain 8 % on four at 46 to 53 tiles.
template <int R>
cudaError_t launch_rank(const LoraParams& p, int sm_count, cudaStream_t s) {
  const long long places = (long long)sm_count * LoraShape<8, R>::RESIDENT;
  auto fit = [&](int ctas, int percent) { return p.n_tiles * 100ll * ctas <= places * percent; };
  if (fit(8, 87)) return launch<LoraShape<8, R>>(p, s);
  if (fit(7, 86)) return launch<LoraShape<7, R>>(p, s);
  if (fit(6, 86)) return launch<LoraShape<6, R>>(p, s);
  if (fit(4, 96)) return launch<LoraShape<4, R>>(p, s);
  if (fit(3, 92)) return launch<LoraShape<3, R>>(p, s);
  return launch<LoraShape<2, R>>(p, s);
}

}  // namespace

cudaError_t lora_apply(const LoraParams& p, int sm_count, cudaStream_t s) {
  if (p.n_tiles < 1 || p.n_in % 32) return cudaErrorInvalidValue;
  switch (p.stride) {
    case 16: return launch_rank<16>(p, sm_count, s);
    case 32: return launch_rank<32>(p, sm_count, s);
    case 64: return launch_rank<64>(p, sm_count, s);
    case 128: return launch_rank<128>(p, sm_count, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace kc
