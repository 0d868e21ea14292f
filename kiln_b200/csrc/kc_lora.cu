// What low-rank adapters add to a projection's rows: out_i = y_i + s_a B_a (A_a x_i), a the adapter of row i.
//
// One launch. Rows are grouped by adapter on the host (kc_adapter_rows_create) into tiles of at most 64, and a tile is a cluster's
// of eight CTAs: each multiplies an eighth of the features of x with an eighth of A's columns, the partial t = A x [rows, rank] meet in
// the cluster's shared memory, and each CTA takes an eighth of the projection's features through B and adds them to y.
// So t never goes through memory, x, y and the adapter are read once a tile, and no workspace or order of atomics is involved.
//
// Both products are mma.sync m16n8k16: what bounds the operator is memory, rank / 2 operations a byte of y, far below what either
// kind of tensor instruction does, and these take their operands from registers as they come from memory. The contraction's order is free,
// so a lane's elements of an operand are neighbours: 16-byte loads of x and A, and of B where ranks are stored by 32; the
// columns of B are dealt so that a lane has eight neighbouring features of y.
//
// t is summed in fp32, multiplied by s and goes into the second product as two bf16 numbers (its rounded value and what that leaves:
// 2^-17 of it is lost, a 256th of the output's own step); y is added in fp32 and the result rounded once.
#include "kc_lora.cuh"

#include "kc_umma.cuh"

#include <algorithm>

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

// Shared memory of a CTA: partial sums of its warps [8][16][pad], its t [16 MT][stride], t in two parts [2][16 MT][stride + 8].
__host__ __device__ constexpr int lora_pad(int stride) { return stride + 8; }
constexpr size_t lora_smem(int stride, int mt) {
  return (size_t)LORA_WARPS * 16 * lora_pad(stride) * 4 + (size_t)16 * mt * stride * 4 + (size_t)2 * 16 * mt * lora_pad(stride) * 2;
}

// MT: row blocks of 16 in a tile; the CTA's eight warps are MT of them times 8 / MT parts of its features. VEC: rows of y and out
// start on 16-byte boundaries.
template <int MT, bool VEC>
__global__ void __launch_bounds__(LORA_THREADS, 2)
lora_kernel(const LoraParams p) {
  constexpr int KP = LORA_WARPS / MT;
  extern __shared__ __align__(16) uint8_t lora_smem_base[];
  const int R = p.stride, pad = lora_pad(R);
  float* part = reinterpret_cast<float*>(lora_smem_base);
  float* sum = part + LORA_WARPS * 16 * pad;
  bf16* th = reinterpret_cast<bf16*>(sum + 16 * MT * R);
  bf16* tl = th + 16 * MT * pad;
  __shared__ int rows[16 * MT];
  pdl_launch_dependents();
  cluster_arrive();                    // waited for before the first access to another CTA's shared memory: it has started by then
  const int rank = blockIdx.x % LORA_CTAS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();
  const LoraTile tile = p.tiles[blockIdx.x / LORA_CTAS];
  const LoraSlot slot = tile.slot >= 0 ? p.slots[tile.slot] : LoraSlot{0, 0.f};
  if (threadIdx.x < 16 * MT) rows[threadIdx.x] = p.rows[tile.first + min((int)threadIdx.x, tile.n - 1)];
  __syncthreads();
  cluster_wait();
  const int blocks = (p.n_out + 31) / 32, b0 = (int)((long long)blocks * rank / LORA_CTAS), b1 = (int)((long long)blocks * (rank + 1) / LORA_CTAS);

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
  // ranks in use, in whole steps
  const int steps = R == 16 ? 1 : (slot.rank + 31) / 32 * 2;   // of 16

  // ---- t = A x over this CTA's features: warp = (row block, part) ----
  {
    const int mt = warp % MT, kp = warp / MT;
    const int chunks = p.n_in / 32, parts = LORA_CTAS * KP, me = rank * KP + kp;
    const int c0 = (int)((long long)chunks * me / parts), c1 = (int)((long long)chunks * (me + 1) / parts);
    const bf16* x0 = p.x + (size_t)rows[mt * 16 + g] * p.n_in + t * 8;
    const bf16* x1 = p.x + (size_t)rows[mt * 16 + g + 8] * p.n_in + t * 8;
    const bf16* a = p.a + ((size_t)tile.slot * R + g) * p.n_in + t * 8;
    // Ranks 32 at a time: four column blocks of eight, or the two there are.
    for (int s = 0; s < steps; s += 2) {
      float acc[4][4] = {};
      if (mt * 16 < tile.n) {
#pragma unroll 4
        for (int c = c0; c < c1; ++c) {
          const uint4 u0 = *reinterpret_cast<const uint4*>(x0 + (size_t)c * 32), u1 = *reinterpret_cast<const uint4*>(x1 + (size_t)c * 32);
          uint4 w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < 2 || steps > 1) w[j] = *reinterpret_cast<const uint4*>(a + (size_t)(s * 16 + j * 8) * p.n_in + (size_t)c * 32);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < 2 || steps > 1) {
              mma_bf16(acc[j], u0.x, u1.x, u0.y, u1.y, w[j].x, w[j].y);
              mma_bf16(acc[j], u0.z, u1.z, u0.w, u1.w, w[j].z, w[j].w);
            }
        }
      }
      float* to = part + (warp * 16 + g) * pad + s * 16 + t * 2;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < 2 || steps > 1) {
          *reinterpret_cast<float2*>(to + j * 8) = make_float2(acc[j][0], acc[j][1]);
          *reinterpret_cast<float2*>(to + 8 * pad + j * 8) = make_float2(acc[j][2], acc[j][3]);
        }
    }
  }
  __syncthreads();
  const int live = min(MT, (tile.n + 15) / 16), used = steps * 16, items = live * 16 * used;
  for (int i = threadIdx.x; i < items; i += LORA_THREADS) {
    const int row = i / used, r = i - row * used, mt = row >> 4;
    float v = 0.f;
#pragma unroll
    for (int kp = 0; kp < KP; ++kp) v += part[((kp * MT + mt) * 16 + (row & 15)) * pad + r];
    sum[row * R + r] = v;
  }
  cluster_sync();
  // ---- the cluster's t, in the order of its CTAs; ranks past the adapter's own have no part, whatever x holds ----
  for (int i = threadIdx.x; i < items; i += LORA_THREADS) {
    const int row = i / used, r = i - row * used;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < LORA_CTAS; ++k) v += peer_float(&sum[row * R + r], k);
    v = r < slot.rank ? v * slot.scale : 0.f;
    const bf16 hi = __float2bfloat16_rn(v);
    const float rest = v - __bfloat162float(hi);
    th[row * pad + r] = hi;
    tl[row * pad + r] = __float2bfloat16_rn(rest == rest ? rest : 0.f);   // of an infinite value nothing is left
  }
  cluster_arrive();                    // no CTA leaves while another one reads its sums; the barrier also joins this CTA's warps
  cluster_wait();

  // ---- out = y + B t: a warp has 32 features at a time. Column 2 t' + e of column block j is feature 8 t' + 2 j + e, so that a
  // lane's columns are eight neighbours ----
  const bf16* bank = p.b + (size_t)tile.slot * p.n_out * R;
  for (int blk = b0 + warp; blk < b1; blk += LORA_WARPS) {
    const int f0 = blk * 32, mine = f0 + t * 8;
    float acc[MT][4][4] = {};
    uint4 y[MT][2];
    if (VEC) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (m * 16 + h * 8 + g < tile.n && mine < p.n_out) y[m][h] = *reinterpret_cast<const uint4*>(p.y + (size_t)rows[m * 16 + h * 8 + g] * p.n_out + mine);
    }
    const int feature = f0 + (g >> 1) * 8 + (g & 1);
    if (R == 16) {
      uint2 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint2*>(bank + (size_t)min(feature + 2 * j, p.n_out - 1) * 16 + t * 4);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m >= live) break;
#pragma unroll
        for (int part2 = 0; part2 < 2; ++part2) {
          const bf16* src = (part2 ? tl : th) + (m * 16 + g) * pad + t * 4;
          const uint2 v0 = *reinterpret_cast<const uint2*>(src), v1 = *reinterpret_cast<const uint2*>(src + 8 * pad);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_bf16(acc[m][j], v0.x, v1.x, v0.y, v1.y, w[j].x, w[j].y);
        }
      }
    } else {
#pragma unroll 1
      for (int s = 0; s < steps; s += 2) {
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint4*>(bank + (size_t)min(feature + 2 * j, p.n_out - 1) * R + s * 16 + t * 8);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (m >= live) break;
#pragma unroll
          for (int part2 = 0; part2 < 2; ++part2) {
            const bf16* src = (part2 ? tl : th) + (m * 16 + g) * pad + s * 16 + t * 8;
            const uint4 v0 = *reinterpret_cast<const uint4*>(src), v1 = *reinterpret_cast<const uint4*>(src + 8 * pad);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mma_bf16(acc[m][j], v0.x, v1.x, v0.y, v1.y, w[j].x, w[j].y);
              mma_bf16(acc[m][j], v0.z, v1.z, v0.w, v1.w, w[j].z, w[j].w);
            }
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = m * 16 + h * 8 + g;
        if (r >= tile.n || mine >= p.n_out) continue;
        const size_t at = (size_t)rows[r] * p.n_out + mine;
        if (VEC) {
          const uint32_t v[4] = {y[m][h].x, y[m][h].y, y[m][h].z, y[m][h].w};
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack_bf162(v[j]);
            o[j] = pack_bf162(f.x + acc[m][j][2 * h], f.y + acc[m][j][2 * h + 1]);
          }
          *reinterpret_cast<uint4*>(p.out + at) = make_uint4(o[0], o[1], o[2], o[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (mine + e < p.n_out) p.out[at + e] = __float2bfloat16_rn(__bfloat162float(p.y[at + e]) + acc[m][e >> 1][2 * h + (e & 1)]);
        }
      }
  }
}

template <int MT, bool VEC>
cudaError_t launch_as(const LoraParams& p, cudaStream_t s) {
  static DeviceOnce configured;   // the attribute belongs to the device's copy of the kernel
  if (configured.first_on_current_device()) {
    cudaError_t e = cudaFuncSetAttribute(lora_kernel<MT, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lora_smem(LORA_MAX_RANK, MT));
    if (e != cudaSuccess) { configured.forget_current_device(); return e; }
  }
  return launch_k_cluster(LORA_CTAS, lora_kernel<MT, VEC>, dim3(p.n_tiles * LORA_CTAS), dim3(LORA_THREADS), lora_smem(p.stride, MT), s, p);
}

}  // namespace

cudaError_t lora_apply(const LoraParams& p, cudaStream_t s) {
  if (p.n_tiles < 1 || p.n_in % 32 || p.stride > LORA_MAX_RANK) return cudaErrorInvalidValue;
  const bool vec = p.n_out % 8 == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  switch (p.tile_rows) {
    case 16: return vec ? launch_as<1, true>(p, s) : launch_as<1, false>(p, s);
    case 32: return vec ? launch_as<2, true>(p, s) : launch_as<2, false>(p, s);
    case 64: return vec ? launch_as<4, true>(p, s) : launch_as<4, false>(p, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace kc
