// Norms of queries and keys for each head and their rotation at given positions, in one pass.
//
//   y = x * w / sqrt(mean(x^2) + epsilon)      per head, where a weight is given
//   (a, b) -> (a cos - b sin, a sin + b cos)   for the rotary / 2 pairs of the first `rotary` values: (i, i + rotary / 2), or
//                                              neighbours (2 i, 2 i + 1); the rest of the head passes through
// All in FP32 with one rounding at the end (the verify step's own kernel keeps the reference's BF16 rounding points).
//
// Bound by the bytes of q and k, in and out. A thread owns 16 values of a head as two 16-byte vectors, chosen so that both
// members of every pair are its own: vectors j and j + rotary / 16 of the rotated part (whole neighbours' pairs lie in any
// vector), two adjacent ones of the rest. So a head is width / 16 lanes, the norm a few shuffles, and nothing passes through
// shared memory. A thread takes the same place of kHeads heads of a row, whose loads are under way together; the table's 64 bytes
// for that place are read once for them. 2048 rows of 32 + 8 heads of 128: 11.8 us = 3.6 TB/s, two waves of blocks that each wait
// for the position, then for the table; 64 rows: 2.4 us, a launch.
#include "context_kernels.cuh"

#include <algorithm>

namespace ei {
namespace {

constexpr int kHeads = 2;  // heads a thread has under way
constexpr int kMostThreads = 512;

__device__ __forceinline__ void unpack(const uint4& v, float* x) {
  x[0] = bf16_lo(v.x), x[1] = bf16_hi(v.x), x[2] = bf16_lo(v.y), x[3] = bf16_hi(v.y);
  x[4] = bf16_lo(v.z), x[5] = bf16_hi(v.z), x[6] = bf16_lo(v.w), x[7] = bf16_hi(v.w);
}
__device__ __forceinline__ uint4 pack(const float* x) {
  return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

// Block (row, chunk of heads); kLanes (a power of two >= width / 16) threads a head.
template <bool kInterleaved, int kLanes>
__global__ void __launch_bounds__(kMostThreads) qk_norm_rope_kernel(const __grid_constant__ QkRopeParams p) {
  constexpr int lanes = kLanes;
  const int row = blockIdx.x;
  const int slot = threadIdx.x / lanes, slots = blockDim.x / lanes, j = threadIdx.x & (lanes - 1);
  const bool active = j < p.width / 16;
  const int pairs = p.rotary / 16;  // threads of a head that rotate
  const bool turns = j < pairs;
  const int first = (turns ? j : p.rotary / 8 + 2 * (j - pairs)) * 8;
  const int second = turns ? first + pairs * 8 : first + 8;
  const int stop = p.heads + p.kv_heads, head0 = blockIdx.y * slots * kHeads;

  // The position first: the table's address waits for it, and both for the whole way to memory.
  const long long position = p.positions ? p.positions[row] : (long long)p.offset + row;
  uint4 held[kHeads][2];
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    const int head = head0 + u * slots + slot;
    held[u][0] = held[u][1] = make_uint4(0, 0, 0, 0);
    if (active && head < stop) {
      const bf16* from = head < p.heads ? p.q + row * p.q_row + size_t(head) * p.width
                                        : p.k + row * p.k_row + size_t(head - p.heads) * p.width;
      held[u][0] = *reinterpret_cast<const uint4*>(from + first);
      held[u][1] = *reinterpret_cast<const uint4*>(from + second);
    }
  }
  const bool known = position >= 0 && position < p.table_rows;
  float turn[16];  // (sine, cosine) of the thread's eight pairs
#pragma unroll
  for (int i = 0; i < 16; ++i) turn[i] = 0.0f;
  if (active && turns && known) {
    const float* entry = p.table + size_t(position) * p.rotary;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // Half layout: pairs first .. first + 7. Neighbours: four pairs of each vector.
      const int at = !kInterleaved ? 2 * first + 4 * i : (i < 2 ? first : second) + 4 * (i & 1);
      const float4 v = __ldg(reinterpret_cast<const float4*>(entry + at));
      turn[4 * i] = v.x, turn[4 * i + 1] = v.y, turn[4 * i + 2] = v.z, turn[4 * i + 3] = v.w;
    }
  }
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    const int head = head0 + u * slots + slot;
    float x[16];
    unpack(held[u][0], x);
    unpack(held[u][1], x + 8);
    const bf16* weight = head < p.heads ? p.q_weight : p.k_weight;
    float squares = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) squares = fmaf(x[i], x[i], squares);
#pragma unroll
    for (int o = lanes >> 1; o > 0; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
    if (!active || head >= stop) continue;
    if (weight) {
      const float inverse = rsqrtf(fmaf(squares, p.inverse_width, p.epsilon));
      float w[16];
      unpack(__ldg(reinterpret_cast<const uint4*>(weight + first)), w);
      unpack(__ldg(reinterpret_cast<const uint4*>(weight + second)), w + 8);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] *= inverse * w[i];
    }
    if (turns) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int a = kInterleaved ? 2 * i : i, b = kInterleaved ? 2 * i + 1 : i + 8;
        const float sine = turn[2 * i], cosine = turn[2 * i + 1], xa = x[a], xb = x[b];
        x[a] = xa * cosine - xb * sine;
        x[b] = xa * sine + xb * cosine;
      }
    }
    if (!known) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 0.0f;
    }
    bf16* to = head < p.heads ? p.q_out + row * p.q_out_row + size_t(head) * p.width
                              : p.k_out + row * p.k_out_row + size_t(head - p.heads) * p.width;
    *reinterpret_cast<uint4*>(to + first) = pack(x);
    *reinterpret_cast<uint4*>(to + second) = pack(x + 8);
  }
}

using RopeKernel = void (*)(QkRopeParams);
template <bool kInterleaved>
RopeKernel rope_kernel_of(int lanes) {
  switch (lanes) {
    case 1: return qk_norm_rope_kernel<kInterleaved, 1>;
    case 2: return qk_norm_rope_kernel<kInterleaved, 2>;
    case 4: return qk_norm_rope_kernel<kInterleaved, 4>;
    case 8: return qk_norm_rope_kernel<kInterleaved, 8>;
    case 16: return qk_norm_rope_kernel<kInterleaved, 16>;
    default: return qk_norm_rope_kernel<kInterleaved, 32>;
  }
}
RopeKernel rope_kernel(bool interleaved, int lanes) { return interleaved ? rope_kernel_of<true>(lanes) : rope_kernel_of<false>(lanes); }

}  // namespace

void launch_qk_norm_rope(const QkRopeParams& p, cudaStream_t stream) {
  int lanes = 1;
  while (lanes < p.width / 16) lanes *= 2;
  // A row's heads make a block where they can. (2048 rows of 32 + 8 heads: 11.8 us; a block that walks rows with the next one's loads
  // under way needs twice the registers and takes 14.8, four heads a thread 14.1, one 13.9.)
  const int all = p.heads + p.kv_heads;
  const int threads = std::min(kMostThreads, ((all + kHeads - 1) / kHeads * lanes + 31) / 32 * 32);
  const int chunk = threads / lanes * kHeads;
  const dim3 grid(unsigned(p.rows), unsigned((all + chunk - 1) / chunk));
  launch(rope_kernel(p.interleaved, lanes), grid, dim3(unsigned(threads)), 0, stream, false, p);
}

}  // namespace ei
