// The router's load: how many of its choices went to each expert, and the loss that keeps the load even.
//
//   counts_e = number of (token, slot) pairs of counted tokens whose id is e       (ids outside 0..E-1 are not counted)
//   f_e = counts_e / sum counts,  p_t = softmax(z_t),  n = counted tokens
//   loss = E * sum_e f_e * mean_t p_te = (E / n) * sum_t d_t,   d_t = sum_e f_e p_te
//   dloss/dz_te = (E / n) * p_te * (f_e - d_t)                                      (the counts carry no gradient)
// The middle form needs no sum per expert: one number per token, added up in FP64 in a fixed order.
// A row without any finite logit has no probabilities: it counts as a token and contributes nothing.

namespace netra {

constexpr int kBalMaxExperts = 1024;
constexpr int kBalThreads = 256;

// ids [tokens, slots] (rows id_pitch apart) -> counts [experts], which the caller cleared
extern "C" __global__ void __launch_bounds__(256)
netra_expert_counts_sm100(const void* __restrict__ ids, uint32_t wide, uint64_t id_pitch, const uint8_t* __restrict__ mask,
                          int32_t* __restrict__ counts, uint64_t tokens, uint32_t slots, uint32_t experts) {
  __shared__ int hist[kBalMaxExperts];
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  const uint64_t pairs = tokens * slots;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < pairs; i += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t t = i / slots, at = t * id_pitch + (i - t * slots);
    if (mask != nullptr && mask[t] == 0) continue;
    const long long id = wide ? reinterpret_cast<const long long*>(ids)[at] : (long long)reinterpret_cast<const int32_t*>(ids)[at];
    if (id >= 0 && id < (long long)experts) atomicAdd(&hist[id], 1);
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x)
    if (hist[e] != 0) atomicAdd(&counts[e], hist[e]);
}

__device__ __forceinline__ float bal_load(const void* z, uint32_t dtype, uint64_t i) { return dense_load(z, dtype, i); }

// share[e] = counts[e] / sum counts (0 where nothing was counted)
__device__ __forceinline__ void bal_shares(float* share, const int32_t* __restrict__ counts, uint32_t experts) {
  __shared__ unsigned long long total;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  unsigned long long mine = 0;
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) mine += (unsigned long long)(long long)counts[e];
  atomicAdd(&total, mine);
  __syncthreads();
  const float inv = total > 0 ? (float)(1.0 / (double)total) : 0.0f;
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) share[e] = (float)counts[e] * inv;
  __syncthreads();
}

// one warp, one row: p[i] = softmax of expert lane + 32 i; returns d = sum_e share_e p_e in every lane
template <int kPer>
__device__ __forceinline__ float bal_row(float p[kPer], const void* __restrict__ z, uint32_t dtype, uint64_t base, const float* share,
                                         uint32_t experts, int lane) {
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t e = lane + 32 * i;
    p[i] = e < experts ? bal_load(z, dtype, base + e) : -INFINITY;
    mx = fmaxf(mx, p[i]);
  }
  mx = warp_max(mx);
  const float shift = mx == -INFINITY ? 0.0f : mx;
  float sum = 0.0f, dot = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t e = lane + 32 * i;
    p[i] = expf(p[i] - shift);
    sum += p[i];
    dot = fmaf(p[i], e < experts ? share[e] : 0.0f, dot);
  }
  sum = warp_sum(sum);
  dot = warp_sum(dot);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int i = 0; i < kPer; ++i) p[i] *= inv;
  return dot * inv;
}

struct BalPartial { double sum; unsigned long long rows; };

// loss, and scale = E / n; partial: one slot per block, ticket: cleared by the caller
template <int kPer>
__global__ void __launch_bounds__(kBalThreads)
netra_balance_loss_sm100(const void* __restrict__ z, uint32_t dtype, uint64_t pitch, const int32_t* __restrict__ counts,
                         const uint8_t* __restrict__ mask, float* __restrict__ loss, float* __restrict__ scale, BalPartial* __restrict__ partial,
                         uint32_t* __restrict__ ticket, uint64_t tokens, uint32_t experts) {
  __shared__ float share[kBalMaxExperts];
  __shared__ double warp_part[kBalThreads / 32];
  __shared__ unsigned long long warp_rows[kBalThreads / 32];
  __shared__ bool last;
  bal_shares(share, counts, experts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double sum = 0.0;
  unsigned long long rows = 0;
  float p[kPer];
  for (uint64_t t = (uint64_t)blockIdx.x * (kBalThreads / 32) + warp; t < tokens; t += (uint64_t)gridDim.x * (kBalThreads / 32)) {
    if (mask != nullptr && mask[t] == 0) continue;
    sum += (double)bal_row<kPer>(p, z, dtype, t * pitch, share, experts, lane);
    ++rows;
  }
  if (lane == 0) { warp_part[warp] = sum; warp_rows[warp] = rows; }
  __syncthreads();
  if (threadIdx.x == 0) {
    BalPartial b = {0.0, 0};
    for (int w = 0; w < kBalThreads / 32; ++w) { b.sum += warp_part[w]; b.rows += warp_rows[w]; }
    partial[blockIdx.x] = b;
    __threadfence();
    last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last || warp != 0) return;
  __threadfence();
  double s = 0.0;
  unsigned long long n = 0;
  for (uint32_t b = lane; b < gridDim.x; b += 32) { s += __ldcg(&partial[b].sum); n += __ldcg(&partial[b].rows); }
  for (int d = 16; d > 0; d >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, d); n += __shfl_xor_sync(0xffffffffu, n, d); }
  if (lane == 0) {
    const double per = n > 0 ? (double)experts / (double)n : 0.0;
    *loss = (float)(s * per);
    *scale = (float)per;
  }
}

template <int kPer>
__global__ void __launch_bounds__(kBalThreads)
netra_balance_loss_grad_sm100(void* __restrict__ grad, uint64_t grad_pitch, const void* __restrict__ z, uint32_t dtype, uint64_t pitch,
                              const int32_t* __restrict__ counts, const uint8_t* __restrict__ mask, const float* __restrict__ scale,
                              const float* __restrict__ upstream, uint64_t tokens, uint32_t experts) {
  __shared__ float share[kBalMaxExperts];
  bal_shares(share, counts, experts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float k = scale[0] * upstream[0];
  float p[kPer];
  for (uint64_t t = (uint64_t)blockIdx.x * (kBalThreads / 32) + warp; t < tokens; t += (uint64_t)gridDim.x * (kBalThreads / 32)) {
    const bool live = mask == nullptr || mask[t] != 0;
    float d = 0.0f;
    if (live) d = bal_row<kPer>(p, z, dtype, t * pitch, share, experts, lane);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = lane + 32 * i;
      if (e < experts) dense_store(grad, dtype, t * grad_pitch + e, live ? p[i] * (share[e] - d) * k : 0.0f);
    }
  }
}

}  // namespace netra

namespace {

constexpr uint32_t kBalMaxBlocks = 1184;      // eight blocks per SM of a 148-SM device

int balance_check(const char* what, const void* z, uint32_t dtype, uint64_t pitch, const void* counts, uint64_t tokens, uint32_t experts) {
  static thread_local char text[128];
  auto bad = [&](const char* why) { snprintf(text, sizeof text, "%s: %s", what, why); return fail(text); };
  if (!z || !counts) return bad("null pointer");
  if (dtype > kDenseF32) return bad("unknown element type");
  if (experts == 0 || experts > (uint32_t)kBalMaxExperts) return bad("experts must be 1..1024");
  if (tokens == 0 || tokens > (1ull << 40)) return bad("tokens out of range");
  if (tokens > 1 && pitch < experts) return bad("a row pitch is smaller than the row");
  if ((uintptr_t)z % dense_element_bytes(dtype)) return bad("logits are not aligned to their element");
  return 0;
}

uint32_t balance_blocks(uint64_t tokens) {
  const uint64_t b = (tokens + kBalThreads / 32 - 1) / (kBalThreads / 32);
  return (uint32_t)(b < kBalMaxBlocks ? b : kBalMaxBlocks);
}

}  // namespace

extern "C" {

int netra_expert_counts_launch(int32_t* counts_i32, const void* ids, uint32_t id_bytes, uint64_t id_pitch, const uint8_t* token_mask,
                               uint64_t tokens, uint32_t slots, uint32_t experts, cudaStream_t stream) {
  if (!counts_i32 || (!ids && tokens && slots)) return fail("expert_counts: null pointer");
  if (id_bytes != 4 && id_bytes != 8) return fail("expert_counts: ids must have 4 or 8 bytes");
  if (experts == 0 || experts > (uint32_t)kBalMaxExperts) return fail("expert_counts: experts must be 1..1024");
  if (tokens > (1ull << 40) || slots > 1024 || tokens * slots > 0x7fffffffull) return fail("expert_counts: at most 2^31 - 1 choices of 1024 slots");
  if (tokens > 1 && id_pitch < slots) return fail("expert_counts: the row pitch is smaller than the row");
  if ((uintptr_t)ids % id_bytes) return fail("expert_counts: ids are not aligned to their element");
  cudaError_t e = cudaMemsetAsync(counts_i32, 0, experts * sizeof(int32_t), stream);
  if (e != cudaSuccess) return fail_cuda("expert_counts memset", e);
  const uint64_t pairs = tokens * slots;
  if (pairs == 0) return 0;
  const uint64_t blocks = (pairs + 1023) / 1024;
  netra_expert_counts_sm100<<<(unsigned)(blocks < 296 ? blocks : 296), 256, 0, stream>>>(ids, id_bytes == 8, id_pitch, token_mask, counts_i32,
                                                                                        tokens, slots, experts);
  return check_launch("expert_counts launch");
}

uint64_t netra_balance_loss_workspace_bytes(void) { return 16 + kBalMaxBlocks * sizeof(BalPartial); }

int netra_balance_loss_launch(float* loss_f32, float* scale_f32, const void* logits, uint32_t dtype, uint64_t pitch, const int32_t* counts_i32,
                              const uint8_t* token_mask, void* workspace, uint64_t workspace_bytes, uint64_t tokens, uint32_t experts,
                              cudaStream_t stream) {
  if (int rc = balance_check("balance_loss", logits, dtype, pitch, counts_i32, tokens, experts)) return rc;
  if (!loss_f32 || !scale_f32 || !workspace) return fail("balance_loss: null pointer");
  if (workspace_bytes < netra_balance_loss_workspace_bytes() || (uintptr_t)workspace % 16) return fail("balance_loss: workspace too small or not 16-byte aligned");
  uint32_t* ticket = (uint32_t*)workspace;
  BalPartial* partial = (BalPartial*)((uint8_t*)workspace + 16);
  cudaError_t e = cudaMemsetAsync(ticket, 0, sizeof(uint32_t), stream);
  if (e != cudaSuccess) return fail_cuda("balance_loss memset", e);
  const uint32_t grid = balance_blocks(tokens);
  auto launch = [&](auto per) {
    netra_balance_loss_sm100<decltype(per)::value><<<grid, kBalThreads, 0, stream>>>(logits, dtype, pitch, counts_i32, token_mask, loss_f32, scale_f32,
                                                                                    partial, ticket, tokens, experts);
  };
  if (experts <= 64) launch(std::integral_constant<int, 2>{});
  else if (experts <= 256) launch(std::integral_constant<int, 8>{});
  else launch(std::integral_constant<int, 32>{});
  return check_launch("balance_loss launch");
}

int netra_balance_loss_grad_launch(void* grad, uint64_t grad_pitch, const void* logits, uint32_t dtype, uint64_t pitch, const int32_t* counts_i32,
                                   const uint8_t* token_mask, const float* scale_f32, const float* upstream_f32, uint64_t tokens,
                                   uint32_t experts, cudaStream_t stream) {
  if (int rc = balance_check("balance_loss_grad", logits, dtype, pitch, counts_i32, tokens, experts)) return rc;
  if (!grad || !scale_f32 || !upstream_f32) return fail("balance_loss_grad: null pointer");
  if (tokens > 1 && grad_pitch < experts) return fail("balance_loss_grad: a row pitch is smaller than the row");
  if ((uintptr_t)grad % dense_element_bytes(dtype)) return fail("balance_loss_grad: the gradient is not aligned to its element");
  const uint32_t grid = balance_blocks(tokens);
  auto launch = [&](auto per) {
    netra_balance_loss_grad_sm100<decltype(per)::value><<<grid, kBalThreads, 0, stream>>>(grad, grad_pitch, logits, dtype, pitch, counts_i32, token_mask,
                                                                                         scale_f32, upstream_f32, tokens, experts);
  };
  if (experts <= 64) launch(std::integral_constant<int, 2>{});
  else if (experts <= 256) launch(std::integral_constant<int, 8>{});
  else launch(std::integral_constant<int, 32>{});
  return check_launch("balance_loss_grad launch");
}

}  // extern "C"
