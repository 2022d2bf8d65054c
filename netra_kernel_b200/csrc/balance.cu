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

constexpr int kBalCluster = 8;            // blocks of the one-cluster forms
constexpr int kBalClusterThreads = 1024;

// hist[e] += the block's share of the choices: blocks first, first + step, ... of blockDim choices each
__device__ __forceinline__ void count_choices(int* hist, const void* ids, uint32_t wide, uint64_t id_pitch,
                                              const uint8_t* mask, uint64_t tokens, uint32_t slots, uint32_t experts) {
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  const uint32_t pairs = (uint32_t)tokens * slots, step = gridDim.x * blockDim.x;       // the host keeps pairs below 2^31
#pragma unroll 4
  for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < pairs; i += step) {
    const uint32_t t = i / slots;
    const uint64_t at = t * id_pitch + (i - t * slots);
    const bool live = mask == nullptr || mask[t] != 0;
    const long long id = wide ? reinterpret_cast<const long long*>(ids)[at] : (long long)reinterpret_cast<const int32_t*>(ids)[at];
    if (live && id >= 0 && id < (long long)experts) atomicAdd(&hist[id], 1);
  }
  __syncthreads();
}

// ids [tokens, slots] (rows id_pitch apart) -> counts [experts], which the caller cleared
extern "C" __global__ void __launch_bounds__(256)
netra_expert_counts_sm100(const void* ids, uint32_t wide, uint64_t id_pitch, const uint8_t* mask,
                          int32_t* counts, uint64_t tokens, uint32_t slots, uint32_t experts) {
  __shared__ int hist[kBalMaxExperts];
  begin_grid();
  count_choices(hist, ids, wide, id_pitch, mask, tokens, slots, experts);
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x)
    if (hist[e] != 0) atomicAdd(&counts[e], hist[e]);
}

// The same in one cluster, whose blocks add up their histograms over distributed shared memory: nothing to clear beforehand
extern "C" __global__ void __cluster_dims__(kBalCluster, 1, 1) __launch_bounds__(kBalClusterThreads)
netra_expert_counts_cluster_sm100(const void* ids, uint32_t wide, uint64_t id_pitch, const uint8_t* mask,
                                  int32_t* counts, uint64_t tokens, uint32_t slots, uint32_t experts) {
  __shared__ int hist[kBalMaxExperts];
  begin_grid();
  count_choices(hist, ids, wide, id_pitch, mask, tokens, slots, experts);
  cluster_barrier();                        // every block's histogram is complete
  for (uint32_t e = cluster_rank() * kBalClusterThreads + threadIdx.x; e < experts * kBalCluster; e += kBalCluster * kBalClusterThreads) {
    // expert e / 8 by eight neighbouring lanes, one block's count each
    int n = ld_cluster_i32(map_to_rank(smem_u32(&hist[e / kBalCluster]), e % kBalCluster));
    const uint32_t group = 0xffu << (threadIdx.x & 24);
#pragma unroll
    for (int d = kBalCluster / 2; d > 0; d >>= 1) n += __shfl_xor_sync(group, n, d);
    if (e % kBalCluster == 0) counts[e / kBalCluster] = n;
  }
  __syncwarp();
  cluster_barrier();                        // nobody leaves while its histogram is being read
}

__device__ __forceinline__ float redux_max_f32(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// A lane holds kVec neighbouring experts (16 bytes) of every 32 * kVec.  kAligned: every row allows 16-byte accesses; without
// it the same lane loads the same experts one by one, so that alignment does not change a sum.
template <typename T, bool kAligned, int kPer>
struct BalLane {
  static constexpr int kVec = 16 / sizeof(T);
  static_assert(kPer % kVec == 0, "a lane holds whole accesses");
  __device__ static __forceinline__ uint32_t expert(int i, int lane) { return (uint32_t)((i / kVec) * 32 * kVec + lane * kVec + i % kVec); }
  __device__ static __forceinline__ void load(float v[kPer], const T* row, uint32_t experts, int lane) {
#pragma unroll
    for (int i = 0; i < kPer; i += kVec) {
      const uint32_t e = expert(i, lane);
      if (kAligned && e < experts) {
        if constexpr (kVec == 8) {
          Eight<T> x8;
          x8.load(row + e);
          x8.values(v + i);
        } else {
          const float4 f = *reinterpret_cast<const float4*>(row + e);
          v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[i + j] = e + j < experts ? dense_load(row, DenseElement<T>::code, e + j) : -INFINITY;
      }
    }
  }
  __device__ static __forceinline__ void store(T* row, const float v[kPer], uint32_t experts, int lane) {
#pragma unroll
    for (int i = 0; i < kPer; i += kVec) {
      const uint32_t e = expert(i, lane);
      if (kAligned && e < experts) {
        if constexpr (kVec == 8) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (std::is_same<T, __half>::value) {
              const __half2 h = __floats2half2_rn(v[i + 2 * j], v[i + 2 * j + 1]);
              w[j] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
              const __nv_bfloat162 h = __floats2bfloat162_rn(v[i + 2 * j], v[i + 2 * j + 1]);
              w[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
          }
          *reinterpret_cast<uint4*>(row + e) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
          *reinterpret_cast<float4*>(row + e) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (e + j < experts) dense_store(row, DenseElement<T>::code, e + j, v[i + j]);
      }
    }
  }
  // The counts of the lane's experts above the smallest count, which goes to least: f_e - d_t, small when the load is nearly
  // even, then comes from whole numbers as small (and is exactly 0 when it is even).  Returns 1 / the sum of the counts (FP32: a
  // common factor, off by a few steps at most).
  __device__ static __forceinline__ float counts(float c[kPer], float& least, const int32_t* all, uint32_t experts, int lane) {
    int n[kPer], low = 0x7fffffff;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = expert(i, lane);
      n[i] = e < experts ? all[e] : 0x7fffffff;
      if (e < experts) sum += (float)n[i];
      low = min(low, n[i]);
    }
    low = __reduce_min_sync(0xffffffffu, low);
    least = (float)low;
#pragma unroll
    for (int i = 0; i < kPer; ++i) c[i] = expert(i, lane) < experts ? (float)(n[i] - low) : 0.0f;
    sum = warp_sum(sum);
    return sum > 0.0f ? 1.0f / sum : 0.0f;
  }
};

// e^x = 2^h (1 + r) for x <= 0, with h = fl(x log2 e) and r = x - h ln 2, which is below 2^-17 and so leaves r^2 / 2 out; ln 2 in
// two parts, as in Cody and Waite's reductions.  The rounding of h alone would cost |x| 2^-24 (a probability of e^-80 off by 60
// units of 2^-24).  2^h is the hardware's, within two steps and measured 0.75 units of 2^-24 too small on average, which r makes
// good (0.7 units then by root mean square, as expf(); 1.05 without).  Two elements share their multiply-adds.  Loss and gradient
// of 16384 x 256 BF16: 18.8 us, 20.5 us with expf() instead; of 16384 x 512 FP32: 22.7 us, 24.7 us, 23.5 us one element at a time.
__device__ __forceinline__ float2 exp_nonpositive2(float a, float b) {
  auto finite = [](float x) {               // keeps a NaN; e^-200 is 0
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(-200.0f));
    return r;
  };
  auto both = [](float c) { return make_float2(c, c); };
  const float2 x = make_float2(finite(a), finite(b));
  const float2 h = fma2(x, both(1.4426950408889634f), both(-0.0f));
  const float2 low = fma2(h, both(1.9046543e-9f), both(0.75f * 0x1p-24f));
  const float2 r = fma2(fma2(h, both(-0.69314718f), x), both(1.0f), low);
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(h.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(h.y));
  return fma2(e, r, e);
}

// v: a row's logits -> its exponentials; returns sum_e c_e p_e in every lane, inv = 1 / sum of the exponentials
template <int kPer>
__device__ __forceinline__ float bal_row(float v[kPer], const float c[kPer], float& inv) {
  float mx = v[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) mx = fmaxf(mx, v[i]);
  mx = redux_max_f32(mx);
  const float shift = mx == -INFINITY ? 0.0f : mx;
  float sum = 0.0f, dot = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; i += 2) {
    const float2 e = exp_nonpositive2(v[i] - shift, v[i + 1] - shift);
    v[i] = e.x; v[i + 1] = e.y;
    sum += e.x;
    sum += e.y;
    dot = fmaf(e.x, c[i], dot);
    dot = fmaf(e.y, c[i + 1], dot);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, d);
    dot += __shfl_xor_sync(0xffffffffu, dot, d);
  }
  inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  return dot * inv;
}

struct BalPartial { double sum; unsigned long long rows; };

// A warp per row, a lane holds its experts' counts in registers (no block-wide step before the first row); the rows' d_t are
// added in FP64: per warp, over the block's warps, over the blocks, always in the same order.  scale = E / n.
// kCluster: the grid is one cluster, whose blocks leave their sums in the first one's shared memory; otherwise partial has one
// slot per block, and the block that draws the last number of ticket (cleared by the caller) adds them up.
template <typename T, bool kAligned, int kPer, bool kCluster>
__device__ __forceinline__ void balance_loss_body(const T* z, uint64_t pitch, const int32_t* counts,
                                                  const uint8_t* mask, float* loss, float* scale,
                                                  BalPartial* partial, uint32_t* ticket, uint64_t tokens,
                                                  uint32_t experts) {
  using L = BalLane<T, kAligned, kPer>;
  constexpr int kWarps = (kCluster ? kBalClusterThreads : kBalThreads) / 32;
  __shared__ double warp_part[kWarps];
  __shared__ unsigned long long warp_rows[kWarps];
  __shared__ BalPartial gathered[kCluster ? kBalCluster : 1];
  __shared__ bool last;
  if (kCluster) cluster_arrive();
  begin_grid();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double sum = 0.0;
  unsigned long long rows = 0;
  float c[kPer], v[kPer], inv, least;
  const float per_count = L::counts(c, least, counts, experts, lane);
  for (uint64_t t = (uint64_t)blockIdx.x * kWarps + warp; t < tokens; t += (uint64_t)gridDim.x * kWarps) {
    if (mask != nullptr && mask[t] == 0) continue;
    L::load(v, z + t * pitch, experts, lane);
    const float above = bal_row<kPer>(v, c, inv);
    sum += inv == 0.0f ? 0.0 : (double)((least + above) * per_count);
    ++rows;
  }
  if (lane == 0) { warp_part[warp] = sum; warp_rows[warp] = rows; }
  __syncthreads();
  auto add_up = [&](BalPartial& b) {
    b = {0.0, 0};
    for (int w = 0; w < kWarps; ++w) { b.sum += warp_part[w]; b.rows += warp_rows[w]; }
  };
  auto finish = [&](const BalPartial& b) {
    const double per = b.rows > 0 ? (double)experts / (double)b.rows : 0.0;
    *loss = (float)(b.sum * per);
    *scale = (float)per;
  };
  BalPartial b;
  if constexpr (kCluster) {
    cluster_wait();                         // every block is running
    if (threadIdx.x == 0) {
      add_up(b);
      const uint32_t to = map_to_rank(smem_u32(&gathered[cluster_rank()]), 0);
      st_cluster_b64(to, (unsigned long long)__double_as_longlong(b.sum));
      st_cluster_b64(to + 8, b.rows);
    }
    __syncwarp();
    cluster_barrier();
    if (cluster_rank() != 0 || threadIdx.x != 0) return;
    b = {0.0, 0};
    for (int r = 0; r < kBalCluster; ++r) { b.sum += gathered[r].sum; b.rows += gathered[r].rows; }
    finish(b);
  } else {
    if (threadIdx.x == 0) {
      add_up(b);
      partial[blockIdx.x] = b;
      __threadfence();
      last = atomicAdd(ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double s = 0.0;
    unsigned long long n = 0;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < gridDim.x; i += kBalThreads) { s += __ldcg(&partial[i].sum); n += __ldcg(&partial[i].rows); }
    for (int d = 16; d > 0; d >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, d); n += __shfl_xor_sync(0xffffffffu, n, d); }
    if (lane == 0) { warp_part[warp] = s; warp_rows[warp] = n; }
    __syncthreads();
    if (threadIdx.x == 0) {
      add_up(b);
      finish(b);
    }
  }
}

template <typename T, bool kAligned, int kPer>
__global__ void __launch_bounds__(kBalThreads)
netra_balance_loss_sm100(const T* z, uint64_t pitch, const int32_t* counts, const uint8_t* mask, float* loss, float* scale, BalPartial* partial,
                         uint32_t* ticket, uint64_t tokens, uint32_t experts) {
  balance_loss_body<T, kAligned, kPer, false>(z, pitch, counts, mask, loss, scale, partial, ticket, tokens, experts);
}

template <typename T, bool kAligned, int kPer>
__global__ void __cluster_dims__(kBalCluster, 1, 1) __launch_bounds__(kBalClusterThreads)
netra_balance_loss_cluster_sm100(const T* z, uint64_t pitch, const int32_t* counts, const uint8_t* mask, float* loss, float* scale,
                                 uint64_t tokens, uint32_t experts) {
  balance_loss_body<T, kAligned, kPer, true>(z, pitch, counts, mask, loss, scale, nullptr, nullptr, tokens, experts);
}

template <typename T, bool kAligned, int kPer>
__global__ void __launch_bounds__(kBalThreads)
netra_balance_loss_grad_sm100(T* grad, uint64_t grad_pitch, const T* z, uint64_t pitch,
                              const int32_t* counts, const uint8_t* mask, const float* scale,
                              const float* upstream, uint64_t tokens, uint32_t experts) {
  using L = BalLane<T, kAligned, kPer>;
  begin_grid();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float c[kPer], v[kPer], inv, least;
  const float per_count = L::counts(c, least, counts, experts, lane);
  const float k = *scale * *upstream;
  for (uint64_t t = (uint64_t)blockIdx.x * (kBalThreads / 32) + warp; t < tokens; t += (uint64_t)gridDim.x * (kBalThreads / 32)) {
    if (mask == nullptr || mask[t] != 0) {
      L::load(v, z + t * pitch, experts, lane);
      const float d = bal_row<kPer>(v, c, inv);
      // p_te (f_e - d_t) = p_te (c_e - sum_j c_j p_tj) / total: whole counts are subtracted, the quotient comes last
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] = v[i] * inv * ((c[i] - d) * per_count) * k;
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] = 0.0f;
    }
    L::store(grad + t * grad_pitch, v, experts, lane);
  }
}

}  // namespace netra

namespace {

// Up to here one cluster of eight blocks does it, without clearing anything first (one cluster against many blocks behind a
// memset: counts of 2,048 choices 2.7 us against 4.2 us, of 65,536 choices 4.7 us against 5.0 us; BF16 loss of 256 tokens and 256
// experts 3.9 us against 7.9 us, of 1,536 tokens 7.7 us against 8.3 us, of 1,800 tokens 8.8 us against 8.2 us).  A row of more than
// 256 experts costs a warp twice as much (512 experts: 768 tokens 8.1 us against 8.2 us, 900 tokens 9.3 us against 8.2 us).
constexpr uint64_t kCountsClusterPairs = 1 << 16, kLossClusterTokens = 1536;
constexpr uint32_t kBalMaxBlocks = 592;       // four blocks per SM of a 148-SM device: more warps only repeat the look at the counts

int balance_check(const char* what, const void* z, uint32_t dtype, uint64_t pitch, const void* counts, uint64_t tokens, uint32_t experts) {
  static thread_local char text[128];
  auto bad = [&](const char* why) { snprintf(text, sizeof text, "%s: %s", what, why); return fail(text); };
  if (!z || !counts) return bad("null pointer");
  if (dtype > kDenseF32) return bad("unknown element type");
  if (experts == 0 || experts > (uint32_t)kBalMaxExperts) return bad("experts must be 1..1024");
  if (tokens == 0 || tokens > (1ull << 40)) return bad("tokens out of range");
  if (tokens > 1 && pitch < experts) return bad("a row pitch is smaller than the row");
  if ((uintptr_t)z % dense_element_bytes(dtype)) return bad("logits are not aligned to their element");
  if ((uintptr_t)counts % 4) return bad("counts are not aligned to their element");
  return 0;
}

bool balance_one_cluster(uint64_t tokens, uint32_t experts) { return experts <= 512 && tokens <= kLossClusterTokens / (experts <= 256 ? 1 : 2); }

uint32_t balance_blocks(uint64_t tokens) {
  const uint64_t b = (tokens + kBalThreads / 32 - 1) / (kBalThreads / 32);
  return (uint32_t)(b < kBalMaxBlocks ? b : kBalMaxBlocks);
}

// Calls f(element, 16-byte accesses?, experts per lane) with the smallest register file that holds a row.
template <typename F>
void balance_shape(uint32_t dtype, bool aligned, uint32_t experts, F&& f) {
  auto sized = [&](auto element, auto access) {
    if constexpr (sizeof(element) == 4) {
      if (experts <= 128) { f(element, access, std::integral_constant<int, 4>{}); return; }
    }
    if (experts <= 256) f(element, access, std::integral_constant<int, 8>{});
    else if (experts <= 512) f(element, access, std::integral_constant<int, 16>{});
    else f(element, access, std::integral_constant<int, 32>{});
  };
  auto typed = [&](auto element) { if (aligned) sized(element, std::true_type{}); else sized(element, std::false_type{}); };
  if (dtype == kDenseF32) typed(0.0f);
  else if (dtype == kDenseF16) typed(__half{});
  else typed(__nv_bfloat16{});
}
bool balance_aligned(const void* p, uint64_t pitch, uint32_t dtype, uint32_t experts) {
  const uint64_t size = dense_element_bytes(dtype);
  return (uintptr_t)p % 16 == 0 && pitch * size % 16 == 0 && experts * size % 16 == 0;
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
  if ((uintptr_t)counts_i32 % 4) return fail("expert_counts: counts are not aligned to their element");
  const uint64_t pairs = tokens * slots;
  if (pairs <= kCountsClusterPairs)
    return launched("expert_counts launch",
                    launch_dependent(netra_expert_counts_cluster_sm100, dim3(kBalCluster), kBalClusterThreads, 0, stream, 1, ids, (uint32_t)(id_bytes == 8),
                                     id_pitch, token_mask, counts_i32, tokens, slots, experts));
  cudaError_t e = cudaMemsetAsync(counts_i32, 0, experts * sizeof(int32_t), stream);
  if (e != cudaSuccess) return fail_cuda("expert_counts memset", e);
  const uint64_t blocks = (pairs + 511) / 512;
  return launched("expert_counts launch",
                  launch_dependent(netra_expert_counts_sm100, dim3((unsigned)(blocks < 296 ? blocks : 296)), 256, 0, stream, 1, ids, (uint32_t)(id_bytes == 8),
                                   id_pitch, token_mask, counts_i32, tokens, slots, experts));
}

uint64_t netra_balance_loss_workspace_bytes(uint64_t tokens, uint32_t experts) {
  return balance_one_cluster(tokens, experts) ? 0 : 16 + kBalMaxBlocks * sizeof(BalPartial);
}

int netra_balance_loss_launch(float* loss_f32, float* scale_f32, const void* logits, uint32_t dtype, uint64_t pitch, const int32_t* counts_i32,
                              const uint8_t* token_mask, void* workspace, uint64_t workspace_bytes, uint64_t tokens, uint32_t experts,
                              cudaStream_t stream) {
  if (int rc = balance_check("balance_loss", logits, dtype, pitch, counts_i32, tokens, experts)) return rc;
  if (!loss_f32 || !scale_f32) return fail("balance_loss: null pointer");
  if ((uintptr_t)loss_f32 % 4 || (uintptr_t)scale_f32 % 4) return fail("balance_loss: an address is not aligned to its element");
  const uint64_t needed = netra_balance_loss_workspace_bytes(tokens, experts);
  if (needed > 0 && (!workspace || workspace_bytes < needed || (uintptr_t)workspace % 16)) return fail("balance_loss: workspace missing, too small or not 16-byte aligned");
  const bool aligned = balance_aligned(logits, pitch, dtype, experts);
  cudaError_t launch = cudaSuccess;
  if (needed == 0) {
    balance_shape(dtype, aligned, experts, [&](auto element, auto access, auto per) {
      using T = decltype(element);
      if constexpr (decltype(per)::value <= 16)
        launch = launch_dependent(netra_balance_loss_cluster_sm100<T, decltype(access)::value, decltype(per)::value>, dim3(kBalCluster), kBalClusterThreads, 0,
                                  stream, 1, (const T*)logits, pitch, counts_i32, token_mask, loss_f32, scale_f32, tokens, experts);
    });
    return launched("balance_loss launch", launch);
  }
  uint32_t* ticket = (uint32_t*)workspace;
  BalPartial* partial = (BalPartial*)((uint8_t*)workspace + 16);
  cudaError_t e = cudaMemsetAsync(ticket, 0, sizeof(uint32_t), stream);
  if (e != cudaSuccess) return fail_cuda("balance_loss memset", e);
  const uint32_t grid = balance_blocks(tokens);
  balance_shape(dtype, aligned, experts, [&](auto element, auto access, auto per) {
    using T = decltype(element);
    launch = launch_dependent(netra_balance_loss_sm100<T, decltype(access)::value, decltype(per)::value>, dim3(grid), kBalThreads, 0, stream, 1,
                              (const T*)logits, pitch, counts_i32, token_mask, loss_f32, scale_f32, partial, ticket, tokens, experts);
  });
  return launched("balance_loss launch", launch);
}

int netra_balance_loss_grad_launch(void* grad, uint64_t grad_pitch, const void* logits, uint32_t dtype, uint64_t pitch, const int32_t* counts_i32,
                                   const uint8_t* token_mask, const float* scale_f32, const float* upstream_f32, uint64_t tokens,
                                   uint32_t experts, cudaStream_t stream) {
  if (int rc = balance_check("balance_loss_grad", logits, dtype, pitch, counts_i32, tokens, experts)) return rc;
  if (!grad || !scale_f32 || !upstream_f32) return fail("balance_loss_grad: null pointer");
  if (tokens > 1 && grad_pitch < experts) return fail("balance_loss_grad: a row pitch is smaller than the row");
  if ((uintptr_t)grad % dense_element_bytes(dtype)) return fail("balance_loss_grad: the gradient is not aligned to its element");
  if ((uintptr_t)scale_f32 % 4 || (uintptr_t)upstream_f32 % 4) return fail("balance_loss_grad: an address is not aligned to its element");
  const uint32_t grid = balance_blocks(tokens);
  const bool aligned = balance_aligned(logits, pitch, dtype, experts) && balance_aligned(grad, grad_pitch, dtype, experts);
  cudaError_t launch = cudaSuccess;
  balance_shape(dtype, aligned, experts, [&](auto element, auto access, auto per) {
    using T = decltype(element);
    launch = launch_dependent(netra_balance_loss_grad_sm100<T, decltype(access)::value, decltype(per)::value>, dim3(grid), kBalThreads, 0, stream, 1,
                              (T*)grad, grad_pitch, (const T*)logits, pitch, counts_i32, token_mask, scale_f32, upstream_f32, tokens, experts);
  });
  return launched("balance_loss_grad launch", launch);
}

}  // extern "C"
