// The dense block-scaled FP8 linear map, the operation the compiler's dense contract names
// (compiler/netra_compiler/contracts.py:175-284): E4M3 codes with one FP32 scale per row and 128 columns on the left, per
// 128 x 128 block on the right, FP32 accumulation.
//
//   quantise   s[m,b] = max(amax |x[m, block b]|, 1e-10) * fl(1/448),  a = e4m3_rne_sat(x * fl(1/s))      (the layer's quantiser)
//   product    y[m,n] = sum_b  sa[m,b] * sw[n/128,b] * sum_{k in b} a[m,k] w[n,k]
//   gradient   dx[m,k] = sum_b sg[m,b] * sw[b,k/128] * sum_{n in b} g[m,n] w[n,k]      (w read as it is stored)
//
// Any M, N, K: codes need 16-byte row pitches (TMA), everything else is masked.  K-blocks are added in ascending order but for few
// rows (parts by warp) and tiles split over a cluster (parts by CTA), whose parts are joined in a fixed order.
#include <type_traits>

namespace netra {

enum : uint32_t { kDenseBf16 = 0, kDenseF16 = 1, kDenseF32 = 2 };

// Where a bounded wait of a dense kernel ran out (kStatus* codes); read by netra_dense_status, which moves the words into
// g_dense_taken in one step each, so that a code written meanwhile is there for the next reading.
__device__ uint32_t g_dense_status[4];
__device__ uint32_t g_dense_taken[4];

extern "C" __global__ void netra_dense_take_status_sm100() { g_dense_taken[threadIdx.x] = atomicExch(&g_dense_status[threadIdx.x], 0u); }

__device__ __forceinline__ float dense_load(const void* p, uint32_t dtype, size_t i) {
  if (dtype == kDenseBf16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
  if (dtype == kDenseF16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void dense_store(void* p, uint32_t dtype, size_t i, float v) {
  if (dtype == kDenseBf16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (dtype == kDenseF16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<float*>(p)[i] = v;
}

// The kernels here are launched while the kernel before them on the stream may still be running (programmatic dependent
// launch): their launch, and the set-up of barriers and TMEM, overlap its end.  Every access to global memory comes after
// begin_grid(), which waits until that kernel has completed and its writes are visible - stream order, as for any launch - and
// lets the next such launch come as early.  Inputs may therefore be written while the grid already exists: no pointer here is
// declared __restrict__ and nothing is read through the non-coherent path, whose data may not change in a kernel's lifetime.
__device__ __forceinline__ void begin_grid() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------------------------------------
// Row quantiser.  Sixteen lanes own one block of 128 columns of kRows neighbouring rows, eight neighbouring columns each: a
// BF16 lane loads 16 bytes and stores 8 codes.  HBM bound; the four rows of the large form keep four loads in flight per
// lane, and let one lane store the block's four scales side by side (scales are stored block by block).
// Scales go to scale[m * scale_row + b * scale_block].  kVector: eight columns are one aligned access and lie wholly inside
// or outside the row.
// 16384 x 2048: FP32 25.5 us = 6.6 TB/s, BF16 18.3 us = 5.6 TB/s (two rows a lane: 25.1 and 19.6 us, eight: 27.5 and 25.3 us).
// ------------------------------------------------------------------------------------------
template <typename T> struct DenseElement;
template <> struct DenseElement<__nv_bfloat16> { static constexpr uint32_t code = kDenseBf16; };
template <> struct DenseElement<__half> { static constexpr uint32_t code = kDenseF16; };
template <> struct DenseElement<float> { static constexpr uint32_t code = kDenseF32; };

// Eight neighbouring elements as they are in memory: 16-bit ones take half the registers until their scale is known (the few-row
// product at 1 x 2048 x 4096: 4.0 -> 3.7 us).
template <typename T>
struct Eight {
  static constexpr bool kWide = sizeof(T) == 4;
  uint4 raw[kWide ? 2 : 1];
  // p is 16-byte aligned
  __device__ __forceinline__ void load(const T* p) {
    raw[0] = reinterpret_cast<const uint4*>(p)[0];
    if constexpr (kWide) raw[1] = reinterpret_cast<const uint4*>(p)[1];
  }
  __device__ __forceinline__ void clear() {
    raw[0] = make_uint4(0, 0, 0, 0);
    if constexpr (kWide) raw[1] = raw[0];
  }
  // the first `left` elements at p, on any boundary, and zeros behind them
  __device__ __forceinline__ void load(const T* p, int left) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (kWide) w[j] = j < left ? __float_as_uint(p[j]) : 0u;
      else w[j] = j < left ? reinterpret_cast<const uint16_t*>(p)[j] : 0u;
    }
    if constexpr (kWide) {
      raw[0] = make_uint4(w[0], w[1], w[2], w[3]);
      raw[1] = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
      raw[0] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
  }
  // In FP32: maxima of packed 16-bit pairs gained 7 % on the largest quantiser calls (16384 x 2048 BF16: 18.2 -> 16.9 us), but cost the
  // latency-bound ones more (1024 x 4096: 2.9 -> 3.6 us, the few-row product at 8 x 4096 x 2048: 4.4 -> 5.6 us).
  __device__ __forceinline__ float amax() const {
    float v[8];
    values(v);
    float m = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
    return m;
  }
  __device__ __forceinline__ void values(float v[8]) const {
    if constexpr (kWide) {
      const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    } else {
      const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (std::is_same<T, __half>::value) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          v[2 * j] = f.x; v[2 * j + 1] = f.y;
        } else {
          v[2 * j] = bf16_bits_to_f32(w[j] & 0xffffu); v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
      }
    }
  }
};

template <typename T, bool kVector, int kRows>
__global__ void __launch_bounds__(256)
netra_dense_quantize_rows_sm100(const T* x, uint64_t x_pitch, uint8_t* codes, uint64_t codes_pitch,
                                float* scale, uint64_t scale_row, uint64_t scale_block, uint32_t m, uint32_t k) {
  begin_grid();
  const uint32_t blocks = (k + kBlock - 1) / kBlock;
  const uint32_t item = (blockIdx.x * 256u + threadIdx.x) >> 4;
  const uint32_t group = item / blocks, b = item - group * blocks;
  const uint64_t row0 = (uint64_t)group * kRows;
  const uint32_t col = b * kBlock + (threadIdx.x & 15) * 8;
  Eight<T> x8[kRows];
  float s[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const T* src = x + (row0 + r) * x_pitch + col;
    if (row0 + r >= m || col >= k) x8[r].clear();
    else if (kVector) x8[r].load(src);
    else x8[r].load(src, (int)min(8u, k - col));
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    float amax = fmaxf(x8[r].amax(), amax_floor());
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    s[r] = amax * inv448();
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (row0 + r >= m) break;
    const float inv = 1.0f / s[r];
    float v[8];
    x8[r].values(v);
    uint8_t* dst = codes + (row0 + r) * codes_pitch + col;
    const uint32_t lo = f32x4_to_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    const uint32_t hi = f32x4_to_e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    if (kVector) {
      if (col < k) *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < k) dst[j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
    }
  }
  if ((threadIdx.x & 15) == 0) {
    float* dst = scale + row0 * scale_row + b * scale_block;
    if (kRows == 4 && scale_row == 1 && row0 + 4 <= m && (uintptr_t)dst % 16 == 0) {
      *reinterpret_cast<float4*>(dst) = make_float4(s[0], s[1 % kRows], s[2 % kRows], s[3 % kRows]);
    } else {
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (row0 + r < m) dst[r * scale_row] = s[r];
    }
  }
}

__device__ __forceinline__ uint32_t pack_16bit(uint32_t dtype, float a, float b) {
  if (dtype == kDenseF16) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// ------------------------------------------------------------------------------------------
// Product on the tensor cores.  A cluster owns 128 rows x kBN columns of the output and splits the K-blocks among
// its CTAs; per K-block the raw sums leave TMEM and are promoted as acc = fma(part, sa * sw, acc), as in the grouped GEMMs.
//   warps 0 and 2: TMA producers (rows, weight), warps 1 and 3: MMA issuers (alternate K-blocks; warp 1 owns TMEM),
//   warps 4..11: promotion (two groups halve the columns)
// With the few K-blocks a CTA has here, what costs is the chain of steps of one thread: a K-block took 750 cycles with one
// producer and one issuer (two barrier waits, four MMAs, two commits), whatever the tile's width.
// At the end every CTA hands each row of its FP32 partial tile to the cluster's CTA that owns the row (stores into that CTA's
// shared memory), which adds the parts in rank order: deterministic, and one cluster barrier.
// ------------------------------------------------------------------------------------------
constexpr int kDnThreads = 384;

template <int kBN>
struct DnCfg {
  static constexpr int kABytes = 128 * kBlock;
  static constexpr int kBBytes = kBN * kBlock;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = kBN >= 128 ? 4 : 6;
  static constexpr int kAccStages = 4;
  static_assert(kStages >= kAccStages, "a stage's barrier may not run two phases ahead of the promotion");
  static constexpr int kTmemCols = kAccStages * kBN;
  static constexpr int kOutPitch = kBN + 4;            // floats; 16-byte row stores fall on different banks
  static constexpr int kOutBytes = 128 * kOutPitch * 4;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kOutBytes + 256;
  static_assert(kSmemBytes <= 232448, "exceeds the shared memory of one SM");
};

struct DnArgs {
  const float* a_scale;
  uint64_t a_scale_row, a_scale_block;
  const float* w_scale;
  uint64_t w_scale_col, w_scale_block;    // per 128 output columns, per K-block
  void* out;
  uint64_t out_pitch;
  uint32_t out_dtype, out_vector;         // out_vector 1: four neighbouring elements are one aligned access; 2: rows start on 32-byte boundaries
  uint32_t m, n, k_blocks;                // rows, output columns, K-blocks
  uint32_t n_tiles;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ int ld_cluster_i32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_b64(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_f4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

__device__ __forceinline__ void prefetch_tensormap(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)map) : "memory"); }

// one look at a barrier by a whole warp
__device__ __forceinline__ bool mbar_try_wait_warp(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "vote.sync.all.pred p, p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag) {
  for (uint32_t spin = 0; spin < kSpinLimit; ++spin) {
    if (mbar_try_wait_warp(bar, parity)) return true;
    if ((spin & 0xff) == 0xff && __any_sync(0xffffffffu, *abort_flag != 0)) return false;
  }
  return false;
}

// MN-major, 128-byte-swizzled operand tile: 128 output columns (bytes) per row, one row per reduction index; groups of
// eight rows are 1,024 bytes apart.
__device__ __forceinline__ uint64_t make_smem_desc_mn(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(1024 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// kTransposed: the weight tile is [128 reduction rows][128 output columns] as stored, an MN-major B operand.
template <int kBN, bool kTransposed>
__global__ void __launch_bounds__(kDnThreads, 1)
netra_dense_fp8_matmul_sm100(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w, const DnArgs g) {
  using C = DnCfg<kBN>;
  static_assert(!kTransposed || kBN == 128, "a transposed weight tile is one 128-byte swizzle atom wide");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* parts = reinterpret_cast<float*>(smem + C::kStages * C::kStageBytes);      // [ranks][128 / ranks rows][kOutPitch]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + C::kStages * C::kStageBytes + C::kOutBytes);
  uint64_t* done_bar = full_bar + C::kStages;          // the MMAs that read the stage are done
  uint64_t* tempty_bar = done_bar + C::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + C::kAccStages);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const uint32_t tile = blockIdx.x / ranks;
  const uint32_t row0 = (tile / g.n_tiles) * 128u, col0 = (tile % g.n_tiles) * (uint32_t)kBN;
  // a whole tile of one CTA, its rows on 32-byte boundaries, goes straight from the registers to memory
  const bool direct = ranks == 1 && g.out_vector == 2 && col0 + kBN <= g.n;
  const uint32_t kb0 = (uint32_t)((uint64_t)g.k_blocks * rank / ranks), kb1 = (uint32_t)((uint64_t)g.k_blocks * (rank + 1) / ranks);

  if (threadIdx.x == 0 || threadIdx.x == 64) prefetch_tensormap(threadIdx.x == 0 ? &tm_a : &tm_w);
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) { mbar_init(smem_u32(&full_bar[s]), 2); mbar_init(smem_u32(&done_bar[s]), 1); }
    for (int a = 0; a < C::kAccStages; ++a) mbar_init(smem_u32(&tempty_bar[a]), 8);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (ranks > 1) cluster_arrive();          // this CTA is running: others may store into its shared memory
  begin_grid();                             // nothing above touches global memory

  if ((warp == 0 || warp == 2) && lane == 0) {
    const uint64_t pol = policy_evict_last();
    const bool rows = warp == 0;
    for (uint32_t kb = kb0; kb < kb1; ++kb) {
      const uint32_t it = kb - kb0, s = it % C::kStages;
      if (it >= C::kStages && !mbar_wait(smem_u32(&done_bar[s]), ((it / C::kStages) & 1) ^ 1, abort_flag)) {
        g_dense_status[0] = kStatusProducerTimeout; *abort_flag = 1; break;
      }
      const uint32_t bar = smem_u32(&full_bar[s]), dst = smem_u32(smem + s * C::kStageBytes);
      mbar_expect_tx(bar, rows ? C::kABytes : C::kBBytes);
      if (rows) tma_load_2d(dst, &tm_a, bar, (int)(kb * kBlock), (int)row0, pol);
      else if (kTransposed) tma_load_2d(dst + C::kABytes, &tm_w, bar, (int)col0, (int)(kb * kBlock), pol);
      else tma_load_2d(dst + C::kABytes, &tm_w, bar, (int)(kb * kBlock), (int)col0, pol);
    }
  } else if ((warp == 1 || warp == 3) && lane == 0) {
    const uint32_t idesc = make_idesc(kBN) | (kTransposed ? 1u << 16 : 0u);
    for (uint32_t it = (uint32_t)warp >> 1; it < kb1 - kb0; it += 2) {
      const uint32_t s = it % C::kStages, a = it % C::kAccStages;
      if (!mbar_wait(smem_u32(&full_bar[s]), (it / C::kStages) & 1, abort_flag) ||
          (it >= C::kAccStages && !mbar_wait(smem_u32(&tempty_bar[a]), ((it / C::kAccStages) & 1) ^ 1, abort_flag))) {
        g_dense_status[0] = kStatusMmaTimeout; *abort_flag = 1; break;
      }
      tc_fence_after();
      const uint32_t sa = smem_u32(smem + s * C::kStageBytes);
      const uint64_t adesc = make_smem_desc(sa);
      const uint64_t bdesc = kTransposed ? make_smem_desc_mn(sa + C::kABytes) : make_smem_desc(sa + C::kABytes);
#pragma unroll
      for (int k = 0; k < kBlock / 32; ++k)
        umma_f8(tmem_base + a * kBN, adesc + 2 * k, bdesc + (kTransposed ? 256 : 2) * k, idesc, k > 0);
      umma_commit(smem_u32(&done_bar[s]));
    }
  } else if (warp >= 4) {
    constexpr int kCols = kBN / 2;                      // columns of this thread
    const int wg = (warp - 4) >> 2, quad = warp & 3;
    const uint32_t r = (uint32_t)(quad * 32 + lane), row = row0 + r;
    const float* sa_ptr = g.a_scale + (uint64_t)min(row, g.m - 1) * g.a_scale_row;
    const float* sw_ptr = g.w_scale + (uint64_t)((col0 + wg * kCols) / kBlock) * g.w_scale_col;
    if ((col0 + wg * kCols) >= g.n) sw_ptr = g.w_scale;         // columns past the end: nothing is stored
    float acc[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[c] = 0.0f;
    // scales of eight K-blocks at a time, the next eight asked for while the second of these is promoted: one at a time, their
    // latency set the loop's pace
    float sa[8], sw[8], sa_next[8], sw_next[8];
    auto load_scales = [&](float to_a[8], float to_w[8], uint32_t from) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t kb = min(from + j, g.k_blocks - 1);
        to_a[j] = __ldcg(sa_ptr + kb * g.a_scale_block);
        to_w[j] = __ldcg(sw_ptr + kb * g.w_scale_block);
      }
    };
    load_scales(sa, sw, kb0);
    bool ok = true;
    for (uint32_t base = kb0; ok && base < kb1; base += 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!ok || base + j >= kb1) break;
        if (j == 1 && base + 8 < kb1) load_scales(sa_next, sw_next, base + 8);
        const float s = __fmul_rn(sa[j], sw[j]);
        const uint32_t it = base + j - kb0, a = it % C::kAccStages;
        if (!mbar_wait_warp(smem_u32(&done_bar[it % C::kStages]), (it / C::kStages) & 1, abort_flag)) {
          g_dense_status[0] = kStatusEpilogueTimeout; *abort_flag = 1; ok = false; break;
        }
        tc_fence_after();
        const uint32_t t = tmem_base + ((uint32_t)(quad * 32) << 16) + a * kBN + wg * kCols;
        uint32_t v[kCols / 32][32];
#pragma unroll
        for (int q = 0; q < kCols / 32; ++q) tmem_ld32_nowait(t + 32 * q, v[q]);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&tempty_bar[a]));
#pragma unroll
        for (int q = 0; q < kCols / 32; ++q)
#pragma unroll
          for (int c = 0; c < 32; ++c) acc[32 * q + c] = fmaf(__uint_as_float(v[q][c]), s, acc[32 * q + c]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) { sa[j] = sa_next[j]; sw[j] = sw_next[j]; }
    }
    if (direct) {
      if (row < g.m) {
        const uint64_t at = (uint64_t)row * g.out_pitch + col0 + wg * kCols;
        if (g.out_dtype == kDenseF32) {
#pragma unroll
          for (int c = 0; c < kCols; c += 8) st_global_v8(reinterpret_cast<float*>(g.out) + at + c, acc + c);
        } else {
#pragma unroll
          for (int c = 0; c < kCols; c += 16) {
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = __uint_as_float(pack_16bit(g.out_dtype, acc[c + 2 * j], acc[c + 2 * j + 1]));
            st_global_v8(reinterpret_cast<float*>(reinterpret_cast<uint16_t*>(g.out) + at + c), p);
          }
        }
      }
    } else {
      __syncwarp();
      if (ranks > 1) cluster_wait();
      // row r belongs to the CTA of rank r / (128 / ranks)
      const uint32_t share = 128u / ranks;
      const uint32_t dst = map_to_rank(smem_u32(parts + ((size_t)(rank * share + r % share) * C::kOutPitch + wg * kCols)), r / share);
#pragma unroll
      for (int c = 0; c < kCols; c += 4) st_cluster_f4(dst + 4 * c, acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
    }
  }
  __syncwarp();
  if (warp < 4 && ranks > 1) cluster_wait();

  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) __nanosleep(200000);   // copies in flight land before the CTA goes on
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
  if (direct) return;
  __syncwarp();
  if (ranks > 1) cluster_barrier();         // every part is in its owner's shared memory, and nothing reaches into a CTA after it
  const uint32_t share = 128u / ranks, first = row0 + rank * share;
  if (first >= g.m) return;
  const uint32_t count = min(share, g.m - first);
  if (g.out_vector && col0 + kBN <= g.n) {
    // a quarter, half or whole warp takes a row, a lane four neighbouring columns
    constexpr uint32_t kLanes = kBN / 4, kRowsAtOnce = kDnThreads / kLanes;
    const uint32_t c = (threadIdx.x % kLanes) * 4;
#pragma unroll 4
    for (uint32_t r = threadIdx.x / kLanes; r < count; r += kRowsAtOnce) {
      const float* p = parts + (size_t)r * C::kOutPitch + c;
      float4 v = *reinterpret_cast<const float4*>(p);
      for (uint32_t j = 1; j < ranks; ++j) {
        const float4 q = *reinterpret_cast<const float4*>(p + (size_t)j * share * C::kOutPitch);
        v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
      }
      const uint64_t at = (uint64_t)(first + r) * g.out_pitch + col0 + c;
      if (g.out_dtype == kDenseF32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(g.out) + at) = v;
      else *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(g.out) + at) = make_uint2(pack_16bit(g.out_dtype, v.x, v.y), pack_16bit(g.out_dtype, v.z, v.w));
    }
  } else {
    // rows on any boundary, or a tile that ends inside: neighbouring lanes store neighbouring elements
    const uint32_t cols = min((uint32_t)kBN, g.n - col0);
    constexpr int kRowsAtOnce = 4, kPerLane = kBN / 32, kWarps = kDnThreads / 32;
    auto store_rows = [&](auto element) {
      using T = decltype(element);
      T* to = reinterpret_cast<T*>(g.out) + (uint64_t)first * g.out_pitch + col0 + lane;
      for (uint32_t r0 = warp; r0 < count; r0 += kRowsAtOnce * kWarps) {
        float v[kRowsAtOnce][kPerLane];
        const float* p = parts + (size_t)r0 * C::kOutPitch + lane;
#pragma unroll
        for (int i = 0; i < kRowsAtOnce; ++i)
#pragma unroll
          for (int j = 0; j < kPerLane; ++j) v[i][j] = r0 + i * kWarps < share ? p[i * kWarps * C::kOutPitch + 32 * j] : 0.0f;
        for (uint32_t q = 1; q < ranks; ++q) {
          p += (size_t)share * C::kOutPitch;
#pragma unroll
          for (int i = 0; i < kRowsAtOnce; ++i)
#pragma unroll
            for (int j = 0; j < kPerLane; ++j)
              if (r0 + i * kWarps < share) v[i][j] += p[i * kWarps * C::kOutPitch + 32 * j];
        }
#pragma unroll
        for (int i = 0; i < kRowsAtOnce; ++i) {
          if (r0 + i * kWarps >= count) break;
#pragma unroll
          for (int j = 0; j < kPerLane; ++j)
            if (lane + 32 * j < cols) dense_store(to + (uint64_t)(r0 + i * kWarps) * g.out_pitch, DenseElement<T>::code, 32 * j, v[i][j]);
        }
      }
    };
    if (g.out_dtype == kDenseF32) store_rows(0.0f);
    else if (g.out_dtype == kDenseF16) store_rows(__half{});
    else store_rows(__nv_bfloat16{});
  }
}

}  // namespace netra

#include "dense_pair.cu"
#include "dense_few.cu"

namespace {

// Launch as a programmatic dependent of the kernel before it (the kernel calls begin_grid); cluster = 1: no cluster.
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, uint32_t block, size_t smem, cudaStream_t stream, uint32_t cluster, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.gridDim = grid; cfg.blockDim = dim3(block); cfg.dynamicSmemBytes = smem;
  cfg.stream = stream; cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
int launched(const char* what, cudaError_t e) { return e == cudaSuccess ? check_launch(what) : fail_cuda(what, e); }

uint64_t dense_element_bytes(uint32_t dtype) { return dtype == kDenseF32 ? 4 : 2; }

// Byte tensor of `rows` rows of `cols` codes, `pitch` bytes apart; box 128 bytes x box_rows, 128-byte swizzle.
int encode_codes(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return fail("cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {pitch};
  cuuint32_t box[2] = {128, box_rows};
  cuuint32_t elem[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    snprintf(g_error, sizeof g_error, "cuTensorMapEncodeTiled (FP8 codes) failed with CUresult %d", (int)r);
    return -1;
  }
  return 0;
}

// Output matrix of 2- or 4-byte elements; box 128 bytes x 32 rows, 128-byte swizzle.
int encode_output(CUtensorMap* map, void* base, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t element_bytes) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return fail("cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {pitch * element_bytes};
  cuuint32_t box[2] = {128 / element_bytes, 32};
  cuuint32_t elem[2] = {1, 1};
  CUresult r = fn(map, element_bytes == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base, dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    snprintf(g_error, sizeof g_error, "cuTensorMapEncodeTiled (output) failed with CUresult %d", (int)r);
    return -1;
  }
  return 0;
}

std::mutex g_dense_mutex, g_dense_taken_mutex;
bool g_dense_pair_ok[kMaxDevices] = {};   // the pair kernels were built with the register allocation they assume
int g_dense_sms[kMaxDevices] = {};      // SM count once the kernels of a device are set up

int dense_setup(int* sms, bool* pair_ok) {
  int device = 0;
  if (int rc = current_device_index(&device)) return rc;
  std::lock_guard<std::mutex> lock(g_dense_mutex);
  if (g_dense_sms[device] == 0) {
    int major = 0, count = 0;
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
    if (major != 10) return fail("this library targets sm_100a (compute capability 10.x)");
    cudaError_t e = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(netra_dense_fp8_matmul_sm100<64, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, DnCfg<64>::kSmemBytes);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(netra_dense_fp8_matmul_sm100<128, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, DnCfg<128>::kSmemBytes);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(netra_dense_fp8_matmul_sm100<128, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, DnCfg<128>::kSmemBytes);
    // the register re-balancing inside the pair kernels is only deadlock-free for the launch allocation it was written for
    bool ok = true;
    auto pair = [&](const void* kernel) {
      cudaFuncAttributes a;
      if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg::kSmemBytes);
      if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, kernel);
      if (e == cudaSuccess) ok = ok && a.numRegs == kPairRegsLaunch;
    };
    pair((const void*)netra_dense_fp8_pair_sm100<false, __nv_bfloat16>);
    pair((const void*)netra_dense_fp8_pair_sm100<false, __half>);
    pair((const void*)netra_dense_fp8_pair_sm100<false, float>);
    pair((const void*)netra_dense_fp8_pair_sm100<true, __nv_bfloat16>);
    pair((const void*)netra_dense_fp8_pair_sm100<true, __half>);
    pair((const void*)netra_dense_fp8_pair_sm100<true, float>);
    if (e != cudaSuccess) return fail_cuda("dense set-up", e);
    g_dense_pair_ok[device] = ok;
    g_dense_sms[device] = count;
  }
  *sms = g_dense_sms[device];
  *pair_ok = g_dense_pair_ok[device];
  return 0;
}

constexpr uint32_t kDenseMaxSize = 1u << 26;
constexpr uint32_t kFewMaxRows = 16, kFewMaxCodeRows = 32;

// Product of few rows; x of type code `source` (kDense*, or 3 for codes with their scales).
int launch_few(const FewArgs& g, uint32_t source, int sms, cudaStream_t stream) {
  // One K-block a warp where every CTA has an SM to itself (16 x 1024 x 1024: 2.7 us, with two a warp 3.4 us), two where they share
  // (16 x 4096 x 2048: 5.6 us with one, 4.4 us with two).  Sixteen warps at most, or eight where more CTAs follow, whose starts then
  // overlap the others' ends (1 x 8192 x 8192: 17.9 us with sixteen, 16.0 us with eight).
  const uint32_t blocks = (g.k + 127) / 128, ctas = (g.n + kFewRows - 1) / kFewRows;
  const uint32_t most = ctas > 2u * (uint32_t)sms ? 8 : 16, wanted = ctas <= (uint32_t)sms ? blocks : (blocks + 1) / 2;
  const uint32_t warps = wanted < most ? wanted : most;
  const uint32_t tiles = g.m <= 8 ? 1 : g.m <= 16 ? 2 : 4;
  const dim3 grid(ctas);
  const size_t smem = warps * tiles * 8 * kFewRows * sizeof(float);
  auto launch = [&](auto element) {
    using T = decltype(element);
    if constexpr (sizeof(T) == 1) {
      if (tiles == 4) return launch_dependent(netra_dense_fp8_few_sm100<T, 4>, grid, 32 * warps, smem, stream, 1, g);
    }
    return launch_dependent(tiles == 1 ? netra_dense_fp8_few_sm100<T, 1> : netra_dense_fp8_few_sm100<T, 2>, grid, 32 * warps, smem, stream, 1, g);
  };
  const cudaError_t e = source == 3 ? launch((uint8_t)0) : source == kDenseF32 ? launch(0.0f) : source == kDenseF16 ? launch(__half{}) : launch(__nv_bfloat16{});
  return launched("dense_fp8 launch (few rows)", e);
}


int check_quantize_operands(const void* x, uint32_t dtype, uint64_t x_pitch, uint32_t m, uint32_t k) {
  if (!x) return fail("dense_quantize_rows: null pointer");
  if (dtype > kDenseF32) return fail("dense_quantize_rows: unknown element type");
  if (m == 0 || k == 0 || m > kDenseMaxSize || k > kDenseMaxSize) return fail("dense_quantize_rows: rows and columns must be 1..2^26");
  if (m > 1 && x_pitch < k) return fail("dense_quantize_rows: a row pitch is smaller than the row");
  if ((uintptr_t)x % dense_element_bytes(dtype)) return fail("dense_quantize_rows: input is not aligned to its element");
  return 0;
}

int check_matmul_operands(const void* out, uint32_t out_dtype, uint64_t out_pitch, const void* w, uint64_t w_pitch, const float* w_scale,
                          uint64_t w_scale_pitch, uint32_t transpose_w, uint32_t m, uint32_t w_rows, uint32_t w_cols) {
  if (!out || !w || !w_scale) return fail("dense_fp8_matmul: null pointer");
  if (out_dtype > kDenseF32) return fail("dense_fp8_matmul: unknown element type");
  if (transpose_w > 1) return fail("dense_fp8_matmul: transpose_w must be 0 or 1");
  if (m == 0 || w_rows == 0 || w_cols == 0 || m > kDenseMaxSize || w_rows > kDenseMaxSize || w_cols > kDenseMaxSize)
    return fail("dense_fp8_matmul: sizes must be 1..2^26");
  if (w_pitch % 16 || (uintptr_t)w % 16) return fail("dense_fp8_matmul: codes need 16-byte aligned addresses and row pitches");
  if (w_pitch < w_cols || out_pitch < (transpose_w ? w_cols : w_rows) || w_scale_pitch < (w_cols + 127) / 128)
    return fail("dense_fp8_matmul: a row pitch is smaller than the row");
  if ((uintptr_t)out % dense_element_bytes(out_dtype) || (uintptr_t)w_scale % 4)
    return fail("dense_fp8_matmul: an address is not aligned to its element");
  return 0;
}

}  // namespace

extern "C" {

int netra_dense_quantize_rows_launch(void* codes_fp8, uint64_t codes_pitch, float* scale_f32, uint64_t scale_row_stride,
                                     uint64_t scale_block_stride, const void* x, uint32_t x_dtype, uint64_t x_pitch, uint32_t m,
                                     uint32_t k, cudaStream_t stream) {
  if (!codes_fp8 || !scale_f32) return fail("dense_quantize_rows: null pointer");
  if (int rc = check_quantize_operands(x, x_dtype, x_pitch, m, k)) return rc;
  if ((uintptr_t)scale_f32 % 4) return fail("dense_quantize_rows: the scales are not aligned to their element");
  if (m > 1 && codes_pitch < k) return fail("dense_quantize_rows: a row pitch is smaller than the row");
  const uint64_t blocks = (k + 127) / 128;
  // four rows per lane once that still leaves every SM a few thousand lanes; below, one row each for the shortest chain
  const bool deep = (uint64_t)m * blocks >= 32768;
  const uint64_t grid = ((deep ? (m + 3) / 4 : m) * blocks + 15) / 16;
  if (grid > 0x00ffffffull) return fail("dense_quantize_rows: too many blocks of 128 in one call");
  const bool vector = k % 8 == 0 && (uintptr_t)x % 16 == 0 && (x_pitch * dense_element_bytes(x_dtype)) % 16 == 0 &&
                      (uintptr_t)codes_fp8 % 8 == 0 && codes_pitch % 8 == 0;
  auto launch = [&](auto element, auto vec, auto rows) {
    using T = decltype(element);
    return launch_dependent(netra_dense_quantize_rows_sm100<T, decltype(vec)::value, decltype(rows)::value>, dim3((unsigned)grid), 256, 0, stream, 1,
                            (const T*)x, x_pitch, (uint8_t*)codes_fp8, codes_pitch, scale_f32, scale_row_stride, scale_block_stride, m, k);
  };
  auto shape = [&](auto element) {
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 1> one;
    if (vector) return deep ? launch(element, std::true_type{}, four) : launch(element, std::true_type{}, one);
    return deep ? launch(element, std::false_type{}, four) : launch(element, std::false_type{}, one);
  };
  return launched("dense_quantize_rows launch", x_dtype == kDenseBf16 ? shape(__nv_bfloat16{}) : x_dtype == kDenseF16 ? shape(__half{}) : shape(0.0f));
}

int netra_dense_fp8_matmul_launch(void* out, uint32_t out_dtype, uint64_t out_pitch, const void* a_fp8, uint64_t a_pitch,
                                  const float* a_scale_f32, uint64_t a_scale_row_stride, uint64_t a_scale_block_stride,
                                  const void* w_fp8, uint64_t w_pitch, const float* w_scale_f32, uint64_t w_scale_pitch,
                                  uint32_t transpose_w, uint32_t m, uint32_t w_rows, uint32_t w_cols, cudaStream_t stream) {
  if (!a_fp8 || !a_scale_f32) return fail("dense_fp8_matmul: null pointer");
  if (int rc = check_matmul_operands(out, out_dtype, out_pitch, w_fp8, w_pitch, w_scale_f32, w_scale_pitch, transpose_w, m, w_rows, w_cols)) return rc;
  const uint32_t n = transpose_w ? w_cols : w_rows, k = transpose_w ? w_rows : w_cols;
  if (a_pitch % 16 || (uintptr_t)a_fp8 % 16) return fail("dense_fp8_matmul: codes need 16-byte aligned addresses and row pitches");
  if (a_pitch < k) return fail("dense_fp8_matmul: a row pitch is smaller than the row");
  if ((uintptr_t)a_scale_f32 % 4) return fail("dense_fp8_matmul: an address is not aligned to its element");
  int sms = 0;
  bool pair_ok = false;
  if (int rc = dense_setup(&sms, &pair_ok)) return rc;
  // Few rows: 16 x 4096 x 2048 4.4 us against 7.4 us on the tensor-core tiles.  More than sixteen are read again by every CTA, which
  // pays while each has an SM to itself and the weight is small (17 x 2048 x 2048: 4.1 us against 7.1 us, 32 x 512 x 1024: 3.7 us
  // against 4.1 us; but 32 x 2048 x 4096 7.6 us against 7.3 us, 32 x 4096 x 4096 13.3 us against 9.1 us).
  if (!transpose_w && (m <= kFewMaxRows || (m <= kFewMaxCodeRows && n <= (uint32_t)sms * kFewRows && (uint64_t)n * k <= (1u << 22)))) {
    const FewArgs f = {a_fp8, a_pitch, a_scale_f32, a_scale_row_stride, a_scale_block_stride, (const uint8_t*)w_fp8, w_pitch, w_scale_f32,
                       w_scale_pitch, out, out_pitch, out_dtype, m, n, k};
    return launch_few(f, 3, sms, stream);
  }
  CUtensorMap tm_a, tm_w;
  if (int rc = encode_codes(&tm_a, a_fp8, m, k, a_pitch, 128)) return rc;
  const uint64_t m256 = (m + 255) / 256, n256 = (n + 255) / 256;
  // Pairs once one CTA per 128 x 128 tile no longer fits the device at once: 1024 x 2048 x 2048 (128 tiles) 10.4 us in one wave of
  // single CTAs against 11.7 us in pairs, 1024 x 2560 x 2048 (160 tiles) 17.0 us against 12.4 us.
  if (pair_ok && (uint64_t)((m + 127) / 128) * ((n + 127) / 128) > (uint64_t)sms) {
    if (m256 * n256 > 0x7fffffffull) return fail("dense_fp8_matmul: too many output tiles in one call");
    PairArgs p;
    p.a_scale = a_scale_f32; p.a_scale_row = a_scale_row_stride; p.a_scale_block = a_scale_block_stride;
    p.w_scale = w_scale_f32;
    p.w_scale_col = transpose_w ? 1 : w_scale_pitch; p.w_scale_block = transpose_w ? w_scale_pitch : 1;
    p.out = out; p.out_pitch = out_pitch;
    p.m = m; p.n = n; p.k_blocks = (k + 127) / 128; p.m_tiles = (uint32_t)m256; p.n_tiles = (uint32_t)n256;
    const uint32_t size = (uint32_t)dense_element_bytes(out_dtype);
    p.tma_store = (uintptr_t)out % 16 == 0 && out_pitch * size % 16 == 0;
    CUtensorMap tm_out = {};
    if (int rc = encode_codes(&tm_w, w_fp8, w_rows, w_cols, w_pitch, 128)) return rc;
    if (p.tma_store)
      if (int rc = encode_output(&tm_out, out, m, n, out_pitch, size)) return rc;
    const uint64_t pairs = m256 * n256 < (uint64_t)(sms / 2) ? m256 * n256 : (uint64_t)(sms / 2);
    auto launch = [&](auto element) {
      using T = decltype(element);
      return launch_dependent(transpose_w ? netra_dense_fp8_pair_sm100<true, T> : netra_dense_fp8_pair_sm100<false, T>, dim3((unsigned)(2 * pairs)),
                              kPairThreads, PairCfg::kSmemBytes, stream, 1, tm_a, tm_w, tm_out, p);
    };
    const cudaError_t e = out_dtype == kDenseF32 ? launch(0.0f) : out_dtype == kDenseF16 ? launch(__half{}) : launch(__nv_bfloat16{});
    return launched("dense_fp8_matmul launch", e);
  }
  DnArgs g;
  g.a_scale = a_scale_f32; g.a_scale_row = a_scale_row_stride; g.a_scale_block = a_scale_block_stride;
  g.w_scale = w_scale_f32;
  g.w_scale_col = transpose_w ? 1 : w_scale_pitch;
  g.w_scale_block = transpose_w ? w_scale_pitch : 1;
  g.out = out; g.out_pitch = out_pitch; g.out_dtype = out_dtype;
  const uint64_t out_bytes = dense_element_bytes(out_dtype);
  g.out_vector = ((uintptr_t)out | out_pitch * out_bytes) % 32 == 0 ? 2 : (uintptr_t)out % (4 * out_bytes) == 0 && out_pitch % 4 == 0 ? 1 : 0;
  g.m = m; g.n = n; g.k_blocks = (k + 127) / 128;
  const uint64_t m_tiles = (m + 127) / 128;
  // 64 columns a tile while that still is one wave (256 x 4096 x 2048: 9.1 us against 10.5 us with 128), or where there are no more
  // (16384 x 64 x 2048: 9.7 us against 11.9 us).  The gradient's weight tile is one swizzle atom of 128 columns.
  const bool narrow = !transpose_w && (n <= 64 || m_tiles * ((n + 127) / 128) * 2 <= (uint64_t)sms);
  const uint32_t bn = narrow ? 64 : 128;
  g.n_tiles = (n + bn - 1) / bn;
  const uint64_t tiles = m_tiles * g.n_tiles;
  uint32_t split = 1;
  // Eight K-blocks and more for every CTA of a cluster (128 x 1024 x 1024: 4.6 us as it is, 5.4 us in two, 6.0 us in four).  Clusters of
  // eight only where few are needed: a GPC holds two of them at one CTA an SM, and a second wave doubles the time (64 x 1024 x 4096:
  // sixteen clusters of eight 11.7 us, of four 6.6 us).
  while (split < (tiles <= 8 ? 8u : 4u) && tiles * split * 2 <= (uint64_t)sms && g.k_blocks >= split * 16) split *= 2;
  if (tiles * split > 0x7fffffffull) return fail("dense_fp8_matmul: too many output tiles in one call");
  if (int rc = encode_codes(&tm_w, w_fp8, w_rows, w_cols, w_pitch, transpose_w ? 128 : bn)) return rc;
  const dim3 grid((unsigned)(tiles * split));
  const cudaError_t e =
      transpose_w ? launch_dependent(netra_dense_fp8_matmul_sm100<128, true>, grid, kDnThreads, DnCfg<128>::kSmemBytes, stream, split, tm_a, tm_w, g)
      : narrow    ? launch_dependent(netra_dense_fp8_matmul_sm100<64, false>, grid, kDnThreads, DnCfg<64>::kSmemBytes, stream, split, tm_a, tm_w, g)
                  : launch_dependent(netra_dense_fp8_matmul_sm100<128, false>, grid, kDnThreads, DnCfg<128>::kSmemBytes, stream, split, tm_a, tm_w, g);
  return launched("dense_fp8_matmul launch", e);
}

// codes [m, k rounded up to 128] and, behind them, scales [ceil(k/128)][m].  Rows of codes on 128-byte boundaries: a box of a row
// that straddles two lines costs the copy engine both (777 x 1043 x 2064: 14.3 us with rows of 2,064 bytes, 12.2 us so).
uint64_t netra_dense_fp8_linear_workspace_bytes(uint32_t m, uint32_t k) {
  const uint64_t blocks = ((uint64_t)k + 127) / 128;
  return (uint64_t)m * blocks * (128 + 4);
}

uint32_t netra_dense_fp8_linear_needs_workspace(const void* x, uint32_t dtype, uint64_t x_pitch, uint32_t transpose_w, uint32_t m, uint32_t k) {
  // Few rows: the product quantises them itself, if whole 16-byte accesses fit them.  Every CTA reads all of them, so FP32 rows
  // pay up to four (4 x 4096 x 2048: 5.4 us against 5.9 us with the quantiser's launch, 8 rows 7.6 us against 6.0 us), 16-bit ones up
  // to sixteen (5.8 us against 6.3 us).
  return transpose_w || m > (dtype == kDenseF32 ? 4u : kFewMaxRows) || k % 8 != 0 || (uintptr_t)x % 16 != 0 ||
         x_pitch * dense_element_bytes(dtype) % 16 != 0;
}

int netra_dense_fp8_linear_launch(void* out, uint64_t out_pitch, const void* x, uint32_t dtype, uint64_t x_pitch, const void* w_fp8,
                                  uint64_t w_pitch, const float* w_scale_f32, uint64_t w_scale_pitch, uint32_t transpose_w, uint32_t m,
                                  uint32_t w_rows, uint32_t w_cols, void* workspace, uint64_t workspace_bytes, cudaStream_t stream) {
  const uint32_t k = transpose_w ? w_rows : w_cols;
  if (!netra_dense_fp8_linear_needs_workspace(x, dtype, x_pitch, transpose_w, m, k)) {
    if (int rc = check_quantize_operands(x, dtype, x_pitch, m, k)) return rc;
    if (int rc = check_matmul_operands(out, dtype, out_pitch, w_fp8, w_pitch, w_scale_f32, w_scale_pitch, transpose_w, m, w_rows, w_cols)) return rc;
    int sms = 0;
    bool pair_ok = false;
    if (int rc = dense_setup(&sms, &pair_ok)) return rc;
    const FewArgs f = {x, x_pitch, nullptr, 0, 0, (const uint8_t*)w_fp8, w_pitch, w_scale_f32, w_scale_pitch, out, out_pitch, dtype, m, w_rows, k};
    return launch_few(f, dtype, sms, stream);
  }
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < netra_dense_fp8_linear_workspace_bytes(m, k))
    return fail("dense_fp8_linear: workspace missing, too small or not 16-byte aligned");
  const uint64_t pitch = ((uint64_t)k + 127) / 128 * 128;
  uint8_t* codes = (uint8_t*)workspace;
  float* scale = (float*)(codes + (uint64_t)m * pitch);
  if (int rc = netra_dense_quantize_rows_launch(codes, pitch, scale, 1, m, x, dtype, x_pitch, m, k, stream)) return rc;
  return netra_dense_fp8_matmul_launch(out, dtype, out_pitch, codes, pitch, scale, 1, m, w_fp8, w_pitch, w_scale_f32, w_scale_pitch,
                                       transpose_w, m, w_rows, w_cols, stream);
}

int netra_dense_status(uint32_t status_out[4]) {
  if (status_out == nullptr) return fail("dense_status: null pointer");
  cudaError_t e = cudaDeviceSynchronize();       // the copy below is ordered behind the default stream only
  if (e != cudaSuccess) return fail_cuda("dense status", e);
  std::lock_guard<std::mutex> lock(g_dense_taken_mutex);
  netra_dense_take_status_sm100<<<1, 4>>>();
  if (int rc = check_launch("dense status launch")) return rc;
  e = cudaMemcpyFromSymbol(status_out, g_dense_taken, 16);
  return e == cudaSuccess ? 0 : fail_cuda("dense status", e);
}

}  // extern "C"
