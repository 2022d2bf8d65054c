// The dense block-scaled product for many rows: a pair of CTAs (cta_group::2) owns 256 rows x 256 columns of the output.
//
// Every K-block of 128 leaves 256 x 256 raw sums in TMEM which the CUDA cores scale by sa[row] * sw[tile] and add up in
// registers, so three things have to overlap: the tensor core (512 cycles a K-block), the operands (32 KB per CTA and
// K-block: a pair fetches its weight tile once, half each; one CTA alone would need 48 KB, more than the L2 delivers in that
// time) and the promotion (128 KB read out of TMEM and 32,768 multiply-adds per CTA).  What bounds it is the chain MMA ->
// commit -> promotion -> release -> MMA on an accumulator stage: 975 cycles per K-block with the stores (4736 x 4096 x 4096, the
// busiest pair), and no unit near its limit (57 % of the issue slots; half of shared memory, a quarter of the L2).  Hence:
//   * sixteen promotion warps, four per scheduler, hide latencies that eight cannot; a thread keeps 64 columns of its row;
//   * a K-block is multiplied and handed over in two halves of 128 columns, each with its own barriers (140 -> 133 us at
//     16384 x 4096 x 2048), by two issuing threads that take alternate K-blocks (151 -> 137 us);
//   * the scales go through shared memory, four K-blocks ahead: loaded by the promotion warps themselves, one K-block ahead,
//     they were what the loop waited for (172 -> 151 us).
// 16384 x 4096 x 2048: 130-133 us = 2.1 PFLOP/s in a burst, 157 us back to back for seconds (1,000 W cap, 1.59 GHz).
//
//   warp 0: TMA producer (each CTA its own 128 rows and its own 128 weight rows; both report to the leader's barrier)
//   warps 1 and 3: MMA issuers (leader CTA) or relays of the peer's releases (warp 1 also owns TMEM), warp 2: scales,
//   warps 4..19: promotion and store
// The grid is persistent; the accumulators are double-buffered in TMEM, so the next item's first two K-blocks run while an
// item is being stored.  Every wait is bounded; on expiry the CTA records a code and drains.
namespace netra {

constexpr int kPairThreads = 640;
// setmaxnreg: the four promotion warpgroups may ask for what the first one gives back, 128 * (96 - 32) = 4 * 128 * (112 - 96)
constexpr int kPairRegsLaunch = 96, kPairRegsLow = 32, kPairRegsHigh = 112;
static_assert(128 * kPairRegsLow + 512 * kPairRegsHigh <= kPairThreads * kPairRegsLaunch, "the promotion warps would wait forever for registers");

struct PairCfg {
  static constexpr int kStages = 4;
  static constexpr int kStageBytes = 2 * 128 * kBlock;            // 128 rows, 128 weight rows (or columns)
  static constexpr int kStagingBytes = 16 * 4096;                 // per promotion warp: 32 rows of 128 bytes, swizzled
  static constexpr int kScaleSlots = 8;                           // K-blocks whose scales are in shared memory or on their way
  static constexpr int kScaleSlotFloats = 128 + 4;                // 128 rows, two weight tiles
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kStagingBytes + kScaleSlots * kScaleSlotFloats * 4 + 256;
  static_assert(kSmemBytes <= 232448, "exceeds the shared memory of one SM");
  // the barriers of the two accumulator stages are 16 bytes apart and told apart by that address bit
  static constexpr int kTemptyOffset = kStages * kStageBytes + kStagingBytes + kScaleSlots * kScaleSlotFloats * 4 + 3 * kStages * 8;
  static_assert(kTemptyOffset % 32 == 0, "the release barriers' address bit");
};

struct PairArgs {
  const float* a_scale;
  uint64_t a_scale_row, a_scale_block;
  const float* w_scale;
  uint64_t w_scale_col, w_scale_block;
  void* out;
  uint64_t out_pitch;
  uint32_t tma_store;                     // rows of the output start on 16-byte boundaries
  uint32_t m, n, k_blocks;
  uint32_t m_tiles, n_tiles;              // of 256
};

// Arrival on a barrier of either CTA of the pair.  It hands over TMEM columns, whose reads tcgen05.wait::ld has completed and
// tcgen05.fence orders; no other memory is handed over.
__device__ __forceinline__ void mbar_arrive_peer(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float ld_shared_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, const uint32_t v[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ void cp_async_f32(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// a load into this CTA's shared memory that reports its bytes to a barrier of the pair's leader
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;"
      ::"r"(dst), "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y), "l"(policy) : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// one arrival on this barrier of both CTAs once the MMAs issued so far are done
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"((uint64_t)map), "r"(src), "r"(x), "r"(y) : "memory");
}
// (a.x, a.y) * (s, s) + (c.x, c.y), each component rounded once
__device__ __forceinline__ float2 fma2(float2 a, float2 s, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r)
      : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&s)), "l"(*reinterpret_cast<const uint64_t*>(&c)));
  return *reinterpret_cast<const float2*>(&r);
}

// Item i -> tile: columns of eight row tiles, so that the items in flight share few weight and activation tiles in the L2.
__device__ __forceinline__ void pair_item(uint32_t i, uint32_t m_tiles, uint32_t n_tiles, uint32_t& mt, uint32_t& nt) {
  const uint32_t band = i / (8 * n_tiles), first = band * 8, rows = min(8u, m_tiles - first), j = i - band * 8 * n_tiles;
  mt = first + j % rows;
  nt = j / rows;
}

template <bool kTransposed, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
netra_dense_fp8_pair_sm100(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                           const __grid_constant__ CUtensorMap tm_out, const PairArgs g) {
  using C = PairCfg;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* staging = smem + C::kStages * C::kStageBytes;
  float* scales = reinterpret_cast<float*>(staging + C::kStagingBytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(scales + C::kScaleSlots * C::kScaleSlotFloats);
  uint64_t* done_bar = full_bar + C::kStages;         // [stage][half]: the MMAs of a stage's half are done and its scales are there
  uint64_t* tempty_bar = done_bar + 2 * C::kStages;   // [accumulator stage][half]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 4);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const uint32_t items = g.m_tiles * g.n_tiles, pairs = gridDim.x >> 1, pair = blockIdx.x >> 1;

  if (threadIdx.x < 96 && lane == 0) prefetch_tensormap(warp == 0 ? &tm_a : warp == 1 ? &tm_w : &tm_out);
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) { mbar_init(smem_u32(&full_bar[s]), 1); mbar_init(smem_u32(&done_bar[2 * s]), 2); mbar_init(smem_u32(&done_bar[2 * s + 1]), 2); }
    for (int a = 0; a < 4; ++a) mbar_init(smem_u32(&tempty_bar[a]), rank == 0 ? 9 : 8);     // promotion warps, and the peer's relay
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();                                  // the peer's barriers exist before anything reports to them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  begin_grid();                                       // nothing above touches global memory

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairRegsLow));
    if (warp == 0 && lane == 0) {
      const uint64_t pol = policy_evict_last();
      uint32_t it = 0;
      bool ok = true;
      for (uint32_t item = pair; ok && item < items; item += pairs) {
        uint32_t mt, nt;
        pair_item(item, g.m_tiles, g.n_tiles, mt, nt);
        const int row = (int)(mt * 256 + rank * 128), col = (int)(nt * 256 + rank * 128);
        for (uint32_t kb = 0; kb < g.k_blocks; ++kb, ++it) {
          const uint32_t s = it % C::kStages;
          if (!mbar_wait(smem_u32(&done_bar[2 * s + 1]), ((it / C::kStages) & 1) ^ 1, abort_flag)) {
            g_dense_status[0] = kStatusProducerTimeout; *abort_flag = 1; ok = false; break;
          }
          if (rank == 0) mbar_expect_tx(smem_u32(&full_bar[s]), 2 * C::kStageBytes);
          const uint32_t bar = map_to_rank(smem_u32(&full_bar[s]), 0), dst = smem_u32(smem + s * C::kStageBytes);
          tma_load_2d_pair(dst, &tm_a, bar, (int)(kb * kBlock), row, pol);
          if (kTransposed) tma_load_2d_pair(dst + 128 * kBlock, &tm_w, bar, col, (int)(kb * kBlock), pol);
          else tma_load_2d_pair(dst + 128 * kBlock, &tm_w, bar, (int)(kb * kBlock), col, pol);
        }
      }
    } else if ((warp == 1 || warp == 3) && lane == 0 && rank == 0) {
      // Two threads take alternate K-blocks, each its own accumulator stage: while one feeds its four MMAs to the tensor pipe,
      // the other is already through its waits.  The operands, which are early, are waited for first.
      const uint32_t idesc = (1u << 4) | (kTransposed ? 1u << 16 : 0u) | ((128u >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
      const uint32_t a = (uint32_t)warp >> 1, mine = pair < items ? (items - 1 - pair) / pairs + 1 : 0;
      const uint64_t total = (uint64_t)mine * g.k_blocks;
      uint32_t phase = 1;
      bool ok = true;
      for (uint64_t it = a; ok && it < total; it += 2, phase ^= 1) {
        const uint32_t s = (uint32_t)it % C::kStages;
        ok = mbar_wait(smem_u32(&full_bar[s]), (uint32_t)(it / C::kStages) & 1, abort_flag);
        const uint32_t sa = smem_u32(smem + s * C::kStageBytes);
        const uint64_t adesc = make_smem_desc(sa);
        const uint64_t bdesc = kTransposed ? make_smem_desc_mn(sa + 128 * kBlock) : make_smem_desc(sa + 128 * kBlock);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ok = ok && mbar_wait(smem_u32(&tempty_bar[2 * a + h]), phase, abort_flag);
          if (!ok) break;
          tc_fence_after();
          // half h: 64 weight rows (or columns) of either CTA
          const uint64_t bhalf = bdesc + (kTransposed ? 64 >> 4 : 64 * kBlock >> 4) * h;
#pragma unroll
          for (int k = 0; k < kBlock / 32; ++k)
            umma_f8_pair(tmem_base + a * 256 + h * 128, adesc + 2 * k, bhalf + (kTransposed ? 256 : 2) * k, idesc, k > 0);
          umma_commit_pair(smem_u32(&done_bar[2 * s + h]));
        }
      }
      if (!ok) { g_dense_status[0] = kStatusMmaTimeout; *abort_flag = 1; }
    } else if ((warp == 1 || warp == 3) && lane == 0) {
      // The peer's eight releases of a half reach the leader as one arrival.
      const uint32_t h = (uint32_t)warp >> 1, mine = pair < items ? (items - 1 - pair) / pairs + 1 : 0;
      const uint64_t total = (uint64_t)mine * g.k_blocks;
      for (uint64_t it = 0; it < total; ++it) {
        const uint32_t bar = smem_u32(&tempty_bar[2 * ((uint32_t)it & 1) + h]);
        if (!mbar_wait(bar, (uint32_t)(it >> 1) & 1, abort_flag)) { g_dense_status[0] = kStatusMmaTimeout; *abort_flag = 1; break; }
        mbar_arrive_peer(map_to_rank(bar, 0));
      }
    } else if (warp == 2) {
      // An accumulator stage counts as full when its MMAs are done and its K-block's scales are in their slot.  Once K-block
      // it - 2 is full, every promotion warp has released it - 4, whose slot takes the scales of it + 4.
      const uint32_t mine = pair < items ? (items - 1 - pair) / pairs + 1 : 0;
      const uint64_t total = (uint64_t)mine * g.k_blocks;
      uint32_t item = pair, kb = 0, row = 0, tile = 0;
      uint64_t next = 0;                                // K-block whose scales are asked for next
      auto load = [&]() {
        if (next < total) {
          if (kb == 0) {
            uint32_t mt, nt;
            pair_item(item, g.m_tiles, g.n_tiles, mt, nt);
            row = mt * 256 + rank * 128 + lane;
            tile = nt * 2 + (lane & 1);
          }
          const uint32_t slot = smem_u32(scales + (next % C::kScaleSlots) * C::kScaleSlotFloats);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            cp_async_f32(slot + (lane + 32 * j) * 4, g.a_scale + (uint64_t)min(row + 32 * j, g.m - 1) * g.a_scale_row + kb * g.a_scale_block);
          if (lane < 2) cp_async_f32(slot + (128 + lane) * 4, g.w_scale + (uint64_t)min(tile, (g.n - 1) / kBlock) * g.w_scale_col + kb * g.w_scale_block);
          if (++kb == g.k_blocks) { kb = 0; item += pairs; }
        }
        ++next;
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      for (int j = 0; j < 4; ++j) load();
      for (uint64_t it = 0; it < total; ++it) {
        if (it >= 2 && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&done_bar[2 * ((it - 2) % C::kStages) + 1]), (uint32_t)((it - 2) / C::kStages) & 1, abort_flag))) {
          g_dense_status[0] = kStatusProducerTimeout; *abort_flag = 1; break;
        }
        load();
        asm volatile("cp.async.wait_group 4;" ::: "memory");
        __syncwarp();
        if (lane < 2) mbar_arrive(smem_u32(&done_bar[2 * (it % C::kStages) + lane]));
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairRegsHigh));
    const int wg = (warp - 4) >> 2, quad = warp & 3;            // 64 columns and 32 rows of this warp
    const uint32_t tile = smem_u32(staging) + (uint32_t)(warp - 4) * 4096u, my_row = tile + (uint32_t)lane * 128u;
    // Every instruction here lengthens the chain above (a leaner loop: 673 -> 618 ns a K-block), so what can be carried from one
    // K-block to the next is carried: the barrier's address and phase, the scales' slot (four stages and two phases make the
    // eight slots), the TMEM column of the accumulator stage.
    const uint32_t bar0 = smem_u32(&done_bar[wg >> 1]);
    const uint32_t slot0 = smem_u32(scales) + (uint32_t)(quad * 32 + lane) * 4u, tile_scale = (uint32_t)(128 + (wg & 1) - (quad * 32 + lane)) * 4u;
    uint32_t stage = 0, phase = 0, column = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(wg * 64);
    static_assert(C::kScaleSlots == 2 * C::kStages, "a slot is a stage and the parity of its phase");
    const bool first_lane = lane == 0;
    uint32_t release = smem_u32(&tempty_bar[wg >> 1]);
    bool ok = true;
    for (uint32_t item = pair; ok && item < items; item += pairs) {
      uint32_t mt, nt;
      pair_item(item, g.m_tiles, g.n_tiles, mt, nt);
      const uint32_t row0 = mt * 256 + rank * 128 + quad * 32, col0 = nt * 256 + (wg & 1) * 128 + (wg >> 1) * 64;
      float2 acc[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) acc[c] = make_float2(0.0f, 0.0f);
#pragma unroll 1
      for (uint32_t kb = 0; kb < g.k_blocks; ++kb) {
        const uint32_t bar = bar0 + 16 * stage;
        if (!mbar_wait_warp(bar, phase, abort_flag)) { ok = false; break; }
        tc_fence_after();
        uint32_t v[32];
        tmem_ld32_nowait(column, v);
        const uint32_t slot = slot0 + (stage + phase * C::kStages) * (C::kScaleSlotFloats * 4);
        const float s = __fmul_rn(ld_shared_f32(slot), ld_shared_f32(slot + tile_scale));
        const float2 s2 = make_float2(s, s);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 16; ++c) acc[c] = fma2(make_float2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])), s2, acc[c]);
        tmem_ld32_nowait(column + 32, v);
        if (++stage == C::kStages) { stage = 0; phase ^= 1; }
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (first_lane) mbar_arrive(release);
        release ^= 16;
        column ^= 256;
#pragma unroll
        for (int c = 0; c < 16; ++c) acc[16 + c] = fma2(make_float2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])), s2, acc[16 + c]);
      }
      if (!ok) { g_dense_status[0] = kStatusEpilogueTimeout; *abort_flag = 1; break; }
      // ---- store: 128 bytes per row at a time through this warp's own staging rows (chunk j of row r at j ^ (r & 7), the
      // 128-byte swizzle of the copy engine), 64 columns of a 16-bit type or 32 of FP32
      constexpr int kPasses = sizeof(T) / 2, kPassCols = 64 / kPasses;
#pragma unroll
      for (int pass = 0; pass < kPasses; ++pass) {
        if (first_lane) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");     // the last copy has left the rows
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t p[4];
          if constexpr (kPasses == 2) {
#pragma unroll
            for (int q = 0; q < 2; ++q) { const float2 f = acc[pass * 16 + 2 * j + q]; p[2 * q] = __float_as_uint(f.x); p[2 * q + 1] = __float_as_uint(f.y); }
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float2 f = acc[4 * j + q];
              if constexpr (std::is_same<T, __half>::value) { const __half2 h = __floats2half2_rn(f.x, f.y); p[q] = *reinterpret_cast<const uint32_t*>(&h); }
              else { const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y); p[q] = *reinterpret_cast<const uint32_t*>(&h); }
            }
          }
          st_shared_v4(my_row + 16 * (j ^ (lane & 7)), p);
        }
        const uint32_t col = col0 + pass * kPassCols;
        if (g.tma_store) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (first_lane) {
            if (row0 < g.m && col < g.n) tma_store_2d(&tm_out, tile, (int)col, (int)row0);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          // rows that do not start on 16-byte boundaries: a lane a column
          __syncwarp();
          T* out = reinterpret_cast<T*>(g.out);
          const uint8_t* rows = staging + (warp - 4) * 4096;
#pragma unroll 1
          for (uint32_t r = 0; r < 32 && row0 + r < g.m; ++r)
#pragma unroll 1
            for (uint32_t c = lane; c < (uint32_t)kPassCols && col + c < g.n; c += 32) {
              const uint32_t byte = c * (uint32_t)sizeof(T);
              out[(uint64_t)(row0 + r) * g.out_pitch + col + c] = *reinterpret_cast<const T*>(rows + r * 128 + 16 * ((byte >> 4) ^ (r & 7)) + (byte & 15));
            }
          __syncwarp();
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) __nanosleep(200000);          // copies in flight land before the CTA exits
  cluster_barrier();                                  // nothing reports to this CTA any more
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

}  // namespace netra
