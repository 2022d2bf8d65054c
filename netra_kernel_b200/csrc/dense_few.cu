// The dense block-scaled product for few rows: y[m,n] for m <= 16 (or <= 32 rows of codes).
//
// The weight is read once and nothing else costs, so the call is bounded by how many weight bytes are in flight and, at the
// sizes of one projection (8 MB: 1.3 us of HBM time), by the latency of its steps.  A warp owns 16 weight rows and a share of
// the K-blocks and multiplies them straight from registers (mma.sync m16n8k32, weights as A, tokens as B): no shared-memory
// ring, no TMEM, no barrier before the sums of the warps are joined, and every weight byte of two K-blocks is asked for
// before the first is used.  The tensor rate of mma.sync is far from what bounds this.
//   * A lane takes 32 neighbouring bytes of a row per K-block instead of the fragment's scattered four-byte words: the order of
//     the K index inside a block does not matter as long as both operands use the same one.
//   * Source rows of BF16 / FP16 / FP32 are quantised by the warp that multiplies them (each warp sees its own K-blocks of all
//     rows: no block of a row is quantised twice by one CTA), which saves the quantiser's launch.
// Per K-block the raw FP32 sums are promoted as acc = fma(part, sa * sw, acc); the warps' sums are added in warp order.
// Measured (BF16 rows, quantising included, in a graph): 1 x 2048 x 4096 3.7-3.8 us, 8 x 4096 x 2048 4.1-4.2 us, 12 x 4096 x 2048 5.7 us.
namespace netra {

constexpr int kFewRows = 16;            // weight rows of a CTA

__device__ __forceinline__ void mma_e4m3_16x8x32(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 codes at p, of which `left` belong to the row; p is 16-byte aligned and nothing behind the row is touched
__device__ __forceinline__ uint4 load_codes16(const uint8_t* p, int left) {
  if (left >= 16) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; i < left; ++i) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

struct FewArgs {
  const void* x;                        // rows of T
  uint64_t x_pitch;
  const float* a_scale;                 // codes only
  uint64_t a_scale_row, a_scale_block;
  const uint8_t* w;
  uint64_t w_pitch;
  const float* w_scale;
  uint64_t w_scale_pitch;
  void* out;
  uint64_t out_pitch;
  uint32_t out_dtype, m, n, k;
};

// eight code words of the lane's 32 columns of one row, and the row's scale (the same in the quad's four lanes)
template <typename T>
__device__ __forceinline__ float few_row(uint32_t word[8], const FewArgs& g, uint32_t row, uint32_t kb, int t) {
  const uint32_t col = kb * kBlock + t * 32;
  if constexpr (sizeof(T) == 1) {
    if (row >= g.m) {
#pragma unroll
      for (int j = 0; j < 8; ++j) word[j] = 0;
      return 0.0f;
    }
    const uint8_t* p = reinterpret_cast<const uint8_t*>(g.x) + row * g.x_pitch + col;
    const uint4 lo = load_codes16(p, (int)g.k - (int)col), hi = load_codes16(p + 16, (int)g.k - (int)col - 16);
    word[0] = lo.x; word[1] = lo.y; word[2] = lo.z; word[3] = lo.w; word[4] = hi.x; word[5] = hi.y; word[6] = hi.z; word[7] = hi.w;
    return g.a_scale[row * g.a_scale_row + kb * g.a_scale_block];
  } else {
    Eight<T> x8[4];
    float amax = amax_floor();
    const T* p = reinterpret_cast<const T*>(g.x) + row * g.x_pitch + col;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (row < g.m && col + 8 * c < g.k) x8[c].load(p + 8 * c);         // the host passes widths that are multiples of eight
      else x8[c].clear();
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) amax = fmaxf(amax, x8[c].amax());
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const float s = amax * inv448(), inv = 1.0f / s;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float v[8];
      x8[c].values(v);
      word[2 * c] = f32x4_to_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
      word[2 * c + 1] = f32x4_to_e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    }
    return s;
  }
}

// kTiles: tiles of eight rows of x.  blockDim = 32 * warps; grid = ceil(n / 16).
template <typename T, int kTiles>
__global__ void __launch_bounds__(512)
netra_dense_fp8_few_sm100(const FewArgs g) {
  extern __shared__ float few_sums[];               // [warps][kTiles * 8 rows of x][16 weight rows]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int grp = lane >> 2, t = lane & 3;
  const uint32_t n0 = blockIdx.x * kFewRows, blocks = (g.k + kBlock - 1) / kBlock;
  begin_grid();
  const uint8_t* w_lo = g.w + (uint64_t)min(n0 + grp, g.n - 1) * g.w_pitch;        // rows past the end: computed, not stored
  const uint8_t* w_hi = g.w + (uint64_t)min(n0 + grp + 8, g.n - 1) * g.w_pitch;
  const float* ws = g.w_scale + (uint64_t)(n0 / kBlock) * g.w_scale_pitch;
  float acc[kTiles][4];
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[i][c] = 0.0f;
  uint4 a[2][4];                                    // two K-blocks: row grp (32 bytes), row grp + 8 (32 bytes)
  auto fetch = [&](uint4 to[4], uint32_t kb) {
    const uint32_t col = kb * kBlock + t * 32;
    const int left = (int)g.k - (int)col;
    to[0] = load_codes16(w_lo + col, left);
    to[1] = load_codes16(w_lo + col + 16, left - 16);
    to[2] = load_codes16(w_hi + col, left);
    to[3] = load_codes16(w_hi + col + 16, left - 16);
  };
  if ((uint32_t)warp < blocks) fetch(a[0], warp);
  if ((uint32_t)(warp + warps) < blocks) fetch(a[1], warp + warps);
  for (uint32_t kb0 = warp; kb0 < blocks; kb0 += 2 * warps) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t kb = kb0 + h * warps;
      if (kb >= blocks) break;
      const uint32_t lo[8] = {a[h][0].x, a[h][0].y, a[h][0].z, a[h][0].w, a[h][1].x, a[h][1].y, a[h][1].z, a[h][1].w};
      const uint32_t hi[8] = {a[h][2].x, a[h][2].y, a[h][2].z, a[h][2].w, a[h][3].x, a[h][3].y, a[h][3].z, a[h][3].w};
      const float sw = ws[kb];
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        uint32_t b[8];
        const float s = few_row<T>(b, g, i * 8 + grp, kb, t) * sw;
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_e4m3_16x8x32(part, lo[2 * j], hi[2 * j], lo[2 * j + 1], hi[2 * j + 1], b[2 * j], b[2 * j + 1]);
        // the sums of a lane belong to rows 2t and 2t + 1 of the tile, whose scales the quads 2t and 2t + 1 hold
        const float s0 = __shfl_sync(0xffffffffu, s, 8 * t), s1 = __shfl_sync(0xffffffffu, s, 8 * t + 4);
        acc[i][0] = fmaf(part[0], s0, acc[i][0]);
        acc[i][1] = fmaf(part[1], s1, acc[i][1]);
        acc[i][2] = fmaf(part[2], s0, acc[i][2]);
        acc[i][3] = fmaf(part[3], s1, acc[i][3]);
      }
      if (kb + 2 * warps < blocks) fetch(a[h], kb + 2 * warps);
    }
  }
  float* mine = few_sums + warp * (kTiles * 8 * kFewRows);
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    mine[(i * 8 + 2 * t) * kFewRows + grp] = acc[i][0];
    mine[(i * 8 + 2 * t + 1) * kFewRows + grp] = acc[i][1];
    mine[(i * 8 + 2 * t) * kFewRows + grp + 8] = acc[i][2];
    mine[(i * 8 + 2 * t + 1) * kFewRows + grp + 8] = acc[i][3];
  }
  __syncthreads();
  for (int o = threadIdx.x; o < kTiles * 8 * kFewRows; o += blockDim.x) {
    const uint32_t row = o / kFewRows, col = n0 + o % kFewRows;
    if (row >= g.m || col >= g.n) continue;
    float sum = 0.0f;
    for (int i = 0; i < warps; ++i) sum += few_sums[i * (kTiles * 8 * kFewRows) + o];
    dense_store(g.out, g.out_dtype, (uint64_t)row * g.out_pitch + col, sum);
  }
}

}  // namespace netra
