// The MXFP4 product's tile kernel, its split over K, and the C entry points.
//
// BT x BT output tiles, four waves of 32 x 32 or eight of 64 x 32, two a SIMD at
// least (a block of 64 x 64 shares its CU with another), so that one issues where the
// other waits: (1024, 4096, 4096) bf16 with four waves of 64 x 64 23.8 us, with eight
// 20.1.  K tiles of 256 values (128 bytes a row, whole lines) go through a ring of
// four stages filled by direct DMA three tiles ahead, or of two; one barrier per K
// tile.  What
// bounds it is the delivery of the tiles into the LDS, some 35 bytes a ns and CU.
//
// Scales come as dwords, those of two K tiles together: a row's 8 bytes a K tile are
// a request as a line of codes is ((512, 4096, 14336) a K tile's at a time 55.6 us,
// two 46.4, four, which read the LDS in conflict, 47.4).  Where a row's scales do not
// start on a dword, or K tiles end inside one (FIT false), a lane loads the three
// dwords that its row's 8 bytes of a K tile lie in and reads single bytes; bytes
// behind the row's last block, which may belong to another row and be 255 (NaN),
// become 0 there.  Such a dword may reach up to 3 bytes past the scales' end or
// before their start; being aligned it lies within what the memory's page holds.
#include <algorithm>
#include <atomic>

#include "gemm_mxfp4.h"

namespace ntops {
namespace {

// Blocks that share a CU.
constexpr int tile_blocks(int bt, int stages) { return (bt == 64 ? 2 : 1) * 4 / stages; }

template <int BT, bool FIT, int STAGES>
struct TileShape {
  static constexpr int kWaves = BT == 128 ? 8 : 4;
  static constexpr int kWN = kWaves / 2;  // waves along a tile's columns
  static constexpr int kRowsPerWave = BT / kWaves;                  // rows of an operand that a wave loads
  static constexpr int kCodes = BT * 128;                      // bytes of an operand's codes per stage
  static constexpr int kStage = 2 * kCodes;
  static constexpr int kGroup = FIT ? 2 : 1;                   // K tiles whose scales are loaded together
  static constexpr int kDwords = FIT ? 4 : 3;                  // of a row's scales in a group
  static constexpr int kScaleInst = (kRowsPerWave * kDwords + 63) / 64;
  static constexpr int kScales = kWaves * kScaleInst * 256;    // bytes of an operand's scales in a group
  static constexpr int kScaleRing = STAGES == 2 ? 4 : 8;       // groups
  static constexpr int kScalesPerTile = 2 * kScaleInst / kGroup;
  static constexpr int kScalesAt = STAGES * kStage;
  static constexpr int kLds = kScalesAt + kScaleRing * 2 * kScales;
  static constexpr int kLoads = 2 * kRowsPerWave / 8 + kScalesPerTile;  // DMA instructions per wave and K tile
  static_assert(kRowsPerWave == 16 && kScalesPerTile * kGroup == 2 * kScaleInst && kLds * tile_blocks(BT, STAGES) <= 163840 && BT * BT * 4 <= kLds, "tile");
};

// A finished tile leaves through the LDS, so that stores are runs of whole rows from
// any address on, not four values of 16 rows each: (8192, 14336, 256) bf16 105.2 ->
// 67.7 us, over 14335 columns 212.7 -> 67.3, (1024, 4096, 4096) 20.2 -> 19.2 (stored
// past the caches (8192, 14336, 256) takes 61.0, but over 14335 columns 112).
// The byte of element (r, c); 16-byte chunks are rotated so that 16 rows' chunks touch
// every bank.
template <typename O, int BT>
__device__ __forceinline__ int out_at(int r, int c) {
  constexpr int kRow = BT * static_cast<int>(sizeof(O));
  const int byte = c * static_cast<int>(sizeof(O));
  return r * kRow + ((byte & ~15) ^ (kRow == 128 ? (r >> 1) & 7 : r & 15) << 4) + (byte & 15);
}

typedef u32x4 u32x4_any __attribute__((aligned(2), may_alias));  // 16 bytes at any address

template <typename O, int BT, int WAVES>
__device__ __forceinline__ void store_staged(const char* smem, O* d, int64_t ldd, int rows, int cols) {
  constexpr int kPer = 16 / sizeof(O), kChunks = BT / kPer;
#pragma unroll
  for (int u = 0; u < BT * kChunks / (64 * WAVES); ++u) {
    const int id = u * (64 * WAVES) + threadIdx.x, r = id / kChunks, c = id % kChunks * kPer;
    const u32x4 v = *reinterpret_cast<const u32x4*>(smem + out_at<O, BT>(r, c));
    O* at = d + r * ldd + c;
    if (r < rows && c + kPer <= cols) {
      *reinterpret_cast<u32x4_any*>(at) = v;
    } else if (r < rows) {
      O o[kPer];
      __builtin_memcpy(o, &v, 16);
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (c + e < cols) at[e] = o[e];
    }
  }
}

template <typename T, int BT, bool FIT, int STAGES>
__global__ __launch_bounds__(64 * (BT == 128 ? 8 : 4), tile_blocks(BT, STAGES)) void k_mx4_tile(Mx4Args g, int tm_count, int tn_count) {
  using S = TileShape<BT, FIT, STAGES>;
  constexpr int TW = BT / 32, TN = BT / S::kWN / 16;  // 16-row and 16-column pieces of a wave's tile
  constexpr int ND = S::kDwords;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / S::kWN, wn = wave % S::kWN;
  const int q = lane >> 4, i16 = lane & 15;
  // Tiles by columns of up to 8 row tiles, so that neighbours share operands, and an
  // XCD (workgroups go round the eight) takes a run of them: (512, 4096, 4096) 17.6 ->
  // 16.2 us.
  const int xcd = blockIdx.x & 7;
  const int t = xcd * static_cast<int>(gridDim.x >> 3) + min(xcd, static_cast<int>(gridDim.x & 7)) + static_cast<int>(blockIdx.x >> 3);
  const int band = t / (8 * tn_count);
  const int rows_here = min(8, tm_count - band * 8);
  const int in = t - band * 8 * tn_count;
  const int m0 = (band * 8 + in % rows_here) * BT, n0 = in / rows_here * BT;
  const int slice = blockIdx.y;
  const int kb0 = slice * g.kchunk, kb1 = min(g.kb, kb0 + g.kchunk);
  const int nt = (kb1 - kb0 + 7) / 8;

  const int mv = min(BT, g.M - m0), nv = min(BT, g.N - n0);
  const u32x4 ra = make_rsrc(g.a + m0 * g.lda, (mv - 1) * g.lda + g.kb * 16);
  const u32x4 rb = make_rsrc(g.b + n0 * g.ldb, (nv - 1) * g.ldb + g.kb * 16);
  // scales from the dword on that holds the tile's first byte
  const uint8_t* sa0 = g.as + m0 * g.ldas;
  const uint8_t* sb0 = g.bs + n0 * g.ldbs;
  const int oa = FIT ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(sa0) & 3u);
  const int ob = FIT ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(sb0) & 3u);
  const u32x4 rsa = make_rsrc(sa0 - oa, (oa + (mv - 1) * g.ldas + g.kb + 3) & ~3ll);
  const u32x4 rsb = make_rsrc(sb0 - ob, (ob + (nv - 1) * g.ldbs + g.kb + 3) & ~3ll);
  const uint32_t smem_addr = lds_addr(smem);

  // this wave's load id of scale group gr: 16 rows of A's or B's (row l / ND, dword l % ND)
  auto issue_scales = [&](int gr, int id) {
    const int u = id % S::kScaleInst;
    const bool of_b = id >= S::kScaleInst;
    const int l = u * 64 + lane;
    const int in_wave = l / ND, row = wave * S::kRowsPerWave + in_wave;
    const int b0 = kb0 + gr * (S::kGroup * 8), blk = b0 + (l - in_wave * ND) * 4;
    const bool ok = in_wave < S::kRowsPerWave && b0 < kb1 && row < (of_b ? nv : mv);
    // (past the row's last dword: the next row's, masked or not read below; past the last row's: zeros)
    const uint32_t off = static_cast<uint32_t>((of_b ? ob + row * g.ldbs : oa + row * g.ldas) + blk) & ~3u;
    const uint32_t dst = smem_addr + S::kScalesAt +
                         static_cast<uint32_t>((gr & (S::kScaleRing - 1)) * (2 * S::kScales) + (of_b ? S::kScales : 0) +
                                               (wave * S::kScaleInst + u) * 256);
    dma4(of_b ? rsb : rsa, dst, ok ? off : kOOB);
  };
  // this wave's loads of K tile j: 16 rows of A and of B, 8 an instruction, and its
  // part of the scales of the next group
  auto issue = [&](int j) {
    const uint32_t st = smem_addr + static_cast<uint32_t>((j & (STAGES - 1)) * S::kStage);
    const int b0 = kb0 + j * 8;
#pragma unroll
    for (int u = 0; u < S::kRowsPerWave / 8; ++u) {
      const int row = wave * S::kRowsPerWave + u * 8 + (lane >> 3);
      const int blk = b0 + kslot<64>(row, lane & 7);
      const uint32_t dst = st + static_cast<uint32_t>((wave * S::kRowsPerWave + u * 8) * 128);
      dma16(ra, dst, blk < kb1 && row < mv ? static_cast<uint32_t>(row * g.lda + blk * 16) : kOOB);
      dma16(rb, dst + S::kCodes, blk < kb1 && row < nv ? static_cast<uint32_t>(row * g.ldb + blk * 16) : kOOB);
    }
#pragma unroll
    for (int u = 0; u < S::kScalesPerTile; ++u) issue_scales(j / S::kGroup + 1, j % S::kGroup * S::kScalesPerTile + u);
  };
  // LDS offset of row r's scales of a K tile (not FIT: of the byte of block q)
  auto scale_at = [&](int r, int o, int64_t ld) {
    const int w = r / S::kRowsPerWave, in_wave = r - w * S::kRowsPerWave;
    return w * S::kScaleInst * 256 + in_wave * ND * 4 + (FIT ? 0 : static_cast<int>((o + r * ld) & 3) + q);
  };
  int sat[TW], sbt[TN];
#pragma unroll
  for (int i = 0; i < TW; ++i) sat[i] = scale_at(wm * (BT / 2) + i * 16 + i16, oa, g.ldas);
#pragma unroll
  for (int i = 0; i < TN; ++i) sbt[i] = S::kScales + scale_at((wn * TN + i) * 16 + i16, ob, g.ldbs);

  f32x4 acc[TW][TN];
#pragma unroll
  for (int i = 0; i < TW; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 2 * S::kScaleInst; ++u) issue_scales(0, u);
#pragma unroll
  for (int j = 0; j < STAGES - 1; ++j)
    if (j < nt) issue(j);
  for (int j = 0; j < nt; ++j) {
    __builtin_amdgcn_sched_barrier(0);
    // K tile j is in: all but the tiles behind it, STAGES - 2 until the last ones
    if (STAGES == 4 && nt - 1 - j >= 2)
      wait_vmcnt<2 * S::kLoads>();
    else if (STAGES == 4 && nt - 1 - j == 1)
      wait_vmcnt<S::kLoads>();
    else
      wait_vmcnt<0>();
    block_barrier();              // for every wave; and tile j - 1's stage is free
    asm volatile("" ::: "memory");
    if (j + STAGES - 1 < nt) issue(j + STAGES - 1);
    const char* st = smem + (j & (STAGES - 1)) * S::kStage;
    const char* sc = smem + S::kScalesAt + (j / S::kGroup & (S::kScaleRing - 1)) * (2 * S::kScales) + j % S::kGroup * 8;
    uint32_t sa[TW], sb[TN];
    // the scales of blocks q and q + 4 of each row, in bytes 0 and 1
    if constexpr (FIT) {
      const uint32_t sel = 0x0400u + q * 0x0101u;
      const auto two = [&](int at) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(sc + at);
        return __builtin_amdgcn_perm(w.y, w.x, sel);
      };
#pragma unroll
      for (int i = 0; i < TW; ++i) sa[i] = two(sat[i]);
#pragma unroll
      for (int i = 0; i < TN; ++i) sb[i] = two(sbt[i]);
    } else {
      const int left = kb1 - kb0 - j * 8 - q;  // blocks from this lane's first on
      const uint32_t mask = left > 4 ? 0xffffu : left > 0 ? 0xffu : 0u;
      const auto two = [&](int at) {
        const uint8_t* p = reinterpret_cast<const uint8_t*>(sc + at);
        return (p[0] | static_cast<uint32_t>(p[4]) << 8) & mask;
      };
#pragma unroll
      for (int i = 0; i < TW; ++i) sa[i] = two(sat[i]);
#pragma unroll
      for (int i = 0; i < TN; ++i) sb[i] = two(sbt[i]);
    }
    const auto frag = [&](int area, int r, int ks) {
      return *reinterpret_cast<const u32x4*>(st + area * S::kCodes + r * 128 + kslot<64>(r, 4 * ks + q) * 16);
    };
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      u32x4 fa[TW], fb[TN];
#pragma unroll
      for (int i = 0; i < TW; ++i) fa[i] = frag(0, wm * (BT / 2) + i * 16 + i16, ks);
#pragma unroll
      for (int i = 0; i < TN; ++i) fb[i] = frag(1, (wn * TN + i) * 16 + i16, ks);
#pragma unroll
      for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int k = 0; k < TN; ++k)
          acc[i][k] = ks == 0 ? mfma_mx4<0, 0>(fb[k], sb[k], fa[i], sa[i], acc[i][k])
                              : mfma_mx4<1, 1>(fb[k], sb[k], fa[i], sa[i], acc[i][k]);
    }
    wait_lgkmcnt0();  // this stage's reads are over before the next barrier frees it
  }
  wait_vmcnt<0>();  // no DMA may land in the LDS that the output is staged in
  __syncthreads();
  const auto stage = [&](auto tag, const auto* bias) {
    using O = decltype(tag);
#pragma unroll
    for (int k = 0; k < TN; ++k) {
      const int c = (wn * TN + k) * 16 + 4 * q;
      float b[4] = {0.f, 0.f, 0.f, 0.f};
      if (bias != nullptr)
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = c + e < nv ? static_cast<float>(bias[n0 + c + e]) : 0.f;
#pragma unroll
      for (int i = 0; i < TW; ++i) {
        O o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = static_cast<O>(acc[i][k][e] + b[e]);
        __builtin_memcpy(smem + out_at<O, BT>(wm * (BT / 2) + i * 16 + i16, c), o, sizeof(o));
      }
    }
    __syncthreads();
  };
  if (g.split > 1) {
    stage(float{}, static_cast<const T*>(nullptr));
    store_staged<float, BT, S::kWaves>(smem, g.part + static_cast<int64_t>(slice) * g.M * g.N + static_cast<int64_t>(m0) * g.N + n0, g.N, mv, nv);
  } else {
    stage(T{}, static_cast<const T*>(g.bias));
    store_staged<T, BT, S::kWaves>(smem, static_cast<T*>(g.d) + static_cast<int64_t>(m0) * g.ldd + n0, g.ldd, mv, nv);
  }
}

// The slices' partial products summed in their order, and the bias: V elements a
// thread, of one row.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_mx4_reduce(Mx4Args g) {
  const int64_t mn = static_cast<int64_t>(g.M) * g.N;
  const int64_t i = (block_id() * 256 + threadIdx.x) * V;
  if (i >= mn) return;
  typedef float vec __attribute__((ext_vector_type(V)));
  typedef T out __attribute__((ext_vector_type(V)));
  vec v = 0.f;
  for (int s = 0; s < g.split; ++s) v += *reinterpret_cast<const vec*>(g.part + s * mn + i);
  const int64_t m = i / g.N, n = i - m * g.N;
  out o;
#pragma unroll
  for (int e = 0; e < V; ++e)
    o[e] = static_cast<T>(g.bias == nullptr ? v[e] : v[e] + static_cast<float>(static_cast<const T*>(g.bias)[n + e]));
  *reinterpret_cast<out*>(static_cast<T*>(g.d) + m * g.ldd + n) = o;
}

constexpr int64_t kMaxSize = int64_t(1) << 30;   // bytes of a tile's rows, or of a row
constexpr int64_t kMaxCount = int64_t(1) << 29;  // rows

// Whether K tiles of 8 blocks are whole dwords of these scale rows.
bool scales_fit(int64_t kb, const void* s, int64_t ld) {
  return kb % 8 == 0 && ld % 4 == 0 && (reinterpret_cast<uintptr_t>(s) & 3u) == 0;
}

// 256 x 256 tiles where 128 x 128 ones, two a CU, are more than a round of the GPU.
// Measured on 128 x 128 and on 256 x 256 (bf16, us): one round, (2048, 4096) over 4096
// 28.8 and 33.9, over 14336 81.5 and 81.5, (1024, 8192) over 14336 82.2 and 84.1, (256,
// 28672) over 14336 104 and 97; more, (1536, 6144) over 4096 38.1 and 34.1, over 14336
// 114 and 83, (4096, 4096) over 2048 30.8 and 29.2, over 4096 50.8 and 41.6, (8192,
// 14336) over 1056 155 and 130, over 2048 201 and 159.  It goes by tiles alone, and so
// wrong over short rows: (1536, 6144) over 1056 19.3 and 23.4, over 2048 23.6 and 25.2,
// (4096, 5120), a quarter of a second round of 256 x 256, over 2048 35.6 and 43.5.
// Up to 128 rows those are half empty: (128, 100000) over 4096 69.2 and 81.6.
bool large_suits(int64_t M, int64_t N) { return M > 128 && ceil_div(M, 128) * ceil_div(N, 128) > 2 * cu_count_cached(); }

// The tile's size and the slices of K: as many slices as bring the blocks near the
// number of CUs (twice as many: (256, 4096, 4096) 11.2 -> 16.1 us), none under eight
// K tiles of 64 x 64 or fourteen of 128 x 128, whose time a reduction's launch takes
// ((500, 1001, 2080) in slices of four 12.3 us, whole 9.1; (64, 4096, 14336) in slices
// of eight or more 17.6, of sixteen or more 19.1; (512, 4096, 4096) on 128 x 128 in
// slices of eight 25.1, whole 18.5).  128 x 128 where they, sliced so, fill three
// quarters of the CUs: with and without, (768, 4096, 4096) 19.3 and 22.5, (192, 14336,
// 4096) 20.8 and 25.5, (256, 4096, 14336) in four slices 26.6 and 29.0; short of that,
// (512, 4096, 4096) 18.5 and 14.7, (128, 4096, 14336) 23.8 and 20.2.
void plan(int64_t M, int64_t N, int64_t kb, int& bt, int& split, int& kchunk) {
  const int64_t cus = cu_count_cached();
  const auto tiles = [&](int64_t t) { return ceil_div(M, t) * ceil_div(N, t); };
  const int64_t kt = ceil_div(kb, 8);
  const auto slices = [&](int64_t t, int64_t least) { return std::max<int64_t>(1, std::min<int64_t>({cus / tiles(t), kt / least, 16})); };
  int64_t s = slices(128, 14);
  bt = M > 64 && 4 * tiles(128) * s >= 3 * cus ? 128 : 64;
  if (bt == 64) s = slices(64, 8);
  const int64_t per = ceil_div(kt, s);
  kchunk = static_cast<int>(per * 8);
  split = static_cast<int>(ceil_div(kt, per));
}

template <typename T>
void launch_reduce(const Mx4Args& g, bool fours, hipStream_t st) {
  const int64_t mn = static_cast<int64_t>(g.M) * g.N;
  if (fours)
    hipLaunchKernelGGL((k_mx4_reduce<T, 4>), blocks_2d(ceil_div(mn, 1024)), dim3(256), 0, st, g);
  else
    hipLaunchKernelGGL((k_mx4_reduce<T, 1>), blocks_2d(ceil_div(mn, 256)), dim3(256), 0, st, g);
}

// Rings of two stages, and twice the blocks a CU: where there are more tiles than
// one round of blocks with four ((8192, 8192, 512) 79.8 -> 62.6 us, (2048, 4096, 4096)
// 35.6 -> 29.2; of 64 x 64 (8192, 14336, 100) 174 -> 97.8), and for up to four K tiles
// ((1000, 1000, 200) 4.8 -> 4.4).  In one round four are needed ((1024, 4096, 14336)
// 53.5, with two 68.3; (64, 14336, 4096) 13.8 and 17.1).
bool two_stages(int64_t M, int64_t N, int64_t kchunk, int64_t split, int bt) {
  return kchunk <= 32 || ceil_div(M, bt) * ceil_div(N, bt) * split > cu_count_cached() * tile_blocks(bt, 4);
}

template <typename T, int BT, bool FIT, int STAGES>
int launch_tile(const Mx4Args& g, hipStream_t st) {
  auto kern = k_mx4_tile<T, BT, FIT, STAGES>;
  using S = TileShape<BT, FIT, STAGES>;
  constexpr int kLds = S::kLds;
  static std::atomic<uint64_t> reserved{0};
  if (const int rc = reserve_lds(reinterpret_cast<const void*>(kern), kLds, reserved, "mxfp4_mm"); rc != NTOPS_OK) return rc;
  const int tm = static_cast<int>(ceil_div(g.M, BT)), tn = static_cast<int>(ceil_div(g.N, BT));
  const int whole = (g.ldd & 3) == 0 && (reinterpret_cast<uintptr_t>(g.d) & (4 * sizeof(T) - 1)) == 0;
  note_kernel("mxfp4_tile%d split%d stages%d%s", BT, g.split, STAGES, FIT ? "" : " bytes");
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(tm * tn), static_cast<unsigned>(g.split)), dim3(64 * S::kWaves), kLds, st, g,
                     tm, tn);
  if (g.split > 1)
    launch_reduce<T>(g, whole && g.N % 4 == 0, st);
  return check_launch("mxfp4_mm");
}

template <typename T, int BT>
int run_tile(const Mx4Args& g, hipStream_t st) {
  const bool fit = scales_fit(g.kb, g.as, g.ldas) && scales_fit(g.kb, g.bs, g.ldbs);
  if (two_stages(g.M, g.N, g.kchunk, g.split, BT)) return fit ? launch_tile<T, BT, true, 2>(g, st) : launch_tile<T, BT, false, 2>(g, st);
  return fit ? launch_tile<T, BT, true, 4>(g, st) : launch_tile<T, BT, false, 4>(g, st);
}

}  // namespace
}  // namespace ntops

using namespace ntops;

extern "C" int64_t ntops_mxfp4_mm_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > kMaxCount || N > kMaxCount || K > kMaxSize) return 0;
  if (M <= kSkinnyRows) return 0;
  if (large_suits(M, N)) return mx4_large_workspace(M, N, ceil_div(K, 32));
  int bt, split, kchunk;
  plan(M, N, ceil_div(K, 32), bt, split, kchunk);
  return split > 1 ? split * M * N * 4 : 0;
}

namespace ntops {
namespace {

// The arguments of ntops_mxfp4_mm, checked (M, N > 0), in g.
int mx4_args(int out_dtype, int64_t M, int64_t N, int64_t K, const void* a, int64_t a_row_stride, const void* a_scales,
             int64_t as_row_stride, const void* b, int64_t b_row_stride, const void* b_scales, int64_t bs_row_stride,
             const void* bias, void* out, int64_t out_row_stride, const void* workspace, int64_t workspace_bytes, Mx4Args& g) {
  if (M < 0 || N < 0 || K < 0) return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: negative size");
  if (out_dtype != NTOPS_F32 && out_dtype != NTOPS_F16 && out_dtype != NTOPS_BF16)
    return set_error(NTOPS_ERR_UNSUPPORTED, "mxfp4_mm: unsupported output dtype %d (F32/F16/BF16 only)", out_dtype);
  if (!out || (K > 0 && (!a || !a_scales || !b || !b_scales))) return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: null pointer");
  const int64_t kb = ceil_div(K, 32);
  if (K == 0) a_row_stride = b_row_stride = as_row_stride = bs_row_stride = 0;  // no rows to read
  if (K > 0 && (!aligned16(a) || !aligned16(b) || a_row_stride % 16 != 0 || b_row_stride % 16 != 0))
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: code rows not aligned to 16 bytes");
  if (a_row_stride < 0 || b_row_stride < 0 || as_row_stride < 0 || bs_row_stride < 0)
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: negative row stride");
  const int64_t lim = kMaxSize;
  const auto span = [&](int64_t ld, int64_t row) { return 256 * ld + row; };  // bytes that one tile's rows cover
  if (M > kMaxCount || N > kMaxCount || kb * 16 > lim || span(a_row_stride, kb * 16) > lim || span(b_row_stride, kb * 16) > lim ||
      span(as_row_stride, kb) > lim || span(bs_row_stride, kb) > lim ||
      ceil_div(M, 64) * ceil_div(N, 64) > 0x7fffff)
    return set_error(NTOPS_ERR_UNSUPPORTED, "mxfp4_mm: operands too large");
  g.a = static_cast<const uint8_t*>(a);
  g.as = static_cast<const uint8_t*>(a_scales);
  g.b = static_cast<const uint8_t*>(b);
  g.bs = static_cast<const uint8_t*>(b_scales);
  g.bias = bias;
  g.d = out;
  g.lda = a_row_stride;
  g.ldas = as_row_stride;
  g.ldb = b_row_stride;
  g.ldbs = bs_row_stride;
  g.ldd = out_row_stride;
  g.M = static_cast<int>(M);
  g.N = static_cast<int>(N);
  g.kb = static_cast<int>(kb);
  if (workspace_bytes < 0 || (workspace != nullptr && !aligned16(workspace)))
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: workspace not aligned to 16 bytes");
  return NTOPS_OK;
}

}  // namespace
}  // namespace ntops

extern "C" int ntops_mxfp4_mm(int out_dtype, int64_t M, int64_t N, int64_t K, const void* a, int64_t a_row_stride,
                              const void* a_scales, int64_t as_row_stride, const void* b, int64_t b_row_stride,
                              const void* b_scales, int64_t bs_row_stride, const void* bias, void* out,
                              int64_t out_row_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  if ((M == 0 || N == 0) && M >= 0 && N >= 0 && K >= 0 &&
      (out_dtype == NTOPS_F32 || out_dtype == NTOPS_F16 || out_dtype == NTOPS_BF16))
    return NTOPS_OK;
  Mx4Args g{};
  if (const int rc = mx4_args(out_dtype, M, N, K, a, a_row_stride, a_scales, as_row_stride, b, b_row_stride, b_scales, bs_row_stride,
                              bias, out, out_row_stride, workspace, workspace_bytes, g);
      rc != NTOPS_OK)
    return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t kb = g.kb;
  return dispatch_float16_32(out_dtype, "mxfp4_mm", [&](auto tag) -> int {
    using T = decltype(tag);
    if (M <= kSkinnyRows && kb > 0) return mx4_skinny(out_dtype, g, st);
    if (large_suits(M, N) && mx4_large_serves(out_dtype, g) && workspace != nullptr &&
        workspace_bytes >= mx4_large_workspace(M, N, kb))
      return mx4_large(out_dtype, g, workspace, st);
    int bt;
    plan(M, N, std::max<int64_t>(kb, 1), bt, g.split, g.kchunk);
    if (g.split > 1 && (workspace == nullptr || workspace_bytes < g.split * M * N * 4)) {
      g.split = 1;
      g.kchunk = (g.kb + 7) / 8 * 8;
    }
    g.part = static_cast<float*>(workspace);
    return bt == 128 ? run_tile<T, 128>(g, st) : run_tile<T, 64>(g, st);
  });
}

namespace ntops {
namespace {

// Whether a product's blocks quantize these activations themselves.
bool fused(int x_dtype, int64_t M, int64_t K, const void* x, int64_t x_row_stride) {
  return (x_dtype == NTOPS_BF16 || x_dtype == NTOPS_F16) && M <= kFusedRows && K % 8 == 0 && aligned16(x) &&
         (M == 1 || (x_row_stride % 8 == 0 && x_row_stride >= 0 && x_row_stride < kMaxSize / (2 * kFusedRows) - K));
}

int64_t round16(int64_t n) { return (n + 15) & ~int64_t(15); }

}  // namespace
}  // namespace ntops

extern "C" int64_t ntops_mxfp4_linear_workspace(int x_dtype, int64_t M, int64_t N, int64_t K, const void* x,
                                                int64_t x_row_stride) {
  if (M <= 0 || N <= 0 || K <= 0 || M > kMaxCount || N > kMaxCount || K > kMaxSize || fused(x_dtype, M, K, x, x_row_stride)) return 0;
  const int64_t kb = ceil_div(K, 32);
  return round16(M * kb * 16) + round16(M * kb) + ntops_mxfp4_mm_workspace(M, N, K);
}

extern "C" int ntops_mxfp4_linear(int x_dtype, int out_dtype, int64_t M, int64_t N, int64_t K, const void* x,
                                  int64_t x_row_stride, const void* b, int64_t b_row_stride, const void* b_scales,
                                  int64_t bs_row_stride, const void* bias, void* out, int64_t out_row_stride, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || K < 0) return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: negative size");
  if (x_dtype != NTOPS_F32 && x_dtype != NTOPS_F16 && x_dtype != NTOPS_BF16)
    return set_error(NTOPS_ERR_UNSUPPORTED, "mxfp4_mm: unsupported input dtype %d (F32/F16/BF16 only)", x_dtype);
  if (M > kMaxCount || N > kMaxCount || K > kMaxSize) return set_error(NTOPS_ERR_UNSUPPORTED, "mxfp4_mm: operands too large");
  if (K > 0 && M > 0 && !x) return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: null pointer");
  const int64_t kb = ceil_div(K, 32);
  if (M == 0 || N == 0 || K == 0)
    return ntops_mxfp4_mm(out_dtype, M, N, 0, nullptr, 0, nullptr, 0, nullptr, 0, nullptr, 0, bias, out, out_row_stride, nullptr, 0, stream);
  // (all but x checked before a kernel starts; A stands in for the codes to come)
  Mx4Args g{};
  if (const int rc = mx4_args(out_dtype, M, N, K, b, kb * 16, b_scales, kb, b, b_row_stride, b_scales, bs_row_stride, bias, out,
                              out_row_stride, nullptr, 0, g);
      rc != NTOPS_OK)
    return rc;
  if (fused(x_dtype, M, K, x, x_row_stride)) {
    g.x = x;
    g.ldx = M == 1 ? 0 : x_row_stride;
    g.K = static_cast<int>(K);
    return mx4_skinny_fused(x_dtype, out_dtype, g, static_cast<hipStream_t>(stream));
  }
  const int64_t codes = round16(M * kb * 16), scales = round16(M * kb);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < codes + scales)
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: needs %lld bytes of workspace, aligned to 16",
                     static_cast<long long>(codes + scales));
  uint8_t* at = static_cast<uint8_t*>(workspace);
  if (const int rc = ntops_quantize_mxfp4(x_dtype, M, K, x, x_row_stride, at, at + codes, stream); rc != NTOPS_OK) return rc;
  return ntops_mxfp4_mm(out_dtype, M, N, K, at, kb * 16, at + codes, kb, b, b_row_stride, b_scales, bs_row_stride, bias, out,
                        out_row_stride, at + codes + scales, workspace_bytes - codes - scales, stream);
}
