// Large MXFP4 products: out (16 bits) = A B^T (+ a bias row).
//
// The persistent 256 x 256 schedule of gemm_large.hip: 4-bit data has the same
// bytes per fragment and per matrix instruction cycle as 16-bit data, so a K tile
// is again 128 bytes a row (256 values) in four half tiles (A0, A1, B0, B1) that
// are refilled one by one, the two waves of a SIMD half a phase apart, and a
// finished quadrant leaves between the next tile's MFMAs.  K is a quarter as many
// tiles as for 16 bits, so what surrounds the K loop weighs four times as much.
// In an output tile's first K tile, where the previous one leaves, the compiler keeps
// 16 to 20 registers in scratch (52 to 68 bytes a lane; gemm_large.hip's kernel none):
// up to four reloads between its MFMAs, each behind a wait for all of the wave's memory
// operations, so that there the loads do not run ahead and the stores are waited for.
//
// Scales, a byte per 32 values, ride along, 4 KiB a K tile, in a ring of three.  A
// kernel before this one lays them out by (256 rows, K tile), and within these 2
// KiB by the lane that needs them, four bytes (two 16-row slices, two k-steps) to
// a register of the MFMAs: they arrive as whole lines and are read by one
// instruction for A and one for each half of B.  Read from the tensors, 8 bytes a
// row were as many requests as the codes' lines (8192 x 4096 x 14336: 246 us against
// 224), and read from the LDS by 2 bytes, twelve reads and six combinations a K
// tile, they took a tenth of the time.
#include <algorithm>
#include <atomic>

#include "gemm_halves.h"
#include "gemm_mxfp4.h"

namespace ntops {
namespace {

// LDS: half h of the K tile in buffer b at (2 b + h) * kHalf of A's area, and of
// B's; per wave 16 rows x 64 rounded outputs, and 2 x 64 columns of the bias; three
// K tiles' scales, 256 rows of A and 256 of B each.
constexpr int kAreaB = 4 * kHalf;
constexpr int kStageOff = 8 * kHalf;
constexpr int kBiasOff = kStageOff + 8 * 2048;
constexpr int kScaleOff = kBiasOff + 8 * 256;
constexpr int kScales = 512 * 8;
constexpr int kNoneOff = kScaleOff + 3 * kScales;
constexpr int kLds = kNoneOff + 1024;
static_assert(kLds <= 163840, "LDS");

typedef __attribute__((address_space(3))) const u32x4 lds_cu32x4_t;
typedef __attribute__((address_space(3))) const u32x2 lds_cu32x2_t;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2_t;

// Loads of an operand's half tiles: 2 instructions of 1 KiB per wave, one whole
// line of 8 blocks a row.
struct CodeLoader {
  uint32_t voff[2];
  uint32_t lds_off;  // of this wave's first instruction

  // the K tile's block that this lane brings with instruction i
  __device__ __forceinline__ static int block(int wave, int lane, int i) {
    const int row = (wave * 2 + i) * 8 + lane / 8;
    return kslot<64>(row, lane % 8);
  }
  __device__ __forceinline__ void init(int64_t ld, int wave, int lane) {
    lds_off = static_cast<uint32_t>(wave * 2048);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      voff[i] = static_cast<uint32_t>(((wave * 2 + i) * 8 + lane / 8) * ld + block(wave, lane, i) * 16);
  }
  // TAIL: K tile t may reach past the row's kb blocks, which read as zero.
  template <bool TAIL>
  __device__ __forceinline__ void issue(u32x4 rsrc, uint32_t lds, int t, int kb, int wave, int lane) const {
    // (opaque, so that no sum of a fixed tile's is kept in a register)
    uint32_t koff = static_cast<uint32_t>(t * 128);
    asm volatile("" : "+s"(koff));
    const int l = TAIL ? here(lane) : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t off = voff[i] + koff;
      if constexpr (TAIL) off = t * 8 + block(wave, l, i) < kb ? off : kOOB;
      dma16(rsrc, lds + lds_off + i * 1024, off);
    }
  }
};

// Resources of an output tile's operand halves (what lies past an edge reads as
// zero) and of what this wave loads of its scales (nothing in waves 4 to 7).
struct TileRsrc {
  u32x4 a[2], b[2], s;
};

template <typename T, bool BIAS>
__global__ __launch_bounds__(512, 1) void k_mx4_large(Mx4Args g, int total) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;  // 32 rows of a half, 64 columns of a half
  const int grp = wave >> 2;
  const int tm_count = (g.M + 255) / 256, tn_count = (g.N + 255) / 256;
  const int np = (g.kb + 15) / 16;  // pairs of K tiles
  const int kt = (g.kb + 7) / 8;    // K tiles that have scales

  // tile `i` of this block: (row, column) or false past the end
  const int nx = (gridDim.x & 7) == 0 ? 8 : 1;
  const int per_x = (total + nx - 1) / nx;
  auto tile_at = [&](int i, int& m0, int& n0) __attribute__((always_inline)) {
    const int x = static_cast<int>(blockIdx.x) % nx;
    const int pos = i * (static_cast<int>(gridDim.x) / nx) + static_cast<int>(blockIdx.x) / nx;
    const int t = x * per_x + pos;
    if (pos >= per_x || t >= total) return false;
    constexpr int kGroupM = 4;
    const int gsz = kGroupM * tn_count;
    const int gi = t / gsz;
    const int gm = min(tm_count - gi * kGroupM, kGroupM);
    const int r = t - gi * gsz;
    n0 = (r / gm) * 256;
    m0 = (gi * kGroupM + r % gm) * 256;
    return true;
  };
  auto rsrc_of = [&](bool ok, int m0, int n0) __attribute__((always_inline)) {
    TileRsrc r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int mh = m0 + h * 128, nh = n0 + h * 128;
      const int mv = ok ? min(g.M - mh, 128) : 0, nv = ok ? min(g.N - nh, 128) : 0;
      r.a[h] = make_rsrc(g.a + (mv > 0 ? mh * g.lda : 0), mv > 0 ? (mv - 1) * g.lda + g.kb * 16ll : 0);
      r.b[h] = make_rsrc(g.b + (nv > 0 ? nh * g.ldb : 0), nv > 0 ? (nv - 1) * g.ldb + g.kb * 16ll : 0);
    }
    // waves 0 and 1: halves of A's 2 KiB a K tile, 2 and 3: of B's
    const int64_t panel = static_cast<int64_t>(kt) * 2048;
    const uint8_t* sc = wave < 2 ? g.as + (m0 >> 8) * panel : g.bs + (n0 >> 8) * panel;
    r.s = make_rsrc(sc, ok && wave < 4 ? panel : 0);
    return r;
  };

  CodeLoader la, lb;
  la.init(g.lda, wave, lane);
  lb.init(g.ldb, wave, lane);
  const uint32_t smem_addr = lds_addr(smem);
  const uint32_t scale_off = static_cast<uint32_t>((wave & 1) * 1024 + lane * 16);

  int m0, n0, nm0 = 0, nn0 = 0;
  if (!tile_at(0, m0, n0)) return;  // (the whole block)
  TileRsrc cur = rsrc_of(true, m0, n0), nxt;

  constexpr auto yes = std::true_type{};
  constexpr auto no = std::false_type{};
  // loads of half tile `half` of operand A / B of K tile t (buffer t & 1)
  auto dma_a = [&](auto tail, const TileRsrc& rs, int half, int t) __attribute__((always_inline)) {
    la.template issue<decltype(tail)::value>(
        rs.a[half], smem_addr + static_cast<uint32_t>(((t & 1) * 2 + half) * kHalf), t, g.kb, wave, lane);
  };
  auto dma_b = [&](auto tail, const TileRsrc& rs, int half, int t) __attribute__((always_inline)) {
    lb.template issue<decltype(tail)::value>(
        rs.b[half], smem_addr + static_cast<uint32_t>(kAreaB + ((t & 1) * 2 + half) * kHalf), t, g.kb, wave, lane);
  };
  // the scales of K tile t (past the last: zeros) into ring slot `slot`
  auto dma_s = [&](const TileRsrc& rs, int t, int slot) __attribute__((always_inline)) {
    uint32_t koff = static_cast<uint32_t>(t * 2048);
    asm volatile("" : "+s"(koff));
    // (waves 4 to 7, whose waits count alike, bring zeros that nobody reads)
    dma16(rs.s, smem_addr + static_cast<uint32_t>(wave < 4 ? kScaleOff + slot * kScales + wave * 1024 : kNoneOff),
          scale_off + koff);
  };

  // [quadrant][row tile][column tile]; quadrants 00, 10, 11, 01 (row half,
  // column half), 32 x 64 per wave
  f32x4 acc[4][2][4];
  u32x4 ax[4], ay[4], bx[4][2];  // A0, A1, one half of B
  // scales: A's [half], one half of B's [column tiles 0 and 1, 2 and 3]; byte 2 (tile & 1)
  // + k-step (lane group q: K tile's block 4 k-step + q)
  uint32_t sa[2], sb[2];
  int slot = 0;  // of the current K tile's scales
  // LDS addresses of this lane's fragments at half 0 of buffer 0, per k-step: row
  // l & 15 of the wave's part, place 4 ks + (l >> 4) of the K tile
  uint32_t abase[2], bbase[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    const int q = lane >> 4, ra = wm * 32 + (lane & 15), rb = wn * 64 + (lane & 15);
    abase[ks] = smem_addr + static_cast<uint32_t>(ra * 128 + kslot<64>(ra, 4 * ks + q) * 16);
    bbase[ks] = smem_addr + static_cast<uint32_t>(kAreaB + rb * 128 + kslot<64>(rb, 4 * ks + q) * 16);
    asm volatile("" : "+v"(abase[ks]), "+v"(bbase[ks]));
  }
  auto read_a = [&](u32x4 (&f)[4], int buf, int half) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e)  // [k-step][row tile]
      f[e] = *reinterpret_cast<lds_cu32x4_t*>(abase[e >> 1] + static_cast<uint32_t>((buf * 2 + half) * kHalf + (e & 1) * 2048));
  };
  auto read_b = [&](int buf, int half) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        bx[j][ks] = *reinterpret_cast<lds_cu32x4_t*>(bbase[ks] + static_cast<uint32_t>((buf * 2 + half) * kHalf + j * 2048));
  };
  auto read_scales = [&](int off, uint32_t (&to)[2]) __attribute__((always_inline)) {
    const u32x2 w = *reinterpret_cast<lds_cu32x2_t*>(smem_addr + static_cast<uint32_t>(kScaleOff + slot * kScales + off + here(lane) * 8));
    to[0] = w.x;
    to[1] = w.y;
  };

  // ---- epilogue: a finished quadrant (32 x 64 per wave) is rounded, 16 x 16
  // pieces between the MFMAs of the next K step, into the wave's 2 KiB of
  // staging (16 rows of 128 bytes, chunk c of row r at slot c ^ (r >> 1)) and
  // leaves as 128-byte row segments.  (A wave's LDS operations are in order:
  // the second row tile may be written once the first's reads are issued.)
  const uint32_t ep = smem_addr + static_cast<uint32_t>(kStageOff + wave * 2048);
  const uint32_t bias_lds = smem_addr + static_cast<uint32_t>(kBiasOff + wave * 256);
  int pm0 = 0, pn0 = 0;  // the tile being stored
  bool pend = false;
  auto row_half = [&](int q) __attribute__((always_inline)) { return q == 1 || q == 2; };
  auto col_half = [&](int q) __attribute__((always_inline)) { return q >= 2; };
  // the bias columns of the tile at n: lanes 0-31 the first half's, 32-63 the
  // second's, two per lane (past N: zero; an odd N's last pair is one dword)
  auto bias_dma = [&](int n) __attribute__((always_inline)) {
    const int l = here(lane);
    dma4(make_rsrc(g.bias, (static_cast<int64_t>(g.N) * 2 + 3) & ~3ll), bias_lds,
         static_cast<uint32_t>((n + (l >> 5) * 128 + wn * 64 + (l & 31) * 2) * 2));
  };
  // LDS address of this lane's 4 columns in column tile 0; column tile ct
  // flips chunk bits 1 and 2: address ^ (ct << 5)
  auto ep_base = [&](int l) __attribute__((always_inline)) {
    const int r = l & 15, c = l >> 5, half = (l >> 4) & 1;
    return ep + static_cast<uint32_t>(r * 128 + ((c ^ (r >> 1)) << 4) + half * 8);
  };
  auto bias_of = [&](int q, int l, u32x2 (&bias)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
      bias[ct] = *reinterpret_cast<lds_cu32x2_t*>(bias_lds + static_cast<uint32_t>(col_half(q) * 128 + ct * 32 + (l >> 4) * 8));
  };
  // rounds row tile i / 4, column tile i % 4 of quadrant q into the staging
  auto convert = [&](int q, int i, uint32_t base, const u32x2 (&bias)[4]) __attribute__((always_inline)) {
    const int rt = i >> 2, ct = i & 3;
    T o[4];
    if constexpr (BIAS) {
      const u32x2 raw = bias[ct];
      const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = static_cast<T>(acc[q][rt][ct][e] + static_cast<float>(t[e]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = static_cast<T>(acc[q][rt][ct][e]);
    }
    *reinterpret_cast<lds_u32x2_t*>(base ^ static_cast<uint32_t>(ct << 5)) = __builtin_bit_cast(u32x2, o);
  };
  // 16 staged rows back, 8 lanes per row: rows l / 8 and l / 8 + 8
  auto load_rows = [&](u32x4 (&rows)[2], int l) __attribute__((always_inline)) {
    const int r = l >> 3, c = l & 7;
    const uint32_t at = ep + static_cast<uint32_t>(r * 128 + ((c ^ (r >> 1)) << 4));
    rows[0] = *reinterpret_cast<lds_cu32x4_t*>(at);
    rows[1] = *reinterpret_cast<lds_cu32x4_t*>((at ^ 64u) + 1024u);
  };
  // Row tile rt of quadrant q to memory: at least 2 store instructions
  // whatever the edges (a lane with nothing to store stores past the
  // resource), which the waits of the following phases count on.  Rows may
  // start at any 2-byte address.
  auto put_rows = [&](const u32x4 (&rows)[2], int q, int rt, int l) __attribute__((always_inline)) {
    const int m = pm0 + row_half(q) * 128 + wm * 32 + rt * 16;
    const int n = pn0 + col_half(q) * 128 + wn * 64;
    const T* D = static_cast<const T*>(g.d) + static_cast<int64_t>(m) * g.ldd + n;
    const __amdgpu_buffer_rsrc_t r = buffer_rsrc_uniform(D, 0x7fffffffu);
    const int c0 = (l & 7) * 8;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = (l >> 3) + 8 * u;
      const bool in = m + row < g.M;
      const uint32_t at = static_cast<uint32_t>(row) * static_cast<uint32_t>(g.ldd) * 2 + c0 * 2;
      __builtin_amdgcn_raw_buffer_store_b128(rows[u], r, in && n + c0 + 8 <= g.N ? at : kOOB, 0, kBufNT);
      if ((g.N & 7) && pn0 + 256 > g.N) {  // the tile of the row's last, partial chunk
#pragma unroll
        for (int e = 0; e < 7; ++e)
          __builtin_amdgcn_raw_buffer_store_b16(
              static_cast<uint16_t>(rows[u][e >> 1] >> (16 * (e & 1))), r,
              in && n + c0 + 8 > g.N && n + c0 + e < g.N ? at + 2 * e : kOOB, 0, 0);
      }
    }
  };

  // the quadrant's 16 MFMAs, A of half ah; LEAVE: finished quadrant cq leaves between them -- its first row tile's
  // rows are stored under its second's conversion, its second's are left in
  // `rows` (put_rows by the caller)
  u32x4 rows[2];
  auto mfma16x = [&](auto first, auto leave, int q, const u32x4 (&af)[4], int ah, int cq) __attribute__((always_inline)) {
    constexpr bool FIRST = decltype(first)::value, LEAVE = decltype(leave)::value;
    int l = 0;
    uint32_t base = 0;
    u32x2 bias[4];
    if constexpr (LEAVE) {
      l = here(lane);
      base = ep_base(l);
      if constexpr (BIAS) bias_of(cq, l, bias);
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) {
          f32x4 c = acc[q][rt][ct];
          if (FIRST && ks == 0) c = f32x4{0.f, 0.f, 0.f, 0.f};
          const auto one = [&](auto bb, auto ab) {
            return mfma_mx4<decltype(bb)::value, decltype(ab)::value>(bx[ct][ks], sb[ct >> 1], af[ks * 2 + rt], sa[ah], c);
          };
          constexpr std::integral_constant<int, 0> i0{};
          constexpr std::integral_constant<int, 1> i1{};
          constexpr std::integral_constant<int, 2> i2{};
          constexpr std::integral_constant<int, 3> i3{};
          if (ks == 0)
            acc[q][rt][ct] = ct & 1 ? (rt ? one(i2, i2) : one(i2, i0)) : (rt ? one(i0, i2) : one(i0, i0));
          else
            acc[q][rt][ct] = ct & 1 ? (rt ? one(i3, i3) : one(i3, i1)) : (rt ? one(i1, i3) : one(i1, i1));
          if constexpr (LEAVE) {
            const int i = ks * 8 + rt * 4 + ct;  // piece i / 2 after every second MFMA
            if (i & 1) {
              __builtin_amdgcn_sched_barrier(0);
              convert(cq, i >> 1, base, bias);
              if (i == 7) load_rows(rows, l);
              if (i == 11) put_rows(rows, cq, 0, l);
              if (i == 15) load_rows(rows, l);
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
    // The compiler takes the scaled MFMA for code that it may move past barriers
    // to the result's use: here the results are used.
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(acc[q][i >> 2][i & 3]));
  };
  // ends a memory phase: its fragments are in registers, and all but the
  // wave's N youngest memory operations are done
  auto end_mem = [&](auto n_tag) __attribute__((always_inline)) {
    constexpr int N = decltype(n_tag)::value;
    __builtin_amdgcn_sched_barrier(0);
    if (N > 9 && pend)
      wait_vm<N>();
    else
      wait_vm<9>();
    wait_lgkmcnt0();
    block_barrier();
    __builtin_amdgcn_s_setprio(1);
  };
  auto end_mfma = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_setprio(0);
    block_barrier();
  };
#define NTOPS_W(n) std::integral_constant<int, (n)> {}

  // One K tile (buffer BUF): two phases.  KIND 0: the first K tile of an
  // output tile (quadrants 1 - 3 of the previous one leave), 3: the second,
  // 1: between, 2: the last (quadrant 0 leaves).  Loads issued: the scales of the
  // K tile after the next (rs2 / t2; into the slot of the K tile before this
  // one, which both groups of waves have read two barriers ago) and B1 of the next
  // (rs1 / t1), then A0, B0, A1 of the one after it.  The waits allow for the 9
  // loads issued since the ones the next phase reads, plus the stores among them
  // while a tile leaves (two per put_rows: 4, 8, 5 and 1 of them).
  auto ktile = [&](auto kind_tag, auto buf_tag, auto tail, const TileRsrc& rs1, int t1, const TileRsrc& rs2, int t2)
                   __attribute__((always_inline)) {
    constexpr int KIND = decltype(kind_tag)::value, BUF = decltype(buf_tag)::value;
    constexpr auto first = std::bool_constant<KIND == 0>{};
    // ---- phase A: quadrants 0 and 1
    read_a(ax, BUF, 0);
    read_b(BUF, 0);
    read_a(ay, BUF, 1);
    __builtin_amdgcn_sched_barrier(0);
    read_scales(wm * 512, sa);
    read_scales(2048 + wn * 512, sb);
    dma_s(rs2, t2, slot == 0 ? 2 : slot - 1);
    dma_b(tail, rs1, 1, t1);
    if constexpr (KIND == 0)
      if (pend) put_rows(rows, 1, 1, here(lane));
    end_mem(NTOPS_W(KIND == 0 ? 17 : KIND == 3 ? 19 : 9));
    if (KIND == 0 && pend) {
      mfma16x(first, yes, 0, ax, 0, 2);
      put_rows(rows, 2, 1, here(lane));
      mfma16x(first, yes, 1, ay, 1, 3);
    } else {
      mfma16x(first, no, 0, ax, 0, 0);
      mfma16x(first, no, 1, ay, 1, 0);
    }
    end_mfma();
    // ---- phase B: quadrants 2 and 3
    read_b(BUF, 1);
    __builtin_amdgcn_sched_barrier(0);
    read_scales(2048 + 1024 + wn * 512, sb);
    dma_a(tail, rs2, 0, t2);
    dma_b(tail, rs2, 0, t2);
    dma_a(tail, rs2, 1, t2);
    if constexpr (KIND == 0)
      if (pend) put_rows(rows, 3, 1, here(lane));
    end_mem(NTOPS_W(KIND == 0 ? 25 : KIND == 3 ? 11 : 9));
    if constexpr (KIND == 2) {
      pm0 = m0;
      pn0 = n0;
      mfma16x(no, yes, 2, ay, 1, 0);
      put_rows(rows, 0, 1, here(lane));
      mfma16x(no, yes, 3, ax, 0, 1);
    } else {
      mfma16x(first, no, 2, ay, 1, 0);
      mfma16x(first, no, 3, ax, 0, 0);
    }
    end_mfma();
    slot = slot == 2 ? 0 : slot + 1;
  };

  // prologue: the first K tile and the scales, A0, B0, A1 of the second in flight
  dma_s(cur, 0, 0);
  dma_a(no, cur, 0, 0);
  dma_b(no, cur, 0, 0);
  dma_a(no, cur, 1, 0);
  dma_s(cur, 1, 1);
  dma_b(no, cur, 1, 0);
  dma_a(no, cur, 0, 1);
  dma_b(no, cur, 0, 1);
  dma_a(no, cur, 1, 1);
  wait_vmcnt<9>();
  block_barrier();
  if (grp == 1) block_barrier();

  constexpr auto b0 = NTOPS_W(0);
  constexpr auto b1 = NTOPS_W(1);
  for (int it = 0;; ++it) {
    ktile(NTOPS_W(0), b0, no, cur, 1, cur, 2);
    ktile(NTOPS_W(3), b1, no, cur, 2, cur, 3);
    int t = 2;
    for (; t < 2 * np - 4; t += 2) {
      ktile(NTOPS_W(1), b0, no, cur, t + 1, cur, t + 2);
      ktile(NTOPS_W(1), b1, no, cur, t + 2, cur, t + 3);
    }
    // the loads of the last two K tiles, which may reach past K
    ktile(NTOPS_W(1), b0, yes, cur, t + 1, cur, t + 2);
    ktile(NTOPS_W(1), b1, yes, cur, t + 2, cur, t + 3);
    if constexpr (BIAS) bias_dma(n0);
    const bool more = tile_at(it + 1, nm0, nn0);
    nxt = rsrc_of(more, nm0, nn0);
    ktile(NTOPS_W(1), b0, yes, cur, t + 3, nxt, 0);
    ktile(NTOPS_W(2), b1, no, nxt, 0, nxt, 1);
    pend = true;
    if (!more) break;
    cur = nxt;
    m0 = nm0;
    n0 = nn0;
  }
#undef NTOPS_W
  if (grp == 0) block_barrier();
  put_rows(rows, 1, 1, lane);
#pragma unroll
  for (int q = 2; q < 4; ++q) {
    u32x2 bias[4];
    if constexpr (BIAS) bias_of(q, lane, bias);
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) convert(q, rt * 4 + ct, ep_base(lane), bias);
      load_rows(rows, lane);
      put_rows(rows, q, rt, lane);
    }
  }
  wait_vmcnt<0>();  // no DMA may land after the workgroup ends
}

// The scales of 256 rows and a K tile of 8 blocks to 2 KiB, by panels of 256 rows,
// then K tiles, in the order of k_mx4_large's registers: A's dword (wave row wm,
// lane, half) has rows 128 half + 32 wm + l & 15 and 16 on, B's (half, wave column
// wn, lane, pair) columns 128 half + 64 wn + 32 pair + l & 15 and 16 on; of each the
// blocks q and q + 4, q = l >> 4.  Zeros past the row's last block and the last
// row.  blockIdx.z 0: A's, 1: B's.  A block takes four K tiles, 32 bytes a row,
// through the LDS (byte by byte from memory: 10.3 us for 8192 + 14336 rows of 128).
constexpr int kLayTiles = 4;
__global__ __launch_bounds__(512) void k_mx4_lay_scales(Mx4Args g, uint8_t* a, uint8_t* b) {
  constexpr int kPitch = kLayTiles * 8 + 4;
  __shared__ uint32_t lds[256 * kPitch / 4];
  const bool of_b = blockIdx.z != 0;
  const int rows = of_b ? g.N : g.M, kt = (g.kb + 7) / 8;
  const int panel = blockIdx.x, t0 = blockIdx.y * kLayTiles;
  if (panel * 256 >= rows) return;  // (the whole block)
  {
    const int r = threadIdx.x >> 1, k = t0 * 8 + (threadIdx.x & 1) * 16;
    const uint8_t* from = (of_b ? g.bs : g.as) + (panel * 256 + r) * (of_b ? g.ldbs : g.ldas) + k;
    const int n = panel * 256 + r < rows ? min(16, g.kb - k) : 0;
    u32x4 w = {0, 0, 0, 0};
    if (n == 16 && (reinterpret_cast<uintptr_t>(from) & 15u) == 0) {
      w = *reinterpret_cast<const u32x4*>(from);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (e < n) w[e >> 2] |= static_cast<uint32_t>(from[e]) << (8 * (e & 3));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) lds[r * (kPitch / 4) + (threadIdx.x & 1) * 4 + e] = w[e];
  }
  __syncthreads();
  const int d = threadIdx.x, l = (d >> 1) & 63, low = d & 1, high = d >> 7;
  const int row = (of_b ? (high >> 1) * 128 + (high & 1) * 64 + low * 32 : low * 128 + high * 32) + (l & 15);
  const uint8_t* at = reinterpret_cast<const uint8_t*>(lds) + row * kPitch + (l >> 4);
  uint32_t* to = reinterpret_cast<uint32_t*>(of_b ? b : a) + (static_cast<int64_t>(panel) * kt + t0) * 512 + d;
#pragma unroll
  for (int t = 0; t < kLayTiles; ++t) {
    if (t0 + t >= kt) break;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) w |= static_cast<uint32_t>(at[(e >> 1) * 16 * kPitch + t * 8 + (e & 1) * 4]) << (8 * e);
    to[t * 512] = w;
  }
}

template <typename T, bool BIAS>
int launch_large(const Mx4Args& g, hipStream_t st) {
  auto kern = k_mx4_large<T, BIAS>;
  static std::atomic<uint64_t> reserved{0};
  if (const int rc = reserve_lds(reinterpret_cast<const void*>(kern), kLds, reserved, "mxfp4_mm"); rc != NTOPS_OK) return rc;
  const int64_t total = ceil_div(g.M, 256) * ceil_div(g.N, 256);
  const int64_t grid = std::min<int64_t>(total, cu_count_cached());
  note_kernel("mxfp4_large");
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(grid)), dim3(512), kLds, st, g, static_cast<int>(total));
  return check_launch("mxfp4_mm");
}

template <typename T>
int run_large(const Mx4Args& g, hipStream_t st) {
  return g.bias != nullptr ? launch_large<T, true>(g, st) : launch_large<T, false>(g, st);
}

}  // namespace

bool mx4_large_serves(int out_dtype, const Mx4Args& g) {
  return out_dtype != NTOPS_F32 && g.kb > 32 && g.kb <= 65535 * 8 && (reinterpret_cast<uintptr_t>(g.bias) & 3u) == 0 && g.ldd >= 0 &&
         (16 * g.ldd + 64) * 2 < (int64_t(1) << 31);
}

int64_t mx4_large_workspace(int64_t M, int64_t N, int64_t kb) {
  return (ceil_div(M, 256) + ceil_div(N, 256)) * ceil_div(kb, 8) * 2048;
}

int mx4_large(int out_dtype, Mx4Args g, void* workspace, hipStream_t st) {
  uint8_t* a = static_cast<uint8_t*>(workspace);
  uint8_t* b = a + ceil_div(g.M, 256) * ceil_div(g.kb, 8) * 2048;
  const unsigned panels = static_cast<unsigned>(ceil_div(std::max(g.M, g.N), 256));
  hipLaunchKernelGGL(k_mx4_lay_scales, dim3(panels, static_cast<unsigned>(ceil_div(g.kb, 8 * kLayTiles)), 2), dim3(512), 0, st, g, a, b);
  g.as = a;
  g.bs = b;
  return out_dtype == NTOPS_BF16 ? run_large<__bf16>(g, st) : run_large<_Float16>(g, st);
}

}  // namespace ntops
