// Attention of a few rows (query heads of one key head x new tokens) over a paged key-value cache, split over the length and joined.
//
// Work: the rows of a sequence that share a key head are a tile of R = 8 or 16 (more rows than that: several tiles).  The keys that a
// tile can see (a prefix and a range behind it) are units of 16 tokens, and a few more stand for its beginning.  All units, in the order
// sequence, tile, key head, unit, are divided evenly among the warps that the GPU holds at once, on the device, from the lengths: any mixture of lengths is balanced, and
// what the host knows is a bound only.  A warp's share is a part of one tile or the end of one, whole ones, and the beginning of another.
// A whole tile goes out from registers; parts are added up in shared memory, and those of tiles that several CTAs share in scratch memory,
// by the CTA that arrives last, in the order of the parts (the same bits whoever comes last).
//
// A warp takes one unit (head_dim 64: two) at a time, straight from global memory into the registers of mma.sync operands, with no
// shared memory between: scores^T [16 tokens x 8 rows] = K q^T, out^T [head_dim x 8 rows] += V^T p.  The dims of a k-step and the rows of
// an output tile are in an order of our own, the one in which a lane's 16-byte load holds what it needs:
//   K    lane (g, t): tokens g and g + 8, dims 32 j + 8 t .. + 7 (two k-steps of 16)
//   V    lane (g, t): tokens 2 t, 2 t + 1, 8 + 2 t, 9 + 2 t, dims 8 g .. + 7 and 64 + 8 g .. + 7: byte permutes pair two tokens of a dim
//   p    from the scores' accumulator by two 8x8 transposes a unit
// The next unit's keys and values are requested as soon as this one's are used.  The running maximum is raised only where a score
// is above it by more than 8 (in the exponent of 2), so the usual unit needs a vote instead of a reduction over lanes; weights
// stay below 2^8, fp32 sums take that.  Weights are rounded to the cache's type for the product with V.
//
// What bounds it: HBM for long caches (131000 tokens of 8 key heads, 537 MB, 90 us: 6.0 TB/s, 0.91 of a copy; 512 sequences of 37 to 2047
// tokens 182 us: 5.9; 64 of them, 135 MB, 31 us: 4.4); latency for short ones (32 heads at 2011, 33 MB, 13.6 us: 2 until the shares are
// known, 7 for two or three units a warp, 4 for the joins).  Before, chunks of equal length as CTAs of their own took 157, 45 and 17.5 us.
#include "paged_common.cuh"

namespace b200 {

namespace {

constexpr int kWarps = 4;
constexpr int kUnit = 16;
// A tile's beginning (its queries, the first page numbers, the way to its first keys) counts as so many units of its share: 0, 1, 2, 3, 4 units
// 15.2, 14.4, 14.1, 13.6, 13.4 us for 32 heads at 2011, 34.4, 31.2, 30.9, 31.1, 31.1 for 64 ragged sequences, 23.9, 23.8, 22.5, 22.4, 22.3 for
// 33 with a window.
constexpr int kStart = 3;
constexpr int kCtasPerSm1 = 3, kCtasPerSm2 = 2;       // of tiles of 8 rows, of 16
__device__ __forceinline__ void mma(__half, float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(__nv_bfloat16, float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
// A tile's part of a warp that is not the whole tile.
struct Piece {
  int64_t first;                                // the tile's first unit, counted over everything
  int row, tile, h, units, rows;                // the sequence's first row; rows of the tile, 0: no piece
};

// kExtra: 1 with a cap or a bias, 2 with a cap for which Cap::any will not do.
template <typename T, int D, int NT, int kExtra>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? kCtasPerSm1 : kCtasPerSm2)
paged_decode_kernel(const PagedAttnParams p) {
  constexpr int R = 8 * NT;                     // rows of a tile
  constexpr int SUB = 128 / D;                  // units a warp takes at a time
  constexpr int KC = D / 32, VC = D / 64, MT = D / 16;
  constexpr int kPitch = D + 4;
  extern __shared__ __align__(16) float sm_o[];           // [2 kWarps][R][kPitch]: a warp's first piece and its last
  __shared__ float sm_m[2 * kWarps][R], sm_l[2 * kWarps][R];
  __shared__ Piece sm_piece[2 * kWarps];
  __shared__ int sm_first[2], sm_parts[2];
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kv = p.c.kv_heads;
  auto tiles_of = [&](const Sequence& x) { return (x.rows * p.group + R - 1) / R; };

  // ---- the units of all sequences, in the order sequence, tile, key head, unit; every warp gets an equal part of them ----------
  auto units_of = [&](int i, int& per_tile) {
    const Sequence x = sequence_of(p.c, i);
    const int tiles = tiles_of(x);
    Range<kUnit> r;
    r.set(p, x, i, 0, x.rows - 1);
    per_tile = tiles > 0 ? kStart + max(r.units, 1) : 0;  // (rows that see nothing have a result too)
    return (int64_t)per_tile * tiles * kv;
  };
  int64_t mine = 0;
  int per_tile0 = 0;                            // of sequence `lane`
  int64_t units0 = 0;
#pragma unroll 1
  for (int i = lane; i < p.c.batch; i += 32) {
    int u;
    const int64_t n = units_of(i, u);
    if (i == lane) { per_tile0 = u; units0 = n; }
    mine += n;
  }
  const int64_t total = warp_sum64(mine);
  const int active = (int)min(max(total / kWarps, (int64_t)1), (int64_t)gridDim.x), warps = active * kWarps;
  if ((int)blockIdx.x >= active) return;
  const bool small = total * warps <= 0xffffffffLL;       // (a 32-bit division is a good deal shorter)
  auto share = [&](int i) { return small ? (int64_t)((unsigned)total * (unsigned)i / (unsigned)warps) : total * i / warps; };
  int64_t at = share(blockIdx.x * kWarps + warp);
  const int64_t end = share(blockIdx.x * kWarps + warp + 1);
  if (lane == 0) sm_piece[2 * warp].rows = sm_piece[2 * warp + 1].rows = 0;

  // the sequence of unit `at`, and how many units lie before it
  int b = 0, per_tile = 0;
  int64_t before = 0, seq_units = 0;
  if (at < end) {
#pragma unroll 1
    for (int base = 0; base < p.c.batch; base += 32) {
      int u = per_tile0;
      int64_t n = units0;
      if (base > 0) {
        n = 0;
        if (base + lane < p.c.batch) n = units_of(base + lane, u);
      }
      int64_t upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > at);
      if (hit) {
        const int l = __ffs(hit) - 1;
        b = base + l;
        before += __shfl_sync(0xffffffffu, upto - n, l);
        seq_units = __shfl_sync(0xffffffffu, n, l);
        per_tile = __shfl_sync(0xffffffffu, u, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  const int page = 1 << p.c.page_log2;
  const int window = p.window ? p.window : 0x7fffffff;
  const float to_log2 = p.scale * kLog2e;

  int pieces = 0;
  // (Lengths that somebody changes under the launch give no result; they must not lead behind the last sequence, or round and round.)
  while (at < end && per_tile > 0) {
    // ---- a part of one tile: units [u_begin, u_end) of all of its ---------------------------------------------------------------
    const Sequence s = sequence_of(p.c, b);
    const int in_seq = (int)(at - before), index = in_seq / per_tile, v_begin = in_seq - index * per_tile;
    const int v_end = (int)min((int64_t)per_tile, v_begin + (end - at));
    const int u_begin = max(v_begin - kStart, 0), u_end = v_end - kStart, units = per_tile - kStart;
    if (u_end > 0) {
      const int tile = index / kv, h = index - tile * kv;
      const int rows = s.rows * p.group, row0 = tile * R, nrows = min(rows - row0, R);
      const int base = s.length - s.rows;
      const int position0 = base + row0 / p.group, position1 = base + (row0 + nrows - 1) / p.group;
      Range<kUnit> range;
      range.set(p, s, b, 0, s.rows - 1);

      const T* kbase = static_cast<const T*>(p.c.k) + (int64_t)h * page * D + 8 * t;
      const T* vbase = static_cast<const T*>(p.c.v) + (int64_t)h * page * D + 8 * g;
      // units of step i; past the end the last one stands in and is masked
      auto unit_at = [&](int i, int sub) { return range.unit(min(u_begin + i * SUB + sub, u_end - 1)); };
      auto page_at = [&](int i, int sub) { return page_of(p.c, b, unit_at(i, sub) >> (p.c.page_log2 - 4)); };
      uint4 kr[SUB][2][KC], vr[SUB][4][VC];
      auto load_k = [&](int i, const int (&id)[SUB]) {
#pragma unroll
        for (int x = 0; x < SUB; ++x) {
          const T* src = kbase + id[x] * p.c.k_stride + (int64_t)((unit_at(i, x) * kUnit) & (page - 1)) * D;
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int j = 0; j < KC; ++j) kr[x][r][j] = load16(src + (g + 8 * r) * D + 32 * j);
        }
      };
      auto load_v = [&](int i, const int (&id)[SUB]) {
#pragma unroll
        for (int x = 0; x < SUB; ++x) {
          const T* src = vbase + id[x] * p.c.v_stride + (int64_t)((unit_at(i, x) * kUnit) & (page - 1)) * D;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < VC; ++j) vr[x][r][j] = load16(src + (2 * t + (r & 1) + 8 * (r >> 1)) * D + 64 * j);
        }
      };
      const int steps = (u_end - u_begin + SUB - 1) / SUB;
      int id[SUB];
#pragma unroll
      for (int x = 0; x < SUB; ++x) id[x] = page_at(0, x);
      // queries: the B operand's row g of a tile of eight
      uint4 qf[NT][KC];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = row0 + 8 * n + g;
        const T* src = static_cast<const T*>(p.q) + (int64_t)(s.first + r / p.group) * p.q_stride + (int64_t)(h * p.group + r % p.group) * D;
#pragma unroll
        for (int j = 0; j < KC; ++j) qf[n][j] = 8 * n + g < nrows ? load16(src + 32 * j + 8 * t) : make_uint4(0, 0, 0, 0);
      }
      load_k(0, id);
      load_v(0, id);
#pragma unroll
      for (int x = 0; x < SUB; ++x) id[x] = 1 < steps ? page_at(1, x) : 0;
      // this lane's rows in the accumulators: 8 n + 2 t + e
      int position[NT][2];
      float slope[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = row0 + 8 * n + 2 * t + e;
          position[n][e] = r < rows ? base + r / p.group : -1;
          slope[n][e] = kExtra && p.slopes && r < rows ? p.slopes[h * p.group + r % p.group] * kLog2e : 0.f;
        }
      float m[NT][2], l[NT][2], acc[NT][MT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) { m[n][e] = -INFINITY; l[n][e] = 0.f; }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[n][i][j] = 0.f;
      }
#pragma unroll 1
      for (int i = 0; i < steps; ++i) {
        const bool more = i + 1 < steps;
        int id_next[SUB];
#pragma unroll
        for (int x = 0; x < SUB; ++x) id_next[x] = i + 2 < steps ? page_at(i + 2, x) : 0;
        // scores of tokens g (0, 1) and g + 8 (2, 3), rows 2 t (0, 2) and 2 t + 1 (1, 3)
        float sc[SUB][NT][4];
#pragma unroll
        for (int x = 0; x < SUB; ++x)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[x][n][j] = 0.f;
#pragma unroll
            for (int j = 0; j < KC; ++j) {
              mma(T(), sc[x][n], kr[x][0][j].x, kr[x][1][j].x, kr[x][0][j].y, kr[x][1][j].y, qf[n][j].x, qf[n][j].y);
              mma(T(), sc[x][n], kr[x][0][j].z, kr[x][1][j].z, kr[x][0][j].w, kr[x][1][j].w, qf[n][j].z, qf[n][j].w);
            }
          }
        if (more) load_k(i + 1, id);
        if (kExtra == 2) {
#pragma unroll
          for (int x = 0; x < SUB; ++x)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 4; ++j) sc[x][n][j] = p.capped.of(sc[x][n][j]);
        } else if (kExtra && p.cap > 0.f) {
#pragma unroll
          for (int x = 0; x < SUB; ++x)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 4; ++j) sc[x][n][j] = p.capped.any(sc[x][n][j]);
        }
        bool above = false;
#pragma unroll
        for (int x = 0; x < SUB; ++x) {
          const int first = unit_at(i, x) * kUnit;
          const bool there = u_begin + i * SUB + x < u_end;
          // every row sees the whole unit (rows past the tile's end come out as something finite that nobody stores)
          const bool whole = there && position0 >= 0 &&
                             (first + kUnit <= range.pre || (first + kUnit - 1 <= position0 && position1 - first < window));
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int token = first + g + 8 * (j >> 1), at = position[n][j & 1];
              float v = sc[x][n][j];
              if (!(kExtra && p.cap > 0.f)) v *= to_log2;
              if (kExtra) v -= slope[n][j & 1] * fabsf((float)(at - token));
              if (!whole) {
                const bool seen = there && at >= 0 && (token < range.pre || (token <= at && at - token < window));
                if (!seen) v = -INFINITY;
              }
              sc[x][n][j] = v;
              above |= v > m[n][j & 1] + kSlack;
            }
          if (!whole) {                             // what nobody sees may be anything, and 0 * NaN is NaN
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int token = first + 2 * t + (r & 1) + 8 * (r >> 1);
              if (!(there && (token < range.pre || (token >= range.low && token < range.high))))
#pragma unroll
                for (int j = 0; j < VC; ++j) vr[x][r][j] = make_uint4(0, 0, 0, 0);
            }
          }
        }
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float v = m[n][e];
#pragma unroll
              for (int x = 0; x < SUB; ++x) v = fmaxf(v, fmaxf(sc[x][n][e], sc[x][n][e + 2]));
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
              const float f = v == -INFINITY ? 1.f : exp2_approx(m[n][e] - v);
              m[n][e] = v;
              l[n][e] *= f;
#pragma unroll
              for (int k = 0; k < MT; ++k) { acc[n][k][e] *= f; acc[n][k][e + 2] *= f; }
            }
        }
#pragma unroll
        for (int x = 0; x < SUB; ++x) {
          uint32_t pb[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              w[j] = sc[x][n][j] == -INFINITY ? 0.f : exp2_approx(sc[x][n][j] - m[n][j & 1]);
              l[n][j & 1] += w[j];
            }
            pb[n][0] = transpose8x8(pack2(T(), w[0], w[1]));
            pb[n][1] = transpose8x8(pack2(T(), w[2], w[3]));
          }
#pragma unroll
          for (int k = 0; k < MT; ++k) {
            // row g of the tile: dim 8 g + k, row g + 8: dim 64 + 8 g + k (head_dim 64: 8 g + 4 + k)
            const int k1 = D == 128 ? k : k + 4, j1 = VC - 1;
            const unsigned s0 = k & 1 ? 0x7632 : 0x5410, s1 = k1 & 1 ? 0x7632 : 0x5410;
            const uint32_t a0 = __byte_perm(word(vr[x][0][0], k / 2), word(vr[x][1][0], k / 2), s0);
            const uint32_t a1 = __byte_perm(word(vr[x][0][j1], k1 / 2), word(vr[x][1][j1], k1 / 2), s1);
            const uint32_t a2 = __byte_perm(word(vr[x][2][0], k / 2), word(vr[x][3][0], k / 2), s0);
            const uint32_t a3 = __byte_perm(word(vr[x][2][j1], k1 / 2), word(vr[x][3][j1], k1 / 2), s1);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma(T(), acc[n][k], a0, a1, a2, a3, pb[n][0], pb[n][1]);
          }
        }
        if (more) load_v(i + 1, id);
#pragma unroll
        for (int x = 0; x < SUB; ++x) id[x] = id_next[x];
      }
      // ---- the warp's rows: a whole tile goes out, a part of one to shared memory -------------------------------------------------
      const bool all = u_begin == 0 && u_end == units;
      const int slot = 2 * warp + (pieces > 0);
      if (!all && lane == 0) sm_piece[slot] = {at - v_begin + kStart, s.first, tile, h, units, nrows};
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o);
          const int r = 8 * n + 2 * t + e;
          // dims 8 g .. + 7 and 64 + 8 g .. + 7 (head_dim 64: 8 g .. + 7)
          if (all) {
            const float sum = l[n][e], inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;       // (NaN stays)
            if (r < nrows) {
              const int x = row0 + r;
              T* out = static_cast<T*>(p.out) + ((int64_t)(s.first + x / p.group) * p.heads + h * p.group + x % p.group) * D + 8 * g;
              uint32_t v[2][4];
#pragma unroll
              for (int k = 0; k < MT; k += 2) {
                v[0][(k / 2) & 3] = pack2(T(), acc[n][k][e] * inv, acc[n][k + 1][e] * inv);
                if (D == 128) v[1][k / 2] = pack2(T(), acc[n][k][e + 2] * inv, acc[n][k + 1][e + 2] * inv);
                else v[0][2 + k / 2] = pack2(T(), acc[n][k][e + 2] * inv, acc[n][k + 1][e + 2] * inv);
              }
              *reinterpret_cast<uint4*>(out) = make_uint4(v[0][0], v[0][1], v[0][2], v[0][3]);
              if (D == 128) *reinterpret_cast<uint4*>(out + 64) = make_uint4(v[1][0], v[1][1], v[1][2], v[1][3]);
            }
          } else {
            if (g == 0) { sm_m[slot][r] = m[n][e]; sm_l[slot][r] = l[n][e]; }
            float* to = sm_o + (slot * R + r) * kPitch;
#pragma unroll
            for (int k = 0; k < MT; k += 4) {
              *reinterpret_cast<float4*>(to + 8 * g + k) = make_float4(acc[n][k][e], acc[n][k + 1][e], acc[n][k + 2][e], acc[n][k + 3][e]);
              *reinterpret_cast<float4*>(to + (D == 128 ? 64 + 8 * g + k : 8 * g + 4 + k)) =
                  make_float4(acc[n][k][e + 2], acc[n][k + 1][e + 2], acc[n][k + 2][e + 2], acc[n][k + 3][e + 2]);
            }
          }
        }
      pieces += !all;
    }
    at += v_end - v_begin;
    if (at < end && at - before == seq_units) {           // the next sequence that has rows
      before += seq_units;
      do {
        ++b;
        per_tile = 0;
        seq_units = b < p.c.batch ? units_of(b, per_tile) : 0;
      } while (seq_units == 0 && b < p.c.batch);
    }
  }

  // ---- pieces of the same tile in this CTA, then those of different CTAs: the one that comes last adds them up --------------------
  // A warp takes a row at a time, a lane four of its dims (head_dim 64: two), and a part's maximum and sum in a lane of its own.
  __syncthreads();
  constexpr int kDims = D / 32;
  float v[kDims];
  auto store = [&](float* to) {
    if (kDims == 4) *reinterpret_cast<float4*>(to + 4 * lane) = make_float4(v[0], v[1], v[kDims - 2], v[kDims - 1]);
    else *reinterpret_cast<float2*>(to + 2 * lane) = make_float2(v[0], v[1]);
  };
  auto put = [&](const Piece& w, int r, float sum) {
    const int x = w.tile * R + r;
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
    T* out = static_cast<T*>(p.out) + ((int64_t)(w.row + x / p.group) * p.heads + w.h * p.group + x % p.group) * D + kDims * lane;
    if (kDims == 4) *reinterpret_cast<uint2*>(out) = make_uint2(pack2(T(), v[0] * inv, v[1] * inv), pack2(T(), v[kDims - 2] * inv, v[kDims - 1] * inv));
    else *reinterpret_cast<uint32_t*>(out) = pack2(T(), v[0] * inv, v[1] * inv);
  };
  auto warp_max = [&](float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
  };
  auto warp_add = [&](float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
  };
  const int64_t cta_begin = share(blockIdx.x * kWarps), cta_end = share(blockIdx.x * kWarps + kWarps);
  int left[2] = {-1, -1};                       // slots of tiles that other CTAs share: begun before this one's part, ended behind it
  {
    // lane x < 2 kWarps has piece x; the pieces of a tile are a group, whose first one stands for it
    const Piece mine = sm_piece[min(lane, 2 * kWarps - 1)];
    const bool there = lane < 2 * kWarps && mine.rows > 0;
    unsigned rest = __ballot_sync(0xffffffffu, there);
    int task = 0;
#pragma unroll 1
    while (rest) {
      const int s0 = __ffs(rest) - 1;
      const Piece w = sm_piece[s0];
      const unsigned group = __ballot_sync(0xffffffffu, there && mine.first == w.first);
      rest &= ~group;
      const bool begun = w.first >= cta_begin, whole = begun && w.first + w.units <= cta_end;
      const int part = (2 * blockIdx.x + begun) * R;
      if (!whole) left[begun] = s0;
#pragma unroll 1
      for (int r = 0; r < w.rows; ++r) {
        if (task++ % kWarps != warp) continue;  // (the rows of all groups in turn)
        const bool in = group >> lane & 1;
        const float m = in ? sm_m[in ? lane : 0][r] : -INFINITY, M = warp_max(m);
        const float f = m == -INFINITY ? 0.f : exp2_approx(m - M);
        const float L = warp_add(in ? sm_l[in ? lane : 0][r] * f : 0.f);
        float o[2 * kWarps][kDims];
#pragma unroll
        for (int y = 0; y < 2 * kWarps; ++y) {  // (all at once; what is in the places of no piece is not used)
          const float* from = sm_o + (y * R + r) * kPitch + kDims * lane;
          if (kDims == 4) {
            const float4 q = *reinterpret_cast<const float4*>(from);
            o[y][0] = q.x; o[y][1] = q.y; o[y][kDims - 2] = q.z; o[y][kDims - 1] = q.w;
          } else {
            const float2 q = *reinterpret_cast<const float2*>(from);
            o[y][0] = q.x; o[y][1] = q.y;
          }
        }
#pragma unroll
        for (int i = 0; i < kDims; ++i) v[i] = 0.f;
#pragma unroll
        for (int y = 0; y < 2 * kWarps; ++y) {
          const float fy = __shfl_sync(0xffffffffu, f, y);
#pragma unroll
          for (int i = 0; i < kDims; ++i) v[i] = fy != 0.f ? fmaf(fy, o[y][i], v[i]) : v[i];
        }
        if (whole) {
          put(w, r, L);
        } else {
          store(p.partial + (int64_t)(part + r) * D);
          if (lane == 0) *reinterpret_cast<float2*>(p.partial_ml + 2 * (part + r)) = make_float2(M, L);
        }
      }
    }
  }
  if (left[0] < 0 && left[1] < 0) return;
  // the CTAs from that of a tile's first unit to that of its last; its counter is the first one's
  int first_cta = 0, last_cta = 0;
  const int shared = threadIdx.x < 2 ? left[threadIdx.x] : -1;
  if (shared >= 0) {
    const Piece w = sm_piece[shared];
    auto owner = [&](int64_t unit) {
      const int64_t n = (unit + 1) * warps - 1;
      return (int)(small ? (unsigned)n / (unsigned)total : n / total) / kWarps;
    };
    first_cta = owner(w.first);
    last_cta = owner(w.first + w.units - 1);
  }
  __syncthreads();
  if (shared >= 0) {
    int n;                                      // (everybody's stores: the barrier has put them before this thread's release)
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(n) : "l"(p.arrived + first_cta) : "memory");
    const bool last = n == last_cta - first_cta;
    if (last) p.arrived[first_cta] = 0;         // (as the next launch expects it)
    sm_first[threadIdx.x] = first_cta;
    sm_parts[threadIdx.x] = last ? n + 1 : 0;
  }
  __syncthreads();
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    if (left[side] < 0 || sm_parts[side] == 0) continue;
    const Piece w = sm_piece[left[side]];
    const int first = sm_first[side], parts = sm_parts[side];
    auto row_of = [&](int c, int r) { return (2 * (first + c) + (c == 0)) * R + r; };
#pragma unroll 1
    for (int r = warp; r < w.rows; r += kWarps) {
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int i = 0; i < kDims; ++i) v[i] = 0.f;
#pragma unroll 1
      for (int c0 = 0; c0 < parts; c0 += 32) {
        const int n = min(32, parts - c0);
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane < n) ml = __ldcg(reinterpret_cast<const float2*>(p.partial_ml + 2 * row_of(c0 + lane, r)));
        float f = 0.f;
#pragma unroll 1
        for (int y0 = 0; y0 < n; y0 += 8) {
          float o[8][kDims];
#pragma unroll
          for (int y = 0; y < 8; ++y) {         // (behind the end the last one again, with weight 0)
            const float* from = p.partial + (int64_t)row_of(c0 + min(y0 + y, n - 1), r) * D + kDims * lane;
            if (kDims == 4) {
              const float4 q = __ldcg(reinterpret_cast<const float4*>(from));
              o[y][0] = q.x; o[y][1] = q.y; o[y][kDims - 2] = q.z; o[y][kDims - 1] = q.w;
            } else {
              const float2 q = __ldcg(reinterpret_cast<const float2*>(from));
              o[y][0] = q.x; o[y][1] = q.y;
            }
          }
          if (y0 == 0) {                        // (behind the loads: the maximum of these parts and those before)
            const float to = fmaxf(M, warp_max(ml.x)), old = M == -INFINITY ? 0.f : exp2_approx(M - to);
            M = to;
            f = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - M);
            L = L * old + ml.y * f;
#pragma unroll
            for (int i = 0; i < kDims; ++i) v[i] *= old;
          }
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const float fy = __shfl_sync(0xffffffffu, f, (y0 + y) & 31);
            if (y0 + y < n)
#pragma unroll
              for (int i = 0; i < kDims; ++i) v[i] = fmaf(fy, o[y][i], v[i]);
          }
        }
      }
      put(w, r, warp_add(L));
    }
  }
}

int launch_decode(const char* who, const B200PagedCache* c, PagedAttnParams p, cudaStream_t stream) {
  const int64_t most = (int64_t)c->max_query * p.group;          // rows of a sequence that share a key head
  const bool narrow = most <= 8;
  const int R = narrow ? 8 : 16;
  p.slots = sm_count() * (narrow ? kCtasPerSm1 : kCtasPerSm2);
  auto launch = [&](auto kern, SmemLimit& limit) {
    const size_t smem = (size_t)2 * kWarps * R * (c->head_dim + 4) * sizeof(float);
    int rc = raise_smem_limit(limit, reinterpret_cast<const void*>(kern), smem, who);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.slots);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = options().gemv_pdl ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return fail(B200_ELAUNCH, "%s launch: %s", who, cudaGetErrorString(e));
    count_launch();
    return B200_OK;
  };
  const int extra = p.cap > 0.f && p.capped.wide() ? 2 : p.cap > 0.f || p.slopes ? 1 : 0;
  auto by_form = [&](auto type, auto dim) {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value;
    static SmemLimit limit[2][3];
    auto by_rows = [&](auto tiles, SmemLimit* of) {
      constexpr int NT = decltype(tiles)::value;
      return extra == 0 ? launch(paged_decode_kernel<T, D, NT, 0>, of[0])
           : extra == 1 ? launch(paged_decode_kernel<T, D, NT, 1>, of[1]) : launch(paged_decode_kernel<T, D, NT, 2>, of[2]);
    };
    return narrow ? by_rows(std::integral_constant<int, 1>(), limit[0]) : by_rows(std::integral_constant<int, 2>(), limit[1]);
  };
  auto by_dim = [&](auto type) {
    return c->head_dim == 128 ? by_form(type, std::integral_constant<int, 128>()) : by_form(type, std::integral_constant<int, 64>());
  };
  return c->dtype == B200_F16 ? by_dim(__half()) : by_dim(__nv_bfloat16());
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

// The counters, the maxima and sums of parts, their partial results.  The few-rows kernel has two parts a CTA at most (a tile that began before
// its share, one that ends behind it) of 8 rows (three CTAs an SM) or 16 (two): 64 rows an SM.  The many-rows kernel has kPartsOfSlots of 256.
static_assert(2 * kCtasPerSm1 * 8 <= kPartsOfSlots * 256 && 2 * kCtasPerSm2 * 16 <= kPartsOfSlots * 256, "partial results of the few-rows kernel");
static int64_t scratch_rows() { return (int64_t)kPartsOfSlots * sm_count() * 256; }

int64_t b200_paged_attention_scratch_bytes(void) {
  if (ensure_device()) return -1;
  return B200_PAGED_ZEROED_BYTES + scratch_rows() * (2 + 128) * (int64_t)sizeof(float);
}

int b200_paged_attention(const B200PagedCache* cache, const B200PagedAttention* a, void* scratch, int64_t scratch_bytes, void* stream) {
  const char* who = "paged_attention";
  PagedAttnParams p = {};
  int rc = paged_params(who, cache, &p.c);
  if (rc) return rc;
  if (!a) return fail(B200_EINVAL, "%s: null argument descriptor", who);
  if (a->heads <= 0 || a->heads % cache->kv_heads || a->heads / cache->kv_heads > 128)
    return fail(B200_EINVAL, "%s: heads is a multiple of kv_heads, up to 128 times as many; got %d and %d", who, a->heads, cache->kv_heads);
  if (a->window < 0 || (a->window && !a->causal)) return fail(B200_EINVAL, "%s: a window is positive and needs causal", who);
  if (!(a->scale == a->scale) || !(a->cap >= 0.f && a->cap <= 1e30f)) return fail(B200_EINVAL, "%s: scale is a number, cap a number from 0 to 1e30", who);
  if (cache->tokens == 0) return B200_OK;
  if (cache->batch == 0 || cache->max_query == 0) return fail(B200_EINVAL, "%s: rows without sequences", who);
  if (a->q_stride < (int64_t)a->heads * cache->head_dim || a->q_stride % 8)
    return fail(B200_EINVAL, "%s: q_stride is a multiple of 8 and at least a row", who);
  if (!a->q || !a->out || !aligned16(a->q) || !aligned16(a->out)) return fail(B200_EINVAL, "%s: q and out must be non-null and 16-byte aligned", who);
  if (!scratch || !aligned16(scratch)) return fail(B200_EINVAL, "%s: scratch must be non-null and 16-byte aligned", who);
  if ((rc = ensure_device())) return rc;
  if (scratch_bytes < b200_paged_attention_scratch_bytes() || sm_count() * kCtasPerSm1 > kFewCounters)
    return fail(B200_EINVAL, "%s: scratch of %lld bytes is less than b200_paged_attention_scratch_bytes()", who, (long long)scratch_bytes);
  p.q = a->q;
  p.out = a->out;
  p.q_stride = a->q_stride;
  p.heads = a->heads;
  p.group = a->heads / cache->kv_heads;
  p.causal = a->causal != 0;
  // A window as long as a row of the table hides nothing.  (Up to 2^30, so that sums with it stay below 2^31.)
  p.window = a->window >= (int64_t)cache->table_width * cache->page_size ? 0 : a->window;
  p.scale = a->scale;
  p.cap = a->cap;
  p.capped = Cap(a->scale, a->cap);
  p.slopes = static_cast<const float*>(a->slopes);
  p.prefix = static_cast<const int*>(a->prefix);
  char* at = static_cast<char*>(scratch);
  p.arrived = reinterpret_cast<int*>(at);
  p.partial_ml = reinterpret_cast<float*>(at + B200_PAGED_ZEROED_BYTES);
  p.partial = p.partial_ml + 2 * scratch_rows();
  // Rows of a sequence that share a key head: up to 16 are two operand tiles of the few-rows kernel; more are cut into tiles that
  // each read the keys again, where the kernel for many rows reads them once for 256.
  if ((int64_t)cache->max_query * p.group <= 16) return launch_decode(who, cache, p, static_cast<cudaStream_t>(stream));
  return launch_paged_prompt(who, cache, p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
