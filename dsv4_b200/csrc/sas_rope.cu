// RMS norm of each head with the position rotation of its last R dims, and the
// append of shared K=V rows to a paged cache with the same norm and rotation
// on the way; forward and backward, for sm_100a.
//
//   y = R(pos) . (x * rstd * w),      rstd = 1 / sqrt(mean(x^2) + eps)
//   d = R(pos)^T . dy,  g = d * w
//   dx = rstd * (g - xh * mean(g * xh)),  dw = sum over rows of d * xh,  xh = x * rstd
//
// R(pos) turns the pair (a, b) of rotated dims by the angle of row `pos` of
// the cos / sin tables: neighbouring dims with INTER, else dim i and i + R/2
// of the rotated part. All arithmetic is fp32; a value is rounded once, when
// it is written.
//
// Everything here should be bound by memory: 4 bytes per value forward (read
// and written once in 16 bits), 6 backward, for 5-12 operations. At the rate of
// the memory an SM has 88 cycles for a forward row of 512 values, 350 issue
// slots, so the instructions of a row count: pairs of fp32 operations in one
// (f32x2), addresses that only advance, weights in registers. A row lies with G
// lanes of a warp (8 values = 16 bytes per lane and vector), so its sums are a
// few shuffles and an interleaved pair is in one lane. Warps work alone: each
// walks runs of heads of one token, which share the position, the table rows
// and the cache slot, and keeps kStages - 1 rows in flight with cp.async into
// its own shared memory, which costs no registers, so that enough warps fit.
// A call with few rows takes short runs, so that they spread over all SMs.
//
// Measured (the memory's rate is that of a plain copy, 6.5 TB/s): forward of
// 16384 tokens x 65 heads x 512 335 us, backward of 8192 tokens 248 us, both at
// that rate; append of 512 tokens with their 128 query heads 27 us (5.0 TB/s), of
// 16384 rows alone 14 us (2.7 TB/s), its backward of 8192 rows 16 us (two
// launches), 64 tokens forward 4.1 us. The calls of under 50 MB are bound by their
// start and end: launch, first loads, partial sums of the weight gradient.
#include "sas_common.cuh"

namespace {

// A set of rows [T, H] of D values: strides in elements, D contiguous.
struct Rows {
  const uint8_t* x;
  int64_t x_ts, x_hs;
  uint8_t* y;  // forward: result; backward: dx
  int64_t y_ts, y_hs;
  const uint8_t* dy;  // backward only
  int64_t dy_ts, dy_hs;
  const float* w;  // [D] or nullptr
  float* dw_part;  // backward: [blocks of this set][D] or nullptr
  int H, run, chunks;   // a token's heads are `chunks` shares of `run` rows (a warp's width each)
  uint32_t most, blocks;  // backward: shares of a warp, blocks
};

struct RopeParams {
  Rows q, k;
  int T, D, R, P, flags;
  uint32_t most;  // forward: shares of a warp
  float eps;
  const void* positions;  // [T] int32 / int64, or nullptr: the cache slot (append), no rotation elsewhere
  const float* cos;
  const float* sin;
  // append: k row t is the shared K=V row of token t; it lives in the paged pool
  uint8_t* pool;
  const int32_t* bt;
  const int32_t* cu;
  const int32_t* seqused;
  int bt_stride, bs, B, S, layout;
  int64_t nblk;
  int32_t* status;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_if(uint32_t dst, const void* src, bool on) {  // zeros if not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two fp32 values in a register pair, and operations on both at once.
struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ float lo() const { return __uint_as_float((uint32_t)v); }
  __device__ __forceinline__ float hi() const { return __uint_as_float((uint32_t)(v >> 32)); }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

template <int DT>
__device__ __forceinline__ void unpack8(const uint4& r, F2 (&f)[4]) {
  const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (DT == SAS_DTYPE_BF16) {
      f[i] = F2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    } else {
      const float2 v = __half22float2(reinterpret_cast<const __half2&>(u[i]));
      f[i] = F2(v.x, v.y);
    }
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const F2 (&f)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (DT == SAS_DTYPE_BF16) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(f[i].lo(), f[i].hi());
      u[i] = reinterpret_cast<const uint32_t&>(v);
    } else {
      const __half2 v = __floats2half2_rn(f[i].lo(), f[i].hi());
      u[i] = reinterpret_cast<const uint32_t&>(v);
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The request that a warp's token is in and the page that its slot is in. A
// warp's tokens are neighbours, so both are mostly those of the token before.
// Every lane of the warp calls it.
struct Slots {
  int b = -1, c0 = 0, n = 0, used = 0, col = -1, blk = -1;
  // TND: the 31 requests around the one that an even split would give are
  // looked at first, then cu_seqlens_q is searched 32 ways at a time. The last
  // round reads the lengths beside it.
  __device__ __forceinline__ void find(const RopeParams& p, int t, int lane) {
    if (b >= 0 && t >= c0 && t < c0 + n) return;
    col = -1;
    if (p.layout == SAS_LAYOUT_TND) {
      int len = min(p.B, 31), lo = min(max((int)((int64_t)t * p.B / p.T) - 15, 0), p.B - len);
      int mine, su;
      auto read = [&]() {
        mine = lane <= len ? __ldg(p.cu + lo + lane) : 0x7fffffff;
        su = lane < len ? __ldg(p.seqused + lo + lane) : 0;
      };
      read();
      if (__shfl_sync(0xffffffffu, mine, 0) > t || __shfl_sync(0xffffffffu, mine, len) <= t) {
        lo = 0, len = p.B;  // the last request in [lo, lo + len) with cu <= t
        while (len > 31) {
          const int stride = (len + 31) >> 5;
          const int c = lo + lane * stride;
          const bool le = c < lo + len && __ldg(p.cu + c) <= t;
          const int last = 31 - __clz(__ballot_sync(0xffffffffu, le) | 1u);
          const int at = lo + last * stride;
          len = min(stride, lo + len - at);
          lo = at;
        }
        read();
      }
      const int k = 31 - __clz(__ballot_sync(0xffffffffu, lane < len && mine <= t) | 1u);
      c0 = __shfl_sync(0xffffffffu, mine, k);
      n = __shfl_sync(0xffffffffu, mine, k + 1) - c0;
      used = __shfl_sync(0xffffffffu, su, k);
      b = lo + k;
    } else {
      b = t / p.S;
      c0 = b * p.S;
      n = p.cu ? __ldg(p.cu + b + 1) - __ldg(p.cu + b) : p.S;
      used = __ldg(p.seqused + b);
    }
  }
  // Slot of token t and, if wanted, the pool row of that slot. -1: none; the
  // column past the table's width or an entry past the pool is also recorded.
  __device__ __forceinline__ int64_t row(const RopeParams& p, int t, int lane, int& slot, bool want_row) {
    find(p, t, lane);
    const int i = t - c0;
    slot = -1;
    if (i < 0 || i >= n) return -1;  // BSND padding, or a token past cu_seqlens_q's end
    slot = used - n + i;
    if (!want_row || slot < 0) return -1;
    const int c = slot / p.bs;
    if (c != col) {
      col = c;
      blk = c < p.bt_stride ? __ldg(p.bt + (int64_t)b * p.bt_stride + c) : 0x7fffffff;
      if (blk >= p.nblk) {
        if (lane == 0 && p.status) atomicCAS(p.status, 0, SAS_ERR_BAD_BLOCK_ENTRY);
        blk = -1;
      }
    }
    return blk < 0 ? -1 : (int64_t)blk * p.bs + (slot - c * p.bs);
  }
};

// Row of the cos / sin tables of token t. A position outside the tables takes
// the nearest row and is recorded, in an append by the token's K=V row and only
// if that has a slot: padding, of which nothing is written to the cache, may have any.
__device__ __forceinline__ int table_row(const RopeParams& p, int t, int slot, int lane) {
  int64_t pos = slot;
  if (p.positions)
    pos = (p.flags & SAS_ROPE_POS64) ? __ldg(static_cast<const long long*>(p.positions) + t)
                               : __ldg(static_cast<const int32_t*>(p.positions) + t);
  if (pos < 0 || pos >= p.P) {
    if (lane == 0 && p.status && !(p.pool && slot < 0)) atomicCAS(p.status, 0, SAS_ERR_BAD_POSITION);
    pos = pos < 0 ? 0 : p.P - 1;
  }
  return (int)pos;
}

// a * b - c * d to about an ulp of the result however much cancels (Kahan's
// difference of products)
__device__ __forceinline__ float diff_of_products(float a, float b, float c, float d) {
  const float cd = c * d;
  return fmaf(a, b, -cd) + fmaf(-c, d, cd);
}

// Where a lane's vector lies in the rotation, the same for every row.
struct Place {
  int angle;    // first angle of the vector, -1: it is not rotated
  int partner;  // halves: the partner's vector
  float sgn;    // halves: the sine's sign, down for the lower half
};
template <bool INTER>
__device__ __forceinline__ Place place_of(int v, int D, int R, float sgn) {
  const int e = v * 8 - (D - R);
  if (e < 0 || v * 8 >= D) return Place{-1, v, sgn};
  if (INTER) return Place{e / 2, v, sgn};
  return e < R / 2 ? Place{e, v + R / 16, -sgn} : Place{e - R / 2, v - R / 16, sgn};
}

// A rotated vector turned; table: its token's [cos R/2][sin R/2]; o: the
// partner's values (halves only). EXACT: values that cancel keep their relative
// accuracy (a weight's gradient is a sum of products of them).
template <bool INTER, bool EXACT>
__device__ __forceinline__ void turn(F2 (&f)[4], const F2 (&o)[4], const float* table, const Place& at, int R) {
  const float4* pc = reinterpret_cast<const float4*>(table + at.angle);
  const float4* ps = reinterpret_cast<const float4*>(table + at.angle + R / 2);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 c4 = pc[INTER ? 0 : i / 2], s4 = ps[INTER ? 0 : i / 2];
    const float cs[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
    const float a = f[i].lo(), b = f[i].hi();
    if (INTER) {
      const float c = cs[i], s = at.sgn * ss[i];
      f[i] = EXACT ? F2(diff_of_products(a, c, b, s), diff_of_products(b, c, -a, s)) : F2(a * c - b * s, a * s + b * c);
    } else {
      const float x = o[i].lo(), y = o[i].hi(), s0 = at.sgn * ss[2 * (i & 1)], s1 = at.sgn * ss[2 * (i & 1) + 1];
      const float c0 = cs[2 * (i & 1)], c1 = cs[2 * (i & 1) + 1];
      f[i] = EXACT ? F2(diff_of_products(a, c0, -x, s0), diff_of_products(b, c1, -y, s1)) : F2(a * c0 + x * s0, b * c1 + y * s1);
    }
  }
}

__device__ __forceinline__ void weight8(const float* w, int v, F2 (&f)[4]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(w + v * 8));
  const float4 b = __ldg(reinterpret_cast<const float4*>(w + v * 8 + 4));
  f[0] = F2(a.x, a.y), f[1] = F2(a.z, a.w), f[2] = F2(b.x, b.y), f[3] = F2(b.z, b.w);
}

constexpr int kWarps = 8;
// blocks of an SM, by registers
__host__ __device__ constexpr int fwd_blocks(int nv) { return nv == 1 ? 3 : 2; }
__host__ __device__ constexpr int bwd_blocks(int nv) { return nv > 2 ? 1 : 2; }
__host__ __device__ constexpr int stages_of(int nv) { return nv > 2 ? 2 : 4; }  // rows of a warp in flight or in work

// The shares of a warp: every warps-th one, so that the GPU's reads stay close
// together (3% faster for 16384 x 64 x 512), or `most` neighbours where
// shares need the token's slot, whose request and page then stay.
struct Walk {
  uint32_t first, end, step;
  __device__ __forceinline__ Walk(uint32_t warp, uint32_t warps, uint32_t all, uint32_t most)
      : first(most ? min(warp * most, all) : warp), end(most ? min(first + most, all) : all), step(most ? 1 : warps) {}
};

// A share's result, from the warp's side that loads to the one that computes.
struct __align__(16) Share {
  uint8_t* y;  // first row (nullptr: nothing is written)
  int n, isk;
};

// DT: type; G lanes hold a row, NV vectors of 8 values each; FULL: D = 8 * G * NV.
template <int DT, int G, int NV, bool FULL, bool INTER>
__global__ void __launch_bounds__(32 * kWarps, fwd_blocks(NV)) rope_fwd_kernel(const __grid_constant__ RopeParams p) {
  constexpr int HW = 32 / G, S = stages_of(NV), STAGE = NV * 512;
  static_assert(HW == 1 || FULL, "rows side by side are whole");
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Share s_share[kWarps][S];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % G, sub = lane / G;
  uint8_t* mine = smem + warp * S * (STAGE + p.R * 4);  // rows, then tables
  const uint32_t base = sas::smem_u32(mine) + lane * 16, tables = sas::smem_u32(mine) + S * STAGE;
  const float invD = 1.f / (float)p.D;
  const bool norm = p.flags & SAS_ROPE_NORM;
  bool on[NV];  // the lane has the vector
  Place at[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    on[j] = FULL || (gl + G * j) * 8 < p.D;
    at[j] = place_of<INTER>(gl + G * j, p.D, p.R, (p.flags & SAS_ROPE_INVERSE) ? -1.f : 1.f);
  }
  // ---- the loading side: units of the walk, rows of the unit
  const uint32_t per = p.q.chunks + p.k.chunks, all = (uint32_t)p.T * per;
  const Walk walk(blockIdx.x * kWarps + warp, gridDim.x * kWarps, all, p.pool && !p.positions || !p.q.H ? p.most : 0);
  uint32_t unit = walk.first, share_in = 0, row_in = 0;
  Slots slots;
  int left = 0, hleft = 0;
  const uint8_t* x = nullptr;
  int64_t xs = 0;
  const uint8_t* rs0 = p.q.H ? p.q.x : p.k.x;  // a valid address for copies of nothing
  auto issue = [&]() {
    if (left == 0 && unit < walk.end) {
      const uint32_t t = unit / per;
      int c = (int)(unit - t * per);
      const bool isk = c >= p.q.chunks;
      const Rows& rs = isk ? p.k : p.q;
      if (isk) c -= p.q.chunks;
      const int h0 = c * rs.run * HW;
      hleft = rs.H - h0;
      left = min(rs.run, (hleft + HW - 1) / HW);
      x = rs.x + ((int64_t)t * rs.x_ts + (int64_t)(h0 + sub) * rs.x_hs) * 2 + gl * 16;
      xs = rs.x_hs * 2 * HW;
      int slot = -1;
      int64_t row = -1;
      if (p.pool && (isk || !p.positions)) row = slots.row(p, t, lane, slot, isk);
      if (p.R > 0) {
        const int64_t tr = (int64_t)table_row(p, t, slot, lane) * (p.R / 2);
        for (int i = lane; i < p.R / 4; i += 32)
          cp16(tables + (share_in % S) * p.R * 4 + i * 16, (i < p.R / 8 ? p.cos : p.sin - p.R / 2) + tr + i * 4);
      }
      if (lane == 0) {
        uint8_t* y = p.pool && isk ? (row < 0 ? nullptr : p.pool + row * p.D * 2)
                                   : rs.y + ((int64_t)t * rs.y_ts + (int64_t)h0 * rs.y_hs) * 2;
        s_share[warp][share_in % S] = Share{y, min(hleft, rs.run * HW), isk};
      }
      ++share_in;
      unit += walk.step;
    }
    if (left > 0) {
      const uint32_t dst = base + (row_in % S) * STAGE;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (FULL && HW == 1) {
          cp16(dst + j * 512, x + G * 16 * j);
        } else {
          const bool there = (HW == 1 || sub < hleft) && on[j];
          cp16_if(dst + j * 512, there ? x + G * 16 * j : rs0, there);
        }
      }
      x += xs;
      hleft -= HW;
      ++row_in;
      --left;
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) issue();
  // ---- the computing side
  F2 w[NV][4];
  int whose = -1;
  uint32_t row_out = 0;
  for (uint32_t u = walk.first, share = 0; u < walk.end; u += walk.step, ++share) {
    uint8_t* y = nullptr;
    int64_t ys = 0;
    int n = 1, hn = 1;
    bool hasw = false;
    const float* wt = nullptr;
    for (int i = 0; i < n; ++i) {
      issue();
      cp_wait<S - 1>();
      __syncwarp();
      if (i == 0) {
        const Share sh = s_share[warp][share % S];
        const Rows& rs = sh.isk ? p.k : p.q;
        hn = sh.n;
        n = (hn + HW - 1) / HW;
        ys = rs.y_hs * 2 * HW;
        y = sh.y ? sh.y + (int64_t)sub * rs.y_hs * 2 + gl * 16 : nullptr;
        wt = rs.w;
        hasw = wt != nullptr;
        if (hasw && whose != sh.isk) {
          whose = sh.isk;
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (on[j]) weight8(wt, gl + G * j, w[j]);
        }
      }
      const uint4* xr = reinterpret_cast<const uint4*>(mine + (row_out % S) * STAGE);
      F2 f[NV][4], ss(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        unpack8<DT>(xr[j * 32 + lane], f[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) ss = fma2(f[j][e], f[j][e], ss);
      }
      if (norm) {
        const float rstd = rsqrtf(group_sum<G>(ss.lo() + ss.hi()) * invD + p.eps);
        const F2 rr(rstd, rstd);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) f[j][e] = mul2(f[j][e], rr);
        if (hasw)
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) f[j][e] = mul2(f[j][e], w[j][e]);
        ss = rr;
      } else {
        ss = F2(1.f, 1.f);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (at[j].angle >= 0) {
          F2 o[4];
          if (!INTER) {
            unpack8<DT>(xr[at[j].partner / G * 32 + sub * G + at[j].partner % G], o);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = mul2(o[e], ss);
            if (hasw) {
              F2 wp[4];
              weight8(wt, at[j].partner, wp);
#pragma unroll
              for (int e = 0; e < 4; ++e) o[e] = mul2(o[e], wp[e]);
            }
          }
          turn<INTER, false>(f[j], o, reinterpret_cast<const float*>(mine + S * STAGE) + (share % S) * p.R, at[j], p.R);
        }
        if (y && on[j] && (HW == 1 || i * HW + sub < hn)) *reinterpret_cast<uint4*>(y + G * 16 * j) = pack8<DT>(f[j]);
      }
      if (y) y += ys;
      ++row_out;
      __syncwarp();  // the stage is overwritten next
    }
  }
}

// Backward. Blocks [0, q.blocks) take the q rows, the rest the k rows; a warp
// keeps the weight gradient of its columns in registers. Each block adds its
// warps' sums in order and writes one row of partials; sum_partials_kernel
// adds the rows in order, so the result does not depend on timing.
template <int DT, int G, int NV, bool FULL, bool INTER, bool HASW>
__global__ void __launch_bounds__(32 * kWarps, bwd_blocks(NV)) rope_bwd_kernel(const __grid_constant__ RopeParams p) {
  constexpr int HW = 32 / G, S = stages_of(NV), STAGE = 2 * NV * 512;
  static_assert(HW == 1 || FULL, "rows side by side are whole");
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % G, sub = lane / G;
  const bool isk = blockIdx.x >= p.q.blocks;
  const Rows& rs = isk ? p.k : p.q;
  const uint32_t blk = isk ? blockIdx.x - p.q.blocks : blockIdx.x;
  uint8_t* mine = smem + warp * S * (STAGE + p.R * 4);
  const uint32_t base = sas::smem_u32(mine) + lane * 16, tables = sas::smem_u32(mine) + S * STAGE;
  const bool norm = p.flags & SAS_ROPE_NORM;
  const float invD = 1.f / (float)p.D;
  bool on[NV];
  Place at[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    on[j] = FULL || (gl + G * j) * 8 < p.D;
    at[j] = place_of<INTER>(gl + G * j, p.D, p.R, (p.flags & SAS_ROPE_INVERSE) ? 1.f : -1.f);  // the transpose turns back
  }
  const uint32_t per = rs.chunks, all = (uint32_t)p.T * per;
  const Walk walk(blk * kWarps + warp, rs.blocks * kWarps, all, p.pool ? rs.most : 0);
  Slots slots;
  uint32_t unit = walk.first, share_in = 0, row_in = 0;
  int left = 0, hleft = 0;
  bool have = true;
  uint32_t skip = 0;  // append, a token being one row: of the last 32 rows asked for, those that were not written
  const uint8_t *x = nullptr, *dy = nullptr;
  const int64_t xs = rs.x_hs * 2 * HW, ds = rs.dy_hs * 2 * HW, ys = rs.y_hs * 2 * HW;
  auto issue = [&]() {
    if (left == 0 && unit < walk.end) {
      const uint32_t t = unit / per;
      const int h0 = (int)(unit - t * per) * rs.run * HW;
      hleft = rs.H - h0;
      left = min(rs.run, (hleft + HW - 1) / HW);
      int slot = -1;
      int64_t row = 0;
      x = rs.x + ((int64_t)t * rs.x_ts + (int64_t)(h0 + sub) * rs.x_hs) * 2 + gl * 16;
      if (p.pool) {
        row = slots.row(p, t, lane, slot, true);
        skip = (skip & ~(1u << (row_in & 31))) | ((row < 0 ? 1u : 0u) << (row_in & 31));
      }
      have = row >= 0;
      dy = (p.pool ? p.pool + (have ? row : 0) * p.D * 2 : rs.dy + (int64_t)t * rs.dy_ts * 2) +
           (int64_t)(h0 + sub) * rs.dy_hs * 2 + gl * 16;
      if (p.R > 0) {
        const int64_t tr = (int64_t)table_row(p, t, slot, lane) * (p.R / 2);
        for (int i = lane; i < p.R / 4; i += 32)
          cp16(tables + (share_in % S) * p.R * 4 + i * 16, (i < p.R / 8 ? p.cos : p.sin - p.R / 2) + tr + i * 4);
      }
      ++share_in;
      unit += walk.step;
    }
    if (left > 0) {
      const uint32_t dst = base + (row_in % S) * STAGE;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const bool there = (HW == 1 || sub < hleft) && on[j];
        if (!(FULL && HW == 1)) cp16_if(dst + j * 512, there ? x + G * 16 * j : rs.x, there && norm);
        else if (norm) cp16(dst + j * 512, x + G * 16 * j);
        cp16_if(dst + (NV + j) * 512, there ? dy + G * 16 * j : rs.x, there && have);
      }
      x += xs;
      dy += ds;
      hleft -= HW;
      ++row_in;
      --left;
    }
    cp_commit();
  };
  // without the norm the gradient is the rotation's and has no part of x, which is not
  // read: zeros stand in its place
  if (!norm)
    for (int i = 0; i < S * NV; ++i)
      *reinterpret_cast<uint4*>(mine + (i / NV) * STAGE + (i % NV) * 512 + lane * 16) = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < S - 1; ++i) issue();
  const bool hasw = rs.w != nullptr;
  F2 acc[NV][4], w[NV][4];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = F2(0.f, 0.f), w[j][e] = F2(1.f, 1.f);
    if (hasw && on[j]) weight8(rs.w, gl + G * j, w[j]);
  }
  uint32_t row_out = 0, share = 0;
  for (uint32_t u = walk.first; u < walk.end; u += walk.step, ++share) {
    const uint32_t t = u / per;
    const int h0 = (int)(u - t * per) * rs.run * HW, hn = min(rs.H - h0, rs.run * HW);
    uint8_t* y = rs.y + ((int64_t)t * rs.y_ts + (int64_t)(h0 + sub) * rs.y_hs) * 2 + gl * 16;
    if (p.pool && ((skip >> (row_out & 31)) & 1u)) {  // zero whatever the raw row holds, and no part of the weight's gradient
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (on[j] && sub == 0) *reinterpret_cast<uint4*>(y + G * 16 * j) = make_uint4(0, 0, 0, 0);
      issue();
      cp_wait<S - 1>();  // its copies are done before the stage is filled again
      __syncwarp();
      ++row_out;
      continue;
    }
    for (int i = 0; i * HW < hn; ++i) {
      issue();
      cp_wait<S - 1>();
      __syncwarp();
      const uint4* xr = reinterpret_cast<const uint4*>(mine + (row_out % S) * STAGE);
      const uint4* dr = xr + NV * 32;
      F2 f[NV][4], g[NV][4], ss(0.f, 0.f), gx(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        unpack8<DT>(xr[j * 32 + lane], f[j]);
        unpack8<DT>(dr[j * 32 + lane], g[j]);
        if (at[j].angle >= 0) {
          F2 o[4];
          if (!INTER) unpack8<DT>(dr[at[j].partner / G * 32 + sub * G + at[j].partner % G], o);
          turn<INTER, true>(g[j], o, reinterpret_cast<const float*>(mine + S * STAGE) + (share % S) * p.R, at[j], p.R);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ss = fma2(f[j][e], f[j][e], ss);
          gx = fma2(mul2(g[j][e], w[j][e]), f[j][e], gx);
        }
      }
      float rstd = 1.f, mean = 0.f;  // mean of g * xhat
      if (norm) {
        rstd = rsqrtf(group_sum<G>(ss.lo() + ss.hi()) * invD + p.eps);
        // lanes past the last head hold zeros: their xh has to be zero with eps = 0 too
        if (HW > 1 && i * HW + sub >= hn) rstd = 0.f;
        mean = rstd * group_sum<G>(gx.lo() + gx.hi()) * invD;
      }
      const F2 r2(rstd, rstd), m2(-mean, -mean);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const F2 xh = mul2(f[j][e], r2);
          if (HASW) acc[j][e] = fma2(g[j][e], xh, acc[j][e]);
          f[j][e] = mul2(r2, fma2(xh, m2, mul2(g[j][e], w[j][e])));
        }
        if (on[j] && (HW == 1 || i * HW + sub < hn)) *reinterpret_cast<uint4*>(y + G * 16 * j) = pack8<DT>(f[j]);
      }
      y += ys;
      ++row_out;
      __syncwarp();  // the stage is overwritten next
    }
  }
  if (HASW && rs.dw_part) {
    __syncthreads();  // every warp is done with its stages
    float* red = reinterpret_cast<float*>(smem);  // [kWarps * HW][D]
    float* my = red + (warp * HW + sub) * p.D;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!on[j]) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) my[(gl + G * j) * 8 + 2 * e] = acc[j][e].lo(), my[(gl + G * j) * 8 + 2 * e + 1] = acc[j][e].hi();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
      float s = 0.f;
      for (int r = 0; r < kWarps * HW; ++r) s += red[r * p.D + d];
      rs.dw_part[(int64_t)blk * p.D + d] = s;
    }
  }
}

// dw[d] = sum over rows of part[row][d], in a fixed order: 32 columns per
// block, 8 warps take every 8th row, then the warps' sums in order.
__global__ void __launch_bounds__(256) sum_partials_kernel(const float* qp, float* qw, int qn, const float* kp,
                                                           float* kw, int kn, int D) {
  __shared__ float s[8][33];
  const float* part = blockIdx.y ? kp : qp;
  float* out = blockIdx.y ? kw : qw;
  const int n = blockIdx.y ? kn : qn;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane;
  if (!out) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (d < D)
    for (int r = warp; r < n; r += 32)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r + 8 * i < n) v[i] += part[(int64_t)(r + 8 * i) * D + d];
  s[warp][lane] = (v[0] + v[1]) + (v[2] + v[3]);
  __syncthreads();
  if (warp == 0 && d < D) {
    float t = 0.f;
    for (int i = 0; i < 8; ++i) t += s[i][lane];
    out[d] = t;
  }
}

// --------------------------------------------------------------- host side
int lanes_of(int D) { return D == 64 ? 8 : (D == 128 ? 16 : 32); }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool rows_ok(const Rows& r, bool bwd) {
  if (r.H <= 0) return r.H == 0;
  if (!r.x || !r.y || !aligned16(r.x) || !aligned16(r.y)) return false;
  if ((r.x_ts | r.x_hs | r.y_ts | r.y_hs) & 7) return false;
  if (r.w && !aligned16(r.w)) return false;
  return !bwd || !r.dy || (aligned16(r.dy) && ((r.dy_ts | r.dy_hs) & 7) == 0);
}

int check(const RopeParams& p, int dtype, bool bwd) {
  if (dtype != SAS_DTYPE_BF16 && dtype != SAS_DTYPE_FP16) return SAS_ERR_UNSUPPORTED;
  if (p.T < 0 || p.D <= 0 || p.D > 1024 || p.D % 8) return SAS_ERR_INVALID_ARG;
  if (p.R < 0 || p.R > p.D || p.R % ((p.flags & SAS_ROPE_INTERLEAVED) ? 8 : 16)) return SAS_ERR_INVALID_ARG;
  if (p.R > 0 && (!p.cos || !p.sin || !aligned16(p.cos) || !aligned16(p.sin) || p.P <= 0)) return SAS_ERR_INVALID_ARG;
  if (p.R > 0 && !p.positions && !p.pool) return SAS_ERR_INVALID_ARG;
  if (!rows_ok(p.q, bwd) || p.q.H + p.k.H <= 0) return SAS_ERR_INVALID_ARG;
  if (!(p.flags & SAS_ROPE_NORM) && (p.q.w || p.k.w)) return SAS_ERR_INVALID_ARG;
  return SAS_OK;
}

int check_paged(const RopeParams& p) {
  if (!p.pool || !aligned16(p.pool) || !p.bt || !p.seqused || p.bs <= 0 || p.bt_stride <= 0 || p.nblk < 0 || p.B <= 0)
    return SAS_ERR_INVALID_ARG;
  if (p.layout == SAS_LAYOUT_TND ? !p.cu : (p.layout != SAS_LAYOUT_BSND || p.S <= 0)) return SAS_ERR_INVALID_ARG;
  if (p.layout == SAS_LAYOUT_BSND && (int64_t)p.B * p.S != p.T) return SAS_ERR_INVALID_ARG;
  return SAS_OK;
}

#define ROPE_SHAPES(F)                      \
  if (D == 64) F(8, 1, true)                \
  else if (D == 128) F(16, 1, true)         \
  else if (D == 256) F(32, 1, true)         \
  else if (D == 512) F(32, 2, true)         \
  else if (D < 256) F(32, 1, false)         \
  else if (D < 512) F(32, 2, false)         \
  else F(32, 4, false)

int vectors_of(int D) {
  const int nv = (D / 8 + lanes_of(D) - 1) / lanes_of(D);
  return nv == 3 ? 4 : nv;
}
int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 1;
  return n;
}

// How T tokens of the sets a and b (b may be nullptr) are shared out over at
// most `warps` warps: rows of a share (up to most_rows) and shares of a warp. The
// slowest warp's time counts: its rows, and about two rows' more per share.
// Measured for 16384 x 64 x 512 forward: up to 8 rows 335 us, 6 377, 16 371;
// 8192 x 64 x 512 backward: up to 4 rows 250 us, 3 257, 8 293.
bool share_out(int64_t T, Rows* a, Rows* b, int hw, int64_t warps, int most_rows, uint32_t* most) {
  double best = 0;
  for (int run = most_rows; run >= 1; --run) {
    const int64_t ca = (a->H + run * hw - 1) / (run * hw), cb = b ? (b->H + run * hw - 1) / (run * hw) : 0;
    const int64_t units = T * (ca + cb), per = (units + warps - 1) / warps;
    if (units >= (1ll << 31) || per * warps >= (1ll << 32)) return false;
    const int64_t widest = a->H > (b ? b->H : 0) ? a->H : b ? b->H : a->H;
    const int64_t rows = (widest + hw - 1) / hw < run ? (widest + hw - 1) / hw : run;
    const double cost = (double)per * ((double)rows + 2);
    if (best == 0 || cost < best) {
      best = cost;
      a->run = run, a->chunks = (int)ca;
      if (b) b->run = run, b->chunks = (int)cb;
      *most = (uint32_t)(per > 0 ? per : 1);
    }
  }
  return true;
}

template <typename K>
int launch(K kern, const RopeParams& p, int blocks, int smem, cudaStream_t st) {
  if (smem > 47 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return SAS_ERR_CUDA;
  kern<<<blocks, 32 * kWarps, smem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
}

template <int DT, bool INTER>
int launch_fwd(const RopeParams& p, int blocks, int smem, cudaStream_t st) {
  const int D = p.D;
#define F(G, NV, FULL) return launch(rope_fwd_kernel<DT, G, NV, FULL, INTER>, p, blocks, smem, st);
  ROPE_SHAPES(F)
#undef F
}

int fwd(RopeParams& p, int dtype, cudaStream_t st) {
  if (p.T == 0) return SAS_OK;
  const int hw = 32 / lanes_of(p.D), nv = vectors_of(p.D);
  const bool inter = p.flags & SAS_ROPE_INTERLEAVED;
  const int64_t most = (int64_t)sm_count() * fwd_blocks(nv);
  if (!share_out(p.T, &p.q, &p.k, hw, most * kWarps, 8, &p.most)) return SAS_ERR_UNSUPPORTED;
  const int64_t fit = ((int64_t)p.T * (p.q.chunks + p.k.chunks) + kWarps - 1) / kWarps;
  const int blocks = (int)(fit < most ? fit : most);
  const int smem = kWarps * stages_of(nv) * (nv * 512 + p.R * 4);
  if (dtype == SAS_DTYPE_BF16)
    return inter ? launch_fwd<SAS_DTYPE_BF16, true>(p, blocks, smem, st) : launch_fwd<SAS_DTYPE_BF16, false>(p, blocks, smem, st);
  return inter ? launch_fwd<SAS_DTYPE_FP16, true>(p, blocks, smem, st) : launch_fwd<SAS_DTYPE_FP16, false>(p, blocks, smem, st);
}

constexpr int kBwdBlocks = 148 * 2;  // most blocks of a set of rows; its partials are one row of D floats per block

template <int DT, bool INTER, bool HASW>
int launch_bwd(const RopeParams& p, int smem, cudaStream_t st) {
  const int D = p.D;
#define F(G, NV, FULL) return launch(rope_bwd_kernel<DT, G, NV, FULL, INTER, HASW>, p, p.q.blocks + p.k.blocks, smem, st);
  ROPE_SHAPES(F)
#undef F
}

int bwd(RopeParams& p, int dtype, float* dqw, float* dkw, void* ws, size_t ws_bytes, cudaStream_t st) {
  if ((dqw && !p.q.w) || (dkw && !p.k.w)) return SAS_ERR_INVALID_ARG;
  const size_t part = (size_t)kBwdBlocks * p.D * 4;
  if ((dqw || dkw) && (!ws || ws_bytes < 2 * part)) return SAS_ERR_WORKSPACE;
  if (p.T == 0) {
    if (dqw && cudaMemsetAsync(dqw, 0, p.D * 4, st) != cudaSuccess) return SAS_ERR_CUDA;
    if (dkw && cudaMemsetAsync(dkw, 0, p.D * 4, st) != cudaSuccess) return SAS_ERR_CUDA;
    return SAS_OK;
  }
  const int hw = 32 / lanes_of(p.D), nv = vectors_of(p.D);
  for (Rows* r : {&p.q, &p.k}) {
    if (!share_out(p.T, r, nullptr, hw, kBwdBlocks * kWarps, 4, &r->most)) return SAS_ERR_UNSUPPORTED;
    const int64_t fit = ((int64_t)p.T * r->chunks + kWarps - 1) / kWarps;
    r->blocks = (uint32_t)(fit < kBwdBlocks ? fit : kBwdBlocks);
  }
  p.q.dw_part = dqw ? static_cast<float*>(ws) : nullptr;
  p.k.dw_part = dkw ? reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + part) : nullptr;
  const bool inter = p.flags & SAS_ROPE_INTERLEAVED, hasw = dqw || dkw;
  int smem = kWarps * stages_of(nv) * (2 * nv * 512 + p.R * 4);
  if (hasw && smem < kWarps * hw * p.D * 4) smem = kWarps * hw * p.D * 4;
  int rc;
#define GO(DT)                                                                                                          \
  rc = inter ? (hasw ? launch_bwd<DT, true, true>(p, smem, st) : launch_bwd<DT, true, false>(p, smem, st))             \
             : (hasw ? launch_bwd<DT, false, true>(p, smem, st) : launch_bwd<DT, false, false>(p, smem, st))
  if (dtype == SAS_DTYPE_BF16) GO(SAS_DTYPE_BF16); else GO(SAS_DTYPE_FP16);
#undef GO
  if (rc != SAS_OK || !hasw) return rc;
  sum_partials_kernel<<<dim3((p.D + 31) / 32, 2), 256, 0, st>>>(p.q.dw_part, dqw, p.q.blocks, p.k.dw_part, dkw,
                                                                p.k.blocks, p.D);
  return cudaGetLastError() == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
}

}  // namespace

extern "C" {

int sas_head_norm_rope_fwd(const void* q, int64_t q_ts, int64_t q_hs, void* q_out, int64_t qo_ts, int64_t qo_hs,
                           int32_t H, const void* k, int64_t k_ts, int64_t k_hs, void* k_out, int64_t ko_ts,
                           int64_t ko_hs, int32_t Hk, int32_t T, int32_t D, int32_t dtype, const void* positions,
                           const float* cos, const float* sin, int32_t P, int32_t R, const float* q_weight,
                           const float* k_weight, float eps, int32_t flags, int32_t* status, void* stream) {
  RopeParams p = {};
  p.q = {static_cast<const uint8_t*>(q), q_ts, q_hs, static_cast<uint8_t*>(q_out), qo_ts, qo_hs, nullptr, 0, 0, q_weight, nullptr, H};
  p.k = {static_cast<const uint8_t*>(k), k_ts, k_hs, static_cast<uint8_t*>(k_out), ko_ts, ko_hs, nullptr, 0, 0, k_weight, nullptr, Hk};
  p.T = T, p.D = D, p.R = R, p.P = P, p.flags = flags, p.eps = eps;
  p.positions = positions, p.cos = cos, p.sin = sin, p.status = status;
  const int rc = check(p, dtype, false);
  if (rc != SAS_OK) return rc;
  if (!rows_ok(p.k, false)) return SAS_ERR_INVALID_ARG;
  if (!sas::select_device_of(q ? q : k)) return SAS_ERR_CUDA;
  return fwd(p, dtype, static_cast<cudaStream_t>(stream));
}

size_t sas_head_norm_rope_bwd_workspace_bytes(int32_t D) { return D > 0 ? 2 * (size_t)kBwdBlocks * D * 4 : 0; }

int sas_head_norm_rope_bwd(const void* dq_out, int64_t dqo_ts, int64_t dqo_hs, const void* q, int64_t q_ts,
                           int64_t q_hs, void* dq, int32_t H, const void* dk_out, int64_t dko_ts, int64_t dko_hs,
                           const void* k, int64_t k_ts, int64_t k_hs, void* dk, int32_t Hk, int32_t T, int32_t D,
                           int32_t dtype, const void* positions, const float* cos, const float* sin, int32_t P,
                           int32_t R, const float* q_weight, const float* k_weight, float* dq_weight,
                           float* dk_weight, float eps, int32_t flags, int32_t* status, void* workspace,
                           size_t workspace_bytes, void* stream) {
  RopeParams p = {};
  const int64_t ts = (int64_t)H * D, tsk = (int64_t)Hk * D;  // dq, dk are dense
  p.q = {static_cast<const uint8_t*>(q), q_ts, q_hs, static_cast<uint8_t*>(dq), ts, D, static_cast<const uint8_t*>(dq_out), dqo_ts, dqo_hs, q_weight, nullptr, H};
  p.k = {static_cast<const uint8_t*>(k), k_ts, k_hs, static_cast<uint8_t*>(dk), tsk, D, static_cast<const uint8_t*>(dk_out), dko_ts, dko_hs, k_weight, nullptr, Hk};
  p.T = T, p.D = D, p.R = R, p.P = P, p.flags = flags, p.eps = eps;
  p.positions = positions, p.cos = cos, p.sin = sin, p.status = status;
  const int rc = check(p, dtype, true);
  if (rc != SAS_OK) return rc;
  if (!rows_ok(p.k, true) || (H > 0 && !dq_out) || (Hk > 0 && !dk_out)) return SAS_ERR_INVALID_ARG;
  if (!sas::select_device_of(q ? q : k)) return SAS_ERR_CUDA;
  return bwd(p, dtype, dq_weight, dk_weight, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int sas_append_sharedkv(const void* kv, int64_t kv_ts, void* pool, int64_t nblk, int32_t bs, const int32_t* block_table,
                        int32_t bt_stride, const int32_t* cu_seqlens_q, const int32_t* seqused_kv, int32_t B, int32_t S,
                        int32_t layout, const void* q, int64_t q_ts, int64_t q_hs, void* q_out, int64_t qo_ts,
                        int64_t qo_hs, int32_t H, int32_t T, int32_t D, int32_t dtype, const void* positions,
                        const float* cos, const float* sin, int32_t P, int32_t R, const float* kv_weight,
                        const float* q_weight, float eps, int32_t flags, int32_t* status, void* stream) {
  RopeParams p = {};
  p.q = {static_cast<const uint8_t*>(q), q_ts, q_hs, static_cast<uint8_t*>(q_out), qo_ts, qo_hs, nullptr, 0, 0, q_weight, nullptr, H};
  p.k = {static_cast<const uint8_t*>(kv), kv_ts, 0, nullptr, 0, 0, nullptr, 0, 0, kv_weight, nullptr, 1};
  p.T = T, p.D = D, p.R = R, p.P = P, p.flags = flags, p.eps = eps;
  p.positions = positions, p.cos = cos, p.sin = sin, p.status = status;
  p.pool = static_cast<uint8_t*>(pool), p.nblk = nblk, p.bs = bs, p.bt = block_table, p.bt_stride = bt_stride;
  p.cu = cu_seqlens_q, p.seqused = seqused_kv, p.B = B, p.S = S, p.layout = layout;
  int rc = check(p, dtype, false);
  if (rc == SAS_OK) rc = check_paged(p);
  if (rc != SAS_OK) return rc;
  if (!kv || !aligned16(kv) || (kv_ts & 7) || (kv_weight && !aligned16(kv_weight))) return SAS_ERR_INVALID_ARG;
  if (!sas::select_device_of(kv)) return SAS_ERR_CUDA;
  return fwd(p, dtype, static_cast<cudaStream_t>(stream));
}

int sas_append_sharedkv_bwd(const void* d_pool, int64_t nblk, int32_t bs, const int32_t* block_table,
                            int32_t bt_stride, const int32_t* cu_seqlens_q, const int32_t* seqused_kv, int32_t B,
                            int32_t S, int32_t layout, const void* kv, int64_t kv_ts, void* dkv, int32_t T, int32_t D,
                            int32_t dtype, const void* positions, const float* cos, const float* sin, int32_t P,
                            int32_t R, const float* kv_weight, float* dkv_weight, float eps, int32_t flags,
                            int32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
  RopeParams p = {};
  p.k = {static_cast<const uint8_t*>(kv), kv_ts, 0, static_cast<uint8_t*>(dkv), D, 0, nullptr, 0, 0, kv_weight, nullptr, 1};
  p.T = T, p.D = D, p.R = R, p.P = P, p.flags = flags, p.eps = eps;
  p.positions = positions, p.cos = cos, p.sin = sin, p.status = status;
  p.pool = const_cast<uint8_t*>(static_cast<const uint8_t*>(d_pool));  // read only here
  p.nblk = nblk, p.bs = bs, p.bt = block_table, p.bt_stride = bt_stride;
  p.cu = cu_seqlens_q, p.seqused = seqused_kv, p.B = B, p.S = S, p.layout = layout;
  int rc = check(p, dtype, true);
  if (rc == SAS_OK) rc = check_paged(p);
  if (rc != SAS_OK) return rc;
  if (!rows_ok(p.k, true)) return SAS_ERR_INVALID_ARG;
  if (!sas::select_device_of(kv)) return SAS_ERR_CUDA;
  return bwd(p, dtype, nullptr, dkv_weight, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
