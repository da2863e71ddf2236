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
// Everything here is bound by memory: 4 bytes per value forward (read and
// written once in 16 bits), 6 backward, for 5-12 operations. A row of D values
// lies with G lanes of a warp (8 values = 16 bytes per lane and vector), so
// the sums are a few shuffles and the rotation stays inside a lane (INTER) or
// takes one more load that hits L1 (halves). A warp takes U heads of ONE token, so the
// position, the table rows and the slot lookup are fetched once for them, and
// all U rows' loads are in flight before the first is used.
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
  int H, chunks, blocks;  // chunks: warps' shares of a token's heads
};

struct RopeParams {
  Rows q, k;
  int T, D, R, P, flags;
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

__device__ __forceinline__ uint4 ldg_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <int DT>
__device__ __forceinline__ void unpack8(const uint4& r, float (&f)[8]) {
  const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 v;
    if (DT == SAS_DTYPE_BF16) {
      v = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162&>(u[i]));
    } else {
      v = __half22float2(reinterpret_cast<const __half2&>(u[i]));
    }
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (DT == SAS_DTYPE_BF16) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      u[i] = reinterpret_cast<const uint32_t&>(v);
    } else {
      const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
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

// Request of token t, its cache slot and the pool row of that slot (-1: no
// row; the column past the table's width or an entry past the pool is also
// recorded). Every lane of the warp calls it. TND: a 32-way search of
// cu_seqlens_q, two rounds up to 1024 requests.
__device__ __forceinline__ int64_t slot_row(const RopeParams& p, int t, int lane, int& slot, bool want_row) {
  int b, i, n;
  if (p.layout == SAS_LAYOUT_TND) {
    int lo = 0, len = p.B;  // the last b in [lo, lo + len) with cu[b] <= t
    while (len > 1) {
      const int step = (len + 31) >> 5;
      const int c = lo + lane * step;
      const bool le = c < lo + len && __ldg(p.cu + c) <= t;
      const int last = 31 - __clz(__ballot_sync(0xffffffffu, le) | 1u);
      const int at = lo + last * step;
      len = min(step, lo + len - at);
      lo = at;
    }
    b = lo;
    const int c0 = __ldg(p.cu + b);
    i = t - c0;
    n = __ldg(p.cu + b + 1) - c0;
  } else {
    b = t / p.S;
    i = t - b * p.S;
    n = p.cu ? __ldg(p.cu + b + 1) - __ldg(p.cu + b) : p.S;
  }
  slot = -1;
  if (i < 0 || i >= n) return -1;  // BSND padding, or a token past cu_seqlens_q's end
  slot = __ldg(p.seqused + b) - n + i;
  if (!want_row || slot < 0) return -1;
  const int col = slot / p.bs;
  if (col >= p.bt_stride) {
    if (lane == 0 && p.status) atomicCAS(p.status, 0, SAS_ERR_BAD_BLOCK_ENTRY);
    return -1;
  }
  const int blk = __ldg(p.bt + (int64_t)b * p.bt_stride + col);
  if (blk < 0) return -1;
  if (blk >= p.nblk) {
    if (lane == 0 && p.status) atomicCAS(p.status, 0, SAS_ERR_BAD_BLOCK_ENTRY);
    return -1;
  }
  return (int64_t)blk * p.bs + (slot - col * p.bs);
}

// Row of the cos / sin tables of token t. A position outside the tables takes
// the nearest row and is recorded.
__device__ __forceinline__ int table_row(const RopeParams& p, int t, int slot, int lane) {
  int64_t pos = slot;
  if (p.positions)
    pos = (p.flags & SAS_ROPE_POS64) ? __ldg(static_cast<const long long*>(p.positions) + t)
                               : __ldg(static_cast<const int32_t*>(p.positions) + t);
  else if (slot < 0)
    return 0;  // a token without a slot: nothing of it is written to the cache
  if (pos < 0 || pos >= p.P) {
    if (lane == 0 && p.status) atomicCAS(p.status, 0, SAS_ERR_BAD_POSITION);
    pos = pos < 0 ? 0 : p.P - 1;
  }
  return (int)pos;
}

// a * b - c * d to about an ulp of the result however much cancels (Kahan's
// difference of products): turned values keep their relative accuracy, which
// the weight's gradient is a product of. Two more FMAs on rotated dims.
__device__ __forceinline__ float diff_of_products(float a, float b, float c, float d) {
  const float cd = c * d;
  return fmaf(a, b, -cd) + fmaf(-c, d, cd);
}

// cos and sin of vector v's 4 (INTER) or 8 (halves) angles; `first` tells the
// lower half. Returns false for a vector that is not rotated.
template <bool INTER>
struct Angles {
  float c[INTER ? 4 : 8], s[INTER ? 4 : 8];
  bool on, first;
  __device__ __forceinline__ void load(const RopeParams& p, int v, int row) {
    const int e = v * 8 - (p.D - p.R);
    on = e >= 0 && v * 8 < p.D;
    first = e < p.R / 2;
    if (!on) return;
    const int a = INTER ? e / 2 : (first ? e : e - p.R / 2);
    const float* pc = p.cos + (int64_t)row * (p.R / 2) + a;
    const float* ps = p.sin + (int64_t)row * (p.R / 2) + a;
#pragma unroll
    for (int i = 0; i < (INTER ? 4 : 8); i += 4) {
      const float4 a4 = __ldg(reinterpret_cast<const float4*>(pc + i));
      const float4 b4 = __ldg(reinterpret_cast<const float4*>(ps + i));
      c[i] = a4.x, c[i + 1] = a4.y, c[i + 2] = a4.z, c[i + 3] = a4.w;
      s[i] = b4.x, s[i + 1] = b4.y, s[i + 2] = b4.z, s[i + 3] = b4.w;
    }
  }
  // f rotated by sgn times the angle; `o`: the partner vector's values (halves only)
  __device__ __forceinline__ void turn(float (&f)[8], const float (&o)[8], float sgn) const {
    if (INTER) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = f[2 * i], b = f[2 * i + 1], sn = sgn * s[i];
        f[2 * i] = diff_of_products(a, c[i], b, sn);
        f[2 * i + 1] = diff_of_products(b, c[i], -a, sn);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float sn = sgn * s[i % (INTER ? 4 : 8)];
        f[i] = diff_of_products(f[i], c[i % (INTER ? 4 : 8)], o[i], first ? sn : -sn);
      }
    }
  }
};

__device__ __forceinline__ void weight8(const float* w, int v, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(w + v * 8));
  const float4 b = __ldg(reinterpret_cast<const float4*>(w + v * 8 + 4));
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

constexpr int kWarps = 8;

// DT: type; G lanes hold a row, NV vectors of 8 values each; U: rows in flight per group of lanes.
template <int DT, int G, int NV, int U, bool INTER>
__global__ void __launch_bounds__(32 * kWarps) rope_fwd_kernel(const __grid_constant__ RopeParams p) {
  constexpr int HW = 32 / G;  // heads side by side in a warp
  const int lane = threadIdx.x & 31;
  const uint32_t cpt = p.q.chunks + p.k.chunks;
  const uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const uint32_t t = unit / cpt;
  if (t >= (uint32_t)p.T) return;
  int c = (int)(unit - t * cpt);
  const bool isk = c >= p.q.chunks;
  const Rows& rs = isk ? p.k : p.q;
  if (isk) c -= p.q.chunks;
  const int h0 = c * (U * HW) + lane / G, gl = lane % G;
  const int V = p.D >> 3;

  uint4 raw[U][NV];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * HW;
    const uint8_t* xr = rs.x + ((int64_t)t * rs.x_ts + (int64_t)h * rs.x_hs) * 2;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = gl + G * j;
      raw[u][j] = h < rs.H && v < V ? ldg_stream(xr + v * 16) : make_uint4(0, 0, 0, 0);
    }
  }
  const bool append = p.pool != nullptr;
  int slot = -1;
  int64_t row = -1;
  if (append && (isk || !p.positions)) row = slot_row(p, t, lane, slot, isk);
  Angles<INTER> an[NV];
  if (p.R > 0) {
    const int tr = table_row(p, t, slot, lane);
#pragma unroll
    for (int j = 0; j < NV; ++j) an[j].load(p, gl + G * j, tr);
  }
  const float sgn = (p.flags & SAS_ROPE_INVERSE) ? -1.f : 1.f;
  const float invD = 1.f / (float)p.D;
  uint8_t* yt = nullptr;
  if (append && isk) {
    if (row < 0) return;
    yt = p.pool + row * p.D * 2;
  } else {
    yt = rs.y + (int64_t)t * rs.y_ts * 2;
  }
  float rstd[U];
  if (p.flags & SAS_ROPE_NORM) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float f[8];
        unpack8<DT>(raw[u][j], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
      }
      rstd[u] = ss;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) rstd[u] = rsqrtf(group_sum<G>(rstd[u]) * invD + p.eps);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) rstd[u] = 1.f;
  }
  // halves: the partner vectors, read before any lane of the warp writes (y may be x)
  uint4 part[INTER ? 1 : U][INTER ? 1 : NV];
  if (!INTER) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * HW;
      const uint8_t* xr = rs.x + ((int64_t)t * rs.x_ts + (int64_t)h * rs.x_hs) * 2;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int v = gl + G * j + (an[j].first ? p.R / 16 : -(p.R / 16));
        part[INTER ? 0 : u][INTER ? 0 : j] =
            p.R > 0 && an[j].on && h < rs.H ? *reinterpret_cast<const uint4*>(xr + v * 16) : make_uint4(0, 0, 0, 0);
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = gl + G * j;
    if (v >= V) continue;
    const bool turn = p.R > 0 && an[j].on;
    const int pv = v + (an[j].first ? p.R / 16 : -(p.R / 16));
    float w[8], wp[8];
    if (rs.w) {
      weight8(rs.w, v, w);
      if (!INTER && turn) weight8(rs.w, pv, wp);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * HW;
      if (h >= rs.H) continue;
      float f[8], o[8];
      unpack8<DT>(raw[u][j], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= rstd[u];
      if (rs.w)
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= w[i];
      if (turn) {
        if (!INTER) {
          unpack8<DT>(part[INTER ? 0 : u][INTER ? 0 : j], o);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] *= rstd[u];
          if (rs.w)
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] *= wp[i];
        }
        an[j].turn(f, o, sgn);
      }
      *reinterpret_cast<uint4*>(yt + ((int64_t)h * rs.y_hs + v * 8) * 2) = pack8<DT>(f);
    }
  }
}

// Backward. Blocks [0, q.blocks) take the q rows, the rest the k rows; a warp
// walks tokens' head shares with the stride of its set's warps, and keeps the
// weight gradient of its columns in registers. Each block adds its warps'
// sums in order and writes one row of partials; sum_partials_kernel adds the
// rows in order, so the result does not depend on timing.
template <int DT, int G, int NV, int U, bool INTER, bool HASW>
__global__ void __launch_bounds__(32 * kWarps) rope_bwd_kernel(const __grid_constant__ RopeParams p) {
  constexpr int HW = 32 / G;
  extern __shared__ float red[];  // [kWarps * HW][D] (HASW)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool isk = (int)blockIdx.x >= p.q.blocks;
  const Rows& rs = isk ? p.k : p.q;
  const int blk = isk ? blockIdx.x - p.q.blocks : blockIdx.x;
  const int gl = lane % G, V = p.D >> 3;
  const bool append = p.pool != nullptr;
  const bool norm = p.flags & SAS_ROPE_NORM;
  const float sgn = (p.flags & SAS_ROPE_INVERSE) ? 1.f : -1.f;  // the transpose turns back
  const float invD = 1.f / (float)p.D;
  float acc[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[j][i] = 0.f;
  const uint32_t units = (uint32_t)p.T * (uint32_t)rs.chunks;
  for (uint32_t unit = blk * kWarps + warp; unit < units; unit += rs.blocks * kWarps) {
    const uint32_t t = unit / rs.chunks;
    const int h0 = (int)(unit - t * rs.chunks) * (U * HW) + lane / G;
    uint4 xr[U][NV], dr[U][NV];
    int slot = -1;
    int64_t row = -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * HW;
      const uint8_t* xp = rs.x + ((int64_t)t * rs.x_ts + (int64_t)h * rs.x_hs) * 2;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int v = gl + G * j;
        xr[u][j] = h < rs.H && v < V ? ldg_stream(xp + v * 16) : make_uint4(0, 0, 0, 0);
      }
    }
    if (append) row = slot_row(p, t, lane, slot, true);
    const uint8_t* db = append ? p.pool + (row < 0 ? 0 : row) * p.D * 2 : rs.dy + (int64_t)t * rs.dy_ts * 2;
    const bool have = !append || row >= 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * HW;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int v = gl + G * j;
        dr[u][j] = have && h < rs.H && v < V ? *reinterpret_cast<const uint4*>(db + ((int64_t)h * rs.dy_hs + v * 8) * 2)
                                             : make_uint4(0, 0, 0, 0);
      }
    }
    Angles<INTER> an[NV];
    if (p.R > 0) {
      const int tr = table_row(p, t, slot, lane);
#pragma unroll
      for (int j = 0; j < NV; ++j) an[j].load(p, gl + G * j, tr);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * HW;
      float ss = 0.f, gx = 0.f;
      float g[NV][8];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int v = gl + G * j;
        float x[8], o[8], w[8];
        unpack8<DT>(xr[u][j], x);
        unpack8<DT>(dr[u][j], g[j]);
        if (p.R > 0 && an[j].on) {
          if (!INTER) {
            const int pv = v + (an[j].first ? p.R / 16 : -(p.R / 16));
            const uint4 pr = have && h < rs.H
                                 ? *reinterpret_cast<const uint4*>(db + ((int64_t)h * rs.dy_hs + pv * 8) * 2)
                                 : make_uint4(0, 0, 0, 0);
            unpack8<DT>(pr, o);
          }
          an[j].turn(g[j], o, sgn);
        }
        if (v >= V) continue;
        if (rs.w) weight8(rs.w, v, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss = fmaf(x[i], x[i], ss);
          gx = fmaf(rs.w ? g[j][i] * w[i] : g[j][i], x[i], gx);
        }
      }
      float rstd = 1.f, mean = 0.f;
      if (norm) {
        ss = group_sum<G>(ss);
        gx = group_sum<G>(gx);
        rstd = rsqrtf(ss * invD + p.eps);
        mean = rstd * gx * invD;  // of g * xhat
      }
      uint8_t* yp = rs.y + ((int64_t)t * rs.y_ts + (int64_t)h * rs.y_hs) * 2;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int v = gl + G * j;
        if (v >= V) continue;
        float x[8], w[8], o[8];
        unpack8<DT>(xr[u][j], x);
        if (rs.w) weight8(rs.w, v, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float xh = x[i] * rstd;
          if (HASW) acc[j][i] = fmaf(g[j][i], xh, acc[j][i]);
          o[i] = rstd * ((rs.w ? g[j][i] * w[i] : g[j][i]) - xh * mean);
        }
        if (h < rs.H) *reinterpret_cast<uint4*>(yp + v * 16) = pack8<DT>(o);
      }
    }
  }
  if (HASW && rs.dw_part) {
    float* mine = red + (warp * HW + lane / G) * p.D;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = gl + G * j;
      if (v < V)
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[v * 8 + i] = acc[j][i];
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
int lanes_of(int D) { return D <= 64 ? 8 : (D <= 128 ? 16 : 32); }

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

#define ROPE_SHAPES(F)                       \
  if (g == 8) F(8, 1)                        \
  else if (g == 16) F(16, 1)                 \
  else if (nv == 1) F(32, 1)                 \
  else if (nv == 2) F(32, 2)                 \
  else F(32, 4)

template <int DT, int U, bool INTER>
void launch_fwd(const RopeParams& p, int blocks, cudaStream_t st) {
  const int g = lanes_of(p.D), nv = (p.D / 8 + g - 1) / g;
#define F(G, NV) rope_fwd_kernel<DT, G, NV, U, INTER><<<blocks, 32 * kWarps, 0, st>>>(p);
  ROPE_SHAPES(F)
#undef F
}

// Rows in flight per lane group: 4 once the call has enough warps to fill the
// GPU that way, else 1, so that a decode step's few rows spread over all SMs.
int fwd(RopeParams& p, int dtype, cudaStream_t st) {
  if (p.T == 0) return SAS_OK;
  const int hw = 32 / lanes_of(p.D);
  const int64_t rows = (int64_t)p.T * ((p.q.H + hw - 1) / hw);
  const int U = rows >= 148 * 64 * 4 ? 4 : 1;
  p.q.chunks = (p.q.H + U * hw - 1) / (U * hw);
  p.k.chunks = (p.k.H + U * hw - 1) / (U * hw);
  const int64_t blocks = ((int64_t)p.T * (p.q.chunks + p.k.chunks) + kWarps - 1) / kWarps;
  if (blocks * kWarps >= (1ll << 31)) return SAS_ERR_UNSUPPORTED;
  const bool inter = p.flags & SAS_ROPE_INTERLEAVED;
#define GO(DT, U_)                                       \
  (inter ? launch_fwd<DT, U_, true>(p, (int)blocks, st)  \
         : launch_fwd<DT, U_, false>(p, (int)blocks, st))
  if (dtype == SAS_DTYPE_BF16) {
    if (U == 4) GO(SAS_DTYPE_BF16, 4); else GO(SAS_DTYPE_BF16, 1);
  } else {
    if (U == 4) GO(SAS_DTYPE_FP16, 4); else GO(SAS_DTYPE_FP16, 1);
  }
#undef GO
  return cudaGetLastError() == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
}

constexpr int kBwdBlocks = 148 * 4;  // most blocks of a set of rows; its partials are one row of D floats per block

template <int DT, bool INTER, bool HASW>
int launch_bwd(const RopeParams& p, cudaStream_t st) {
  const int g = lanes_of(p.D), nv = (p.D / 8 + g - 1) / g;
  const size_t smem = HASW ? (size_t)kWarps * (32 / g) * p.D * 4 : 0;  // at most 32 KB
#define F(G, NV) rope_bwd_kernel<DT, G, NV, 1, INTER, HASW><<<p.q.blocks + p.k.blocks, 32 * kWarps, smem, st>>>(p);
  ROPE_SHAPES(F)
#undef F
  return cudaGetLastError() == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
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
  const int hw = 32 / lanes_of(p.D);
  for (Rows* r : {&p.q, &p.k}) {
    r->chunks = (r->H + hw - 1) / hw;
    const int64_t units = (int64_t)p.T * r->chunks;
    if (units >= (1ll << 31) - kBwdBlocks * kWarps) return SAS_ERR_UNSUPPORTED;
    r->blocks = (int)((units + kWarps - 1) / kWarps < kBwdBlocks ? (units + kWarps - 1) / kWarps : kBwdBlocks);
  }
  p.q.dw_part = dqw ? static_cast<float*>(ws) : nullptr;
  p.k.dw_part = dkw ? reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + part) : nullptr;
  const bool inter = p.flags & SAS_ROPE_INTERLEAVED, hasw = dqw || dkw;
  int rc;
#define GO(DT)                                                                                              \
  rc = inter ? (hasw ? launch_bwd<DT, true, true>(p, st) : launch_bwd<DT, true, false>(p, st))             \
             : (hasw ? launch_bwd<DT, false, true>(p, st) : launch_bwd<DT, false, false>(p, st))
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
  p.q = {static_cast<const uint8_t*>(q), q_ts, q_hs, static_cast<uint8_t*>(q_out), qo_ts, qo_hs, nullptr, 0, 0, q_weight, nullptr, H, 0, 0};
  p.k = {static_cast<const uint8_t*>(k), k_ts, k_hs, static_cast<uint8_t*>(k_out), ko_ts, ko_hs, nullptr, 0, 0, k_weight, nullptr, Hk, 0, 0};
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
  p.q = {static_cast<const uint8_t*>(q), q_ts, q_hs, static_cast<uint8_t*>(dq), ts, D, static_cast<const uint8_t*>(dq_out), dqo_ts, dqo_hs, q_weight, nullptr, H, 0, 0};
  p.k = {static_cast<const uint8_t*>(k), k_ts, k_hs, static_cast<uint8_t*>(dk), tsk, D, static_cast<const uint8_t*>(dk_out), dko_ts, dko_hs, k_weight, nullptr, Hk, 0, 0};
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
  p.q = {static_cast<const uint8_t*>(q), q_ts, q_hs, static_cast<uint8_t*>(q_out), qo_ts, qo_hs, nullptr, 0, 0, q_weight, nullptr, H, 0, 0};
  p.k = {static_cast<const uint8_t*>(kv), kv_ts, 0, nullptr, 0, 0, nullptr, 0, 0, kv_weight, nullptr, 1, 0, 0};
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
  p.k = {static_cast<const uint8_t*>(kv), kv_ts, 0, static_cast<uint8_t*>(dkv), D, 0, nullptr, 0, 0, kv_weight, nullptr, 1, 0, 0};
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
