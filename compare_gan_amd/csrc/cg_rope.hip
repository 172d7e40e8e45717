// Rotary positions, and the RMS norm of every head of the queries and keys with the rotation in the
// same pass (forward and backward).
//
//   angle(t, i) = positions[t, axis(i)] * 2 pi freq[i]          i = pair of the turned part
//   y_a = A (a cos - b sin),  y_b = A (a sin + b cos)           A = amplitude; entries >= rot are copied
//   norm:  a, b <- x * rsqrt(mean_d x^2 + eps) * gain_d          in front of the rotation
//   backward (the rotation is orthogonal up to A, so its adjoint turns by -angle):
//     g = R^T dy,  dgain_d = sum g xhat,  g <- g gain,  dx = inv (g - xhat mean_d(g xhat))
//
// Both are bound by HBM: every element is read once and written once (backward: two reads, one
// write), about 3 / 6 / 10 flops an element.  What the layout has to avoid is (a) the angles costing
// more than the data and (b) short loads.  (a) A block takes tb tokens; the cosine and sine of each
// (token, pair) are formed once, by one thread, kept in LDS and read by all heads of q and k.  The
// product position * frequency is taken in 64 bits in TURNS and reduced there (a fp32 angle at position
// 10^5 is off by 10^-2 rad), the rest in 32.  (b) A row (one head of one token) belongs to a group of
// `lanes` lanes, each with VP pairs = 2 VP elements in two loads of VP: 16 bytes each where sizes and
// alignment allow it.  The head's sum of squares is a butterfly over the group.
//
// Measured (a copy of 1 GiB: 5.0 TB/s read and written; of 128 MiB, which stays in the last-level cache, 7.1):
//   rotation, 262 144 tokens x 3 heads of 64, bf16, 201 MB:   42 us between other work, 33 us behind itself (6.1 TB/s)
//   rotation, fp32, 30 011 tokens x 5 heads of 80, 96 MB:     19 us (5 TB/s)
//   norm + rotation, 65 536 x (32 + 8) heads of 128, 1.34 GB: 254 to 280 us (4.8 to 5.3 TB/s)
//   its forward / backward, 65 536 x (6 + 6) heads of 32:     20 / 33 us (101 / 151 MB), gains behind it 6 us
//   forward / backward, 65 536 x (8 + 2) heads of 128, fp32:  142 / 217 us (671 MB / 1.0 GB, 4.7 / 4.6 TB/s)
// A call of a few tokens is 3 to 6 us, what a launch and one trip to memory take.  A row's lanes are a power of two:
// 72 wide heads leave 7 of 16 lanes without data (30 011 x (8 + 4) heads: 34 / 57 us, 3.1 / 2.7 TB/s; 64 wide ones 19 /
// 37 us, 4.8 / 3.8 TB/s).
#include "cg_common.h"

namespace {

struct RopeTensor {
  const void* x;     // [T, heads, D], strides in elements
  const void* dy;    // backward: gradient of the output, contiguous
  void* out;         // contiguous
  const float* gain; // [D] or null
  int64_t st, sh;
  int heads;
  FastDiv dheads;
};
struct RopeArgs {
  RopeTensor t[2];   // q (or the one tensor), k
  int ntensors;
  const int32_t* positions;
  const double* freq;
  float* partial;    // [blocks][2][D] gain gradients
  float amplitude, eps, inv_d, sign;
  int T, D, rot, pairs, slots, per_axis, axes, interleaved;   // slots: pairs of whole units
  int tb, lanes, lanes_log, units, pair_units, chunks;
  FastDiv dslots, dper;
};

template <typename T, int VP>
__device__ __forceinline__ void load_vp(const T* p, float* v) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (VP == 8) {
      unpack8_bf16(*reinterpret_cast<const uint4*>(p), v);
    } else if constexpr (VP == 4) {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      v[0] = __uint_as_float(q.x << 16); v[1] = __uint_as_float(q.x & 0xffff0000u);
      v[2] = __uint_as_float(q.y << 16); v[3] = __uint_as_float(q.y & 0xffff0000u);
    } else if constexpr (VP == 2) {
      const uint32_t q = *reinterpret_cast<const uint32_t*>(p);
      v[0] = __uint_as_float(q << 16); v[1] = __uint_as_float(q & 0xffff0000u);
    } else {
      v[0] = bf2f(*p);
    }
  } else {
    if constexpr (VP >= 4) {
#pragma unroll
      for (int j = 0; j < VP; j += 4) {
        const float4 q = *reinterpret_cast<const float4*>(p + j);
        v[j] = q.x; v[j + 1] = q.y; v[j + 2] = q.z; v[j + 3] = q.w;
      }
    } else if constexpr (VP == 2) {
      const float2 q = *reinterpret_cast<const float2*>(p);
      v[0] = q.x; v[1] = q.y;
    } else {
      v[0] = *p;
    }
  }
}
template <typename T, int VP>
__device__ __forceinline__ void store_vp(T* p, const float* v) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (VP == 8) *reinterpret_cast<uint4*>(p) = pack8_bf16(v);
    else if constexpr (VP == 4) *reinterpret_cast<uint2*>(p) = pack4_bf16(v);
    else if constexpr (VP == 2)
      *reinterpret_cast<uint32_t*>(p) = (uint32_t)f2bf(v[0]) | ((uint32_t)f2bf(v[1]) << 16);
    else *p = f2bf(v[0]);
  } else {
    if constexpr (VP >= 4) {
#pragma unroll
      for (int j = 0; j < VP; j += 4)
        *reinterpret_cast<float4*>(p + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else if constexpr (VP == 2) {
      *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    } else {
      *p = v[0];
    }
  }
}

// cosine and sine of `turns` in [-1/2, 1/2].  bf16 data: the hardware functions (v_sin_f32 / v_cos_f32
// take turns; their error of about 2^-20 is far below bf16's half step, up to 2^-8 of the value); fp32
// data: the library's, good to the last bits.
template <typename T>
__device__ __forceinline__ float2 turn_cos_sin(float turns) {
  if constexpr (sizeof(T) == 2) {
    return make_float2(__builtin_amdgcn_cosf(turns), __builtin_amdgcn_sinf(turns));
  } else {
    float s, c;
    sincospif(2.f * turns, &s, &c);
    return make_float2(c, s);
  }
}

// 16 KiB: cosines and sines, then the gain partials (rows of a block x D <= 256 lanes x 16 elements); eight blocks a
// CU, so that the angles of one are formed while others move data
constexpr int ROPE_LDS_FLOATS = 4096;

// UPL: units (2 VP elements) a lane holds.  PART: the last pairs of a unit are copied entries, which stay as they are
// (turned by the identity, 0 times an infinite neighbour would be NaN); a form of its own, since choosing costs every
// unit of the others something: 262 144 tokens x 3 heads of 64, 36 us in place of 33 behind itself
template <typename T, int VP, int UPL, bool NORM, bool BWD, bool PART>
__global__ __launch_bounds__(256, NORM && VP == 8 ? 3 : BWD ? 4 : 6) void rope_kernel(RopeArgs a) {
  __shared__ __attribute__((aligned(16))) float lds[ROPE_LDS_FLOATS];
  float2* cs = reinterpret_cast<float2*>(lds);
  constexpr int E = 2 * VP * UPL;
  const int lane_r = threadIdx.x & (a.lanes - 1), row_in_block = threadIdx.x >> a.lanes_log;
  const int rows_step = 256 >> a.lanes_log;
  float acc[2][E];
  if constexpr (BWD) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[s][e] = 0.f;
  }
  // offsets of this lane's pieces within a head
  int off_a[UPL], off_b[UPL], cs_at[UPL];
  bool live[UPL], pair_unit[UPL];
#pragma unroll
  for (int u = 0; u < UPL; ++u) {
    const int unit = lane_r + u * a.lanes;
    live[u] = unit < a.units;
    pair_unit[u] = unit < a.pair_units;
    cs_at[u] = unit * VP;
    if (pair_unit[u] && !a.interleaved) {
      off_a[u] = unit * VP;
      off_b[u] = a.rot / 2 + unit * VP;
    } else {       // interleaved pairs and the copied rest: 2 VP consecutive elements
      off_a[u] = unit * 2 * VP;
      off_b[u] = off_a[u] + VP;
    }
  }
  for (int chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    const int t0 = chunk * a.tb;
    const int nt = min(a.tb, a.T - t0);
    __syncthreads();      // the previous chunk's angles are no longer read
    for (int i = threadIdx.x; i < nt * a.slots; i += 256) {
      const int tok = fdiv(i, a.dslots), pair = i - tok * a.slots;
      if (PART && pair >= a.pairs) continue;        // (read below and not used)
      const int axis = fdiv(pair, a.dper);
      const double turns = (double)a.positions[(int64_t)(t0 + tok) * a.axes + axis] * a.freq[pair];
      const float2 v = turn_cos_sin<T>((float)(turns - rint(turns)));
      cs[i] = make_float2(v.x * a.amplitude, v.y * a.amplitude * a.sign);
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s >= a.ntensors) break;
      const RopeTensor& ten = a.t[s];
      float gain[E];
      if constexpr (NORM) {
#pragma unroll
        for (int u = 0; u < UPL; ++u)
#pragma unroll
          for (int j = 0; j < VP; ++j) {
            gain[u * 2 * VP + j] = (live[u] && ten.gain) ? ten.gain[off_a[u] +
                (pair_unit[u] && a.interleaved ? 2 * j : j)] : 1.f;
            gain[u * 2 * VP + VP + j] = (live[u] && ten.gain) ? ten.gain[
                (pair_unit[u] && a.interleaved) ? off_a[u] + 2 * j + 1 : off_b[u] + j] : 1.f;
          }
      }
      const int nrows = nt * ten.heads;
      for (int row = row_in_block; row < nrows; row += rows_step) {
        const int tok = fdiv(row, ten.dheads), h = row - tok * ten.heads;
        const T* x = reinterpret_cast<const T*>(ten.x) + (int64_t)(t0 + tok) * ten.st + (int64_t)h * ten.sh;
        const int64_t dense = ((int64_t)(t0 + tok) * ten.heads + h) * a.D;
        // v[0 .. VP): first of the pairs, v[VP .. 2 VP): second (the copied rest: in order)
        float v[E], g[BWD ? E : 1];
        auto fetch = [&](const T* p, float* dst) {
#pragma unroll
          for (int u = 0; u < UPL; ++u) {
            float lo[VP], hi[VP];
#pragma unroll
            for (int j = 0; j < VP; ++j) lo[j] = hi[j] = 0.f;
            if (live[u]) {
              load_vp<T, VP>(p + off_a[u], lo);
              load_vp<T, VP>(p + off_b[u], hi);
            }
            if (VP > 1 && pair_unit[u] && a.interleaved) {
#pragma unroll
              for (int j = 0; j < VP; ++j) {
                const int k0 = 2 * j, k1 = 2 * j + 1;
                dst[u * 2 * VP + j] = k0 < VP ? lo[k0 % VP] : hi[k0 % VP];
                dst[u * 2 * VP + VP + j] = k1 < VP ? lo[k1 % VP] : hi[k1 % VP];
              }
            } else {
#pragma unroll
              for (int j = 0; j < VP; ++j) {
                dst[u * 2 * VP + j] = lo[j];
                dst[u * 2 * VP + VP + j] = hi[j];
              }
            }
          }
        };
        auto turn = [&](float* w) {
#pragma unroll
          for (int u = 0; u < UPL; ++u) {
            if (!pair_unit[u]) continue;
            const float2* c = cs + tok * a.slots + cs_at[u];
#pragma unroll
            for (int j = 0; j < VP; ++j) {
              const float2 q = c[j];
              const float p0 = w[u * 2 * VP + j], p1 = w[u * 2 * VP + VP + j];
              const bool in = !PART || cs_at[u] + j < a.pairs;
              w[u * 2 * VP + j] = in ? p0 * q.x - p1 * q.y : p0;
              w[u * 2 * VP + VP + j] = in ? p0 * q.y + p1 * q.x : p1;
            }
          }
        };
        fetch(x, v);
        if constexpr (BWD) fetch(reinterpret_cast<const T*>(ten.dy) + dense, g);
        float inv = 0.f;
        if constexpr (NORM) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) ss += v[e] * v[e];
          for (int o = a.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
          inv = 1.f / sqrtf(ss * a.inv_d + a.eps);
        }
        if constexpr (BWD) {
          turn(g);
          float dot = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float unit = v[e] * inv;
            acc[s][e] += g[e] * unit;
            g[e] *= gain[e];
            dot += g[e] * unit;
            v[e] = unit;
          }
          for (int o = a.lanes >> 1; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
          dot *= a.inv_d;
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = inv * (g[e] - v[e] * dot);
        } else {
          if constexpr (NORM) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = v[e] * inv * gain[e];
          }
          turn(v);
        }
        T* y = reinterpret_cast<T*>(ten.out) + dense;
#pragma unroll
        for (int u = 0; u < UPL; ++u) {
          if (!live[u]) continue;
          float lo[VP], hi[VP];
          if (VP > 1 && pair_unit[u] && a.interleaved) {
#pragma unroll
            for (int j = 0; j < VP; ++j) {
              const int k0 = j, k1 = VP + j;
              lo[j] = (k0 & 1) ? v[u * 2 * VP + VP + k0 / 2] : v[u * 2 * VP + k0 / 2];
              hi[j] = (k1 & 1) ? v[u * 2 * VP + VP + k1 / 2] : v[u * 2 * VP + k1 / 2];
            }
          } else {
#pragma unroll
            for (int j = 0; j < VP; ++j) {
              lo[j] = v[u * 2 * VP + j];
              hi[j] = v[u * 2 * VP + VP + j];
            }
          }
          store_vp<T, VP>(y + off_a[u], lo);
          store_vp<T, VP>(y + off_b[u], hi);
        }
      }
    }
  }
  if constexpr (BWD) {
    // rows of the block summed in a fixed order, one partial a block
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s >= a.ntensors) break;
      __syncthreads();
#pragma unroll
      for (int u = 0; u < UPL; ++u) {
        if (!live[u]) continue;
#pragma unroll
        for (int j = 0; j < VP; ++j) {
          const bool il = pair_unit[u] && a.interleaved;
          lds[row_in_block * a.D + (il ? off_a[u] + 2 * j : off_a[u] + j)] = acc[s][u * 2 * VP + j];
          lds[row_in_block * a.D + (il ? off_a[u] + 2 * j + 1 : off_b[u] + j)] = acc[s][u * 2 * VP + VP + j];
        }
      }
      __syncthreads();
      for (int d = threadIdx.x; d < a.D; d += 256) {
        float sum = 0.f;
        for (int r = 0; r < rows_step; ++r) sum += lds[r * a.D + d];
        a.partial[((int64_t)blockIdx.x * 2 + s) * a.D + d] = sum;
      }
    }
  }
}

// dgain[s][d] = sum over blocks of partial[block][s][d]; 16 columns a workgroup, 64 rows of threads, four loads in
// flight each
__global__ __launch_bounds__(1024) void rope_gain_kernel(const float* __restrict__ partial, int blocks, int D,
                                                         float* __restrict__ dq, float* __restrict__ dk) {
  __shared__ float lds[64][17];
  const int c = threadIdx.x & 15, col = blockIdx.x * 16 + c, part = threadIdx.x >> 4;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (col < 2 * D)
    for (int b = part; b < blocks; b += 256) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (b + 64 * j < blocks) sum[j] += partial[(int64_t)(b + 64 * j) * 2 * D + col];
    }
  lds[part][c] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  __syncthreads();
  if (part == 0 && col < 2 * D) {
    float all = 0.f;
    for (int p = 0; p < 64; ++p) all += lds[p][c];
    float* out = col < D ? dq : dk;
    if (out) out[col < D ? col : col - D] = all;
  }
}

constexpr int ROPE_MAX_BLOCKS_BWD = 1024;   // gain partials: blocks x 2 x D floats of workspace

bool aligned_for(const void* p, int64_t st, int64_t sh, int vp, int esize) {
  return ((uintptr_t)p % (size_t)(vp * esize)) == 0 && st % vp == 0 && sh % vp == 0;
}

int rope_check(const char* name, const cgHeadRows* x, int T, int D, int dtype) {
  if (!x || (!x->x && T != 0)) CG_FAIL(CG_ERR_BAD_ARG, "%s: null tensor", name);
  if (x->heads < 1 || T < 0 || D < 2) CG_FAIL(CG_ERR_BAD_ARG, "%s: bad sizes T=%d heads=%d D=%d", name, T, x->heads, D);
  if (x->heads > 0x3fffffff) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: %d heads (at most 2^30 - 1)", name, x->heads);
  if (x->stride_t < 0 || x->stride_h < 0) CG_FAIL(CG_ERR_BAD_ARG, "%s: negative strides", name);
  if (D % 2 || D > 256) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: head width %d (even, at most 256)", name, D);
  if (dtype != 0 && dtype != 1) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: dtype %d (0 bf16, 1 fp32)", name, dtype);
  return CG_OK;
}
int rope_check_rot(const char* name, const cgRotation* r, int T, int D) {
  if (!r) return CG_OK;
  if ((!r->positions && T != 0) || !r->freq) CG_FAIL(CG_ERR_BAD_ARG, "%s: null positions or frequencies", name);
  if (r->axes < 1 || r->rot < 2 || r->rot > D || r->rot % (2 * r->axes))
    CG_FAIL(CG_ERR_BAD_ARG, "%s: rotated width %d of %d over %d axes", name, r->rot, D, r->axes);
  return CG_OK;
}

// fills what depends on sizes; returns VP
int rope_plan(RopeArgs* a, const cgRotation* rot, int T, int D, int esize, bool bwd, int* grid) {
  a->T = T;
  a->D = D;
  a->inv_d = 1.f / (float)D;
  a->rot = rot ? rot->rot : 0;
  a->pairs = a->rot / 2;
  a->axes = rot ? rot->axes : 1;
  a->per_axis = rot ? a->pairs / rot->axes : 1;
  a->interleaved = rot ? rot->interleaved : 0;
  a->positions = rot ? rot->positions : nullptr;
  a->freq = rot ? rot->freq : nullptr;
  a->amplitude = rot ? rot->amplitude : 1.f;
  a->dper = make_fastdiv(a->per_axis);
  // 16-byte loads; the backward pass of bf16 data takes 8-byte ones: with 16 elements a lane it has 188 registers and
  // two waves a SIMD (65 536 tokens, 12 heads of 32: 51 us, with 8 elements 38)
  int vp = bwd || esize == 4 ? 4 : 8;
  for (; vp > 1; vp >>= 1) {
    // interleaved pairs lie one behind the other: a unit may hold the last pairs and the first copied entries; with
    // halves the two parts of a unit have to end together
    bool ok = D % (2 * vp) == 0 && (a->interleaved || (a->pairs % vp == 0 && (D - a->rot) % (2 * vp) == 0));
    for (int s = 0; s < a->ntensors; ++s)
      ok = ok && aligned_for(a->t[s].x, a->t[s].st, a->t[s].sh, vp, esize) &&
           (uintptr_t)a->t[s].out % (vp * esize) == 0 && (uintptr_t)a->t[s].dy % (vp * esize) == 0;
    if (ok) break;
  }
  a->pair_units = cdiv(a->pairs, vp);
  a->slots = a->pair_units * vp;
  a->dslots = make_fastdiv(a->slots > 0 ? a->slots : 1);
  a->units = D / (2 * vp);
  a->lanes = 1;
  a->lanes_log = 0;
  while (a->lanes < a->units && a->lanes < 64) {
    a->lanes <<= 1;
    ++a->lanes_log;
  }
  int64_t token = 0;      // elements
  for (int s = 0; s < a->ntensors; ++s) token += (int64_t)a->t[s].heads * D;
  // Tokens a block, so that its angles and its launch are spread over enough data, but not so many that fewer than 1024
  // blocks are left for 256 CUs.  A rotation alone: about 6 K elements (262 144 tokens x 3 heads of 64: 32 us, with 16 K
  // 34 us; 65 536 x 16 heads of 128: 94 us, 98 us); with the norm, whose gains are read once a block: 32 K (65 536 x 40
  // heads of 128: 277 us, with 16 K 306 us).
  int tb = (int)((a->ntensors == 2 ? 32768 : 6144) / token);
  const int room = a->slots > 0 ? ROPE_LDS_FLOATS / 2 / a->slots : tb;
  if (tb > room) tb = room;
  if (tb > cdiv(T, 1024)) tb = cdiv(T, 1024);
  a->tb = tb < 1 ? 1 : tb;
  a->chunks = cdiv(T, a->tb);
  *grid = a->chunks;
  if (bwd && *grid > ROPE_MAX_BLOCKS_BWD) *grid = ROPE_MAX_BLOCKS_BWD;
  return vp;
}

template <typename T, int VP, int UPL, bool NORM, bool BWD>
void rope_launch_form(const RopeArgs& a, int grid, hipStream_t st) {
  if constexpr (VP > 1) {
    if (a.slots != a.pairs) {
      rope_kernel<T, VP, UPL, NORM, BWD, true><<<grid, 256, 0, st>>>(a);
      return;
    }
  }
  rope_kernel<T, VP, UPL, NORM, BWD, false><<<grid, 256, 0, st>>>(a);
}

template <typename T, bool NORM, bool BWD>
void rope_launch(const RopeArgs& a, int vp, int grid, hipStream_t st) {
  if constexpr (sizeof(T) == 2 && !BWD) {
    if (vp == 8) return rope_launch_form<T, 8, 1, NORM, BWD>(a, grid, st);
  }
  switch (vp) {
    case 4: return rope_launch_form<T, 4, 1, NORM, BWD>(a, grid, st);
    case 2: return rope_launch_form<T, 2, 1, NORM, BWD>(a, grid, st);
    default: return rope_launch_form<T, 1, 2, NORM, BWD>(a, grid, st);
  }
}

void rope_tensor(RopeTensor* t, const cgHeadRows* x, const void* dy, void* out) {
  t->x = x->x;
  t->dy = dy;
  t->out = out;
  t->gain = x->gain;
  t->st = x->stride_t;
  t->sh = x->stride_h;
  t->heads = x->heads;
  t->dheads = make_fastdiv((uint32_t)x->heads);
}

}  // namespace

extern "C" int cg_rotary(const cgHeadRows* x, int T, int D, int dtype, const cgRotation* rot, int inverse,
                         void* y, cgStream stream) {
  int rc = rope_check("cg_rotary", x, T, D, dtype);
  if (rc) return rc;
  if (!rot) CG_FAIL(CG_ERR_BAD_ARG, "cg_rotary: null rotation");
  if ((rc = rope_check_rot("cg_rotary", rot, T, D))) return rc;
  if (T == 0) return CG_OK;
  if (!y) CG_FAIL(CG_ERR_BAD_ARG, "cg_rotary: null output");
  RopeArgs a = {};
  a.ntensors = 1;
  rope_tensor(&a.t[0], x, nullptr, y);
  a.sign = inverse ? -1.f : 1.f;
  int grid;
  const int vp = rope_plan(&a, rot, T, D, dtype ? 4 : 2, false, &grid);
  if (dtype) rope_launch<float, false, false>(a, vp, grid, (hipStream_t)stream);
  else rope_launch<bf16_t, false, false>(a, vp, grid, (hipStream_t)stream);
  CG_CHECK_LAUNCH("cg_rotary");
  return CG_OK;
}

extern "C" int cg_qk_norm_rotary_fwd(const cgHeadRows* q, const cgHeadRows* k, int T, int D, int dtype,
                                     float eps, const cgRotation* rot, void* q_out, void* k_out,
                                     cgStream stream) {
  const char* name = "cg_qk_norm_rotary_fwd";
  int rc = rope_check(name, q, T, D, dtype);
  if (rc || (rc = rope_check(name, k, T, D, dtype)) || (rc = rope_check_rot(name, rot, T, D))) return rc;
  if (!(eps >= 0.f)) CG_FAIL(CG_ERR_BAD_ARG, "%s: eps", name);
  if (T == 0) return CG_OK;
  if (!q_out || !k_out) CG_FAIL(CG_ERR_BAD_ARG, "%s: null output", name);
  RopeArgs a = {};
  a.ntensors = 2;
  rope_tensor(&a.t[0], q, nullptr, q_out);
  rope_tensor(&a.t[1], k, nullptr, k_out);
  a.sign = 1.f;
  a.eps = eps;
  int grid;
  const int vp = rope_plan(&a, rot, T, D, dtype ? 4 : 2, false, &grid);
  if (dtype) rope_launch<float, true, false>(a, vp, grid, (hipStream_t)stream);
  else rope_launch<bf16_t, true, false>(a, vp, grid, (hipStream_t)stream);
  CG_CHECK_LAUNCH(name);
  return CG_OK;
}

extern "C" size_t cg_qk_norm_rotary_bwd_workspace_bytes(int T, int D) {
  if (T < 1 || D < 1) return 0;
  return (size_t)(T < ROPE_MAX_BLOCKS_BWD ? T : ROPE_MAX_BLOCKS_BWD) * 2 * (size_t)D * sizeof(float);
}

extern "C" int cg_qk_norm_rotary_bwd(const cgHeadRows* q, const cgHeadRows* k, const void* dq_out,
                                     const void* dk_out, int T, int D, int dtype, float eps,
                                     const cgRotation* rot, void* dq, void* dk, float* dq_gain,
                                     float* dk_gain, void* ws, size_t ws_bytes, cgStream stream) {
  const char* name = "cg_qk_norm_rotary_bwd";
  int rc = rope_check(name, q, T, D, dtype);
  if (rc || (rc = rope_check(name, k, T, D, dtype)) || (rc = rope_check_rot(name, rot, T, D))) return rc;
  if (!(eps >= 0.f)) CG_FAIL(CG_ERR_BAD_ARG, "%s: eps", name);
  if (T > 0 && (!dq_out || !dk_out || !dq || !dk)) CG_FAIL(CG_ERR_BAD_ARG, "%s: null gradient", name);
  if (T > 0 && (!ws || ws_bytes < cg_qk_norm_rotary_bwd_workspace_bytes(T, D)))
    CG_FAIL(CG_ERR_WORKSPACE, "%s: workspace of %zu bytes", name, ws_bytes);
  RopeArgs a = {};
  int grid = 0;
  if (T > 0) {
    a.ntensors = 2;
    rope_tensor(&a.t[0], q, dq_out, dq);
    rope_tensor(&a.t[1], k, dk_out, dk);
    a.sign = -1.f;
    a.eps = eps;
    a.partial = (float*)ws;
    const int vp = rope_plan(&a, rot, T, D, dtype ? 4 : 2, true, &grid);
    if (dtype) rope_launch<float, true, true>(a, vp, grid, (hipStream_t)stream);
    else rope_launch<bf16_t, true, true>(a, vp, grid, (hipStream_t)stream);
    CG_CHECK_LAUNCH(name);
  }
  if (dq_gain || dk_gain) {   // (T == 0: no partials, zeros)
    rope_gain_kernel<<<cdiv(2 * D, 16), 1024, 0, (hipStream_t)stream>>>((const float*)ws, grid, D, dq_gain,
                                                                       dk_gain);
    CG_CHECK_LAUNCH(name);
  }
  return CG_OK;
}
