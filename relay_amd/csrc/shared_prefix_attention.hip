// Decode attention for sequences that share the blocks of a prefix (relay's prefix cache,
// block_manager.cpp): softmax(scale q K^T) V over each token's context, where the keys of the
// shared prefix are read once for all members of a group and not once for each.
//
// Per kv head the members' query heads form one matrix of members * G rows against the prefix's K
// and V; the keys behind the prefix are each token's own. Both are the same work on another
// list of rows and range of keys: a workgroup takes 32 rows and a slice of keys,
//
//   S^T[32 keys x 32 rows] = K[32 keys x D] * Q^T[D x 32 rows]          (MFMA 32x32x16)
//   online softmax per row in the log2 domain, in fp32 (lanes c and c + 32 hold row c)
//   O^T[D x 32 rows] += V^T[D x 32 keys] * P^T[32 keys x 32 rows]       (MFMA 32x32x16)
//
// its waves taking every kWaves-th step of 32 keys, and leaves (maximum, sum, O) of the slice; the
// slices of a row are joined by log-sum-exp in a second launch.
#include <algorithm>
#include <string>

#include "../../include/relay_hip.h"
#include "common.h"

namespace relay_hip {
namespace {

constexpr int kRows = 32;   // query rows of a workgroup
constexpr int kStep = 32;   // keys of a wave's step
constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;

struct SharedArgs {
  const half_t* q;
  int64_t q_stride;
  const half_t *kpool, *vpool;
  const int4* meta;    // per token: row, context, table offset, shared keys
  const int4* groups;  // first token, members, shared keys, table offset
  const int* tables;
  int n_dec, n_groups, heads, kv_heads, group, block, bs_shift;
  int shared_slice, shared_parts, own_slice, own_parts, tiles, own_tiles;  // tiles: row tiles of a group, of a token
  int shared_wgs;                                                          // workgroups on prefixes, the first ones
  float scale_log2;
  float *part_o, *part_ml;
  half_t* out;
  int64_t out_stride;
};

// Slices of `keys` keys where the launch has room for `most`; the last takes what is left.
__device__ __forceinline__ int parts_of(int keys, int slice, int most) {
  return keys <= 0 ? 0 : min(most, (keys + slice - 1) / slice);
}

__device__ __forceinline__ float row_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_sum(float x) { return x + __shfl_xor(x, 32); }

// Swizzle of a key's 16-byte chunks in the V staging rows.
template <int D>
__device__ __forceinline__ int vswz(int key) {
  return D == 128 ? ((key & 3) << 2) | ((key >> 2) & 3) : D == 64 ? key & 7 : (key >> 2) & 3;
}

// D: compute width, DR: head size of the rows (16 runs at width 32 with zeros behind).
template <int D, int DR>
__global__ __launch_bounds__(kThreads) void shared_attention_kernel(const SharedArgs a) {
  constexpr int CH = D / 8;             // 16-byte chunks a row
  constexpr int MK = D / 16;            // QK products a step
  constexpr int DT = D / 32;            // 32-wide tiles of O^T
  constexpr int VL = kStep * CH / kWave;
  constexpr int XWAVE = DT * 16 * 64 + 2 * 64;  // floats that a wave hands over
  constexpr int SMEM = std::max(kWaves * kStep * D * 2, kWaves / 2 * XWAVE * 4);
  __shared__ __attribute__((aligned(16))) char smem[SMEM];

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, hh = lane >> 5;

  // The workgroup's rows (as tokens and heads), table and keys.
  int b = blockIdx.x, first, members, table_off, begin, end, part, tile, tile_step, kvh;
  if (b < a.shared_wgs) {
    tile = b % a.tiles, b /= a.tiles;
    part = b % a.shared_parts, b /= a.shared_parts;
    kvh = b % a.kv_heads;
    const int4 g = a.groups[b / a.kv_heads];
    first = g.x, members = g.y, table_off = g.w;
    const int parts = parts_of(g.z, a.shared_slice, a.shared_parts);
    if (part >= parts) return;
    begin = part * a.shared_slice;
    end = part == parts - 1 ? g.z : begin + a.shared_slice;
    tile_step = a.tiles;
  } else {
    b -= a.shared_wgs;
    tile = b % a.own_tiles, b /= a.own_tiles;
    part = b % a.own_parts, b /= a.own_parts;
    kvh = b % a.kv_heads;
    first = b / a.kv_heads, members = 1;
    const int4 m = a.meta[first];
    table_off = m.z;
    const int from = max(m.w, 0), parts = parts_of(m.y - from, a.own_slice, a.own_parts);
    if (part >= parts) return;
    begin = from + part * a.own_slice;
    end = part == parts - 1 ? m.y : begin + a.own_slice;
    part += parts_of(m.w, a.shared_slice, a.shared_parts);
    tile_step = a.own_tiles;
  }
  const int* table = a.tables + table_off;
  const int G = a.group, bs = a.block, sh = a.bs_shift;

  for (; tile * kRows < members * G; tile += tile_step) {
    const int r = tile * kRows + c;
    const bool on = r < members * G;
    const int token = first + (on ? r / G : 0), head = kvh * G + (on ? r % G : 0);
    const int4 m = a.meta[token];
    const int lim = on ? min(m.y, end) : 0;  // the row sees the keys before this

    half8 qb[MK];
#pragma unroll
    for (int i = 0; i < MK; ++i) {
      if (lim > 0 && (DR == D || 16 * i + 8 * hh < DR)) {
        qb[i] = load_half8(a.q + m.x * a.q_stride + static_cast<int64_t>(head) * DR + 16 * i + 8 * hh);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) qb[i][e] = 0;
      }
    }
    float16v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    float m_run = -INFINITY, l_run = 0.0f;
    half_t* const sv = reinterpret_cast<half_t*>(smem) + w * kStep * D;

    const auto offset = [&](int key) {
      key = min(key, end - 1);
      const int blk = table[sh >= 0 ? key >> sh : key / bs];
      return kv_row_offset(blk, a.kv_heads, kvh, bs, sh >= 0 ? key & (bs - 1) : key % bs, DR);
    };
    for (int k0 = begin + w * kStep; k0 < end; k0 += kWaves * kStep) {
      half8 k[MK], v[VL];
      const int64_t krow = offset(k0 + c);
#pragma unroll
      for (int i = 0; i < MK; ++i) {
        if (DR == D || 16 * i + 8 * hh < DR) {
          k[i] = load_half8(a.kpool + krow + 16 * i + 8 * hh);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) k[i][e] = 0;
        }
      }
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int kl = i * (kWave / CH) + lane / CH, cc = lane % CH;
        if ((DR == D || 8 * cc < DR) && k0 + kl < end) {
          v[i] = load_half8(a.vpool + offset(k0 + kl) + 8 * cc);
        } else {  // its weight is 0, its bytes may be anything
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = 0;
        }
        *reinterpret_cast<half8*>(sv + kl * D + ((cc ^ vswz<D>(kl)) << 3)) = v[i];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

      float16v s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < MK; ++i) s = mfma32x32x16(k[i], qb[i], s);
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = k0 + 8 * (e >> 2) + 4 * hh + (e & 3);
        s[e] = key < lim ? s[e] * a.scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[e]);
      }
      const float m_new = fmaxf(m_run, row_max(mx));
      const float ref = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = fast_exp2(m_run - ref);
      m_run = m_new;
      half8 p[2];
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = fast_exp2(s[e] - ref);
        sum += x;
        p[e >> 3][e & 7] = static_cast<half_t>(x);
      }
      l_run = l_run * alpha + sum;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
      // V^T: a transposing read gives a lane rows kr .. kr + 3 of its column (S^T's key order).
      const int i16 = lane & 15;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          const int col = 32 * i + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
          const int kr = 16 * u + 4 * hh + (i16 >> 2);
          const half4 lo = tr_read_b64(sv + kr * D + (((col >> 3) ^ vswz<D>(kr)) << 3) + (col & 7));
          const half4 hi = tr_read_b64(sv + (kr + 8) * D + (((col >> 3) ^ vswz<D>(kr + 8)) << 3) + (col & 7));
          o[i] = mfma32x32x16(half8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, p[u], o[i]);
        }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    l_run = row_sum(l_run);

    // The waves' halves join pairwise through LDS until the first holds the slice.
    for (int n = kWaves / 2; n > 0; n >>= 1) {
      __syncthreads();
      float* const x = reinterpret_cast<float*>(smem) + (w % n) * XWAVE;
      if (w >= n && w < 2 * n) {
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[(i * 16 + e) * 64 + lane] = o[i][e];
        x[DT * 16 * 64 + lane] = m_run;
        x[DT * 16 * 64 + 64 + lane] = l_run;
      }
      __syncthreads();
      if (w < n) {
        const float m2 = x[DT * 16 * 64 + lane], l2 = x[DT * 16 * 64 + 64 + lane];
        const float mm = fmaxf(m_run, m2), ref = mm == -INFINITY ? 0.0f : mm;
        const float f1 = fast_exp2(m_run - ref), f2 = fast_exp2(m2 - ref);
        m_run = mm;
        l_run = l_run * f1 + l2 * f2;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[i][e] = o[i][e] * f1 + x[(i * 16 + e) * 64 + lane] * f2;
      }
    }
    if (w == 0 && on && m.y > 0) {
      const int64_t at = (static_cast<int64_t>(token) * a.heads + head) * (a.shared_parts + a.own_parts) + part;
      if (hh == 0) {
        a.part_ml[2 * at] = m_run;
        a.part_ml[2 * at + 1] = l_run;
      }
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int d = 32 * i + 2 * e + 4 * hh;
          if (DR == D || d < DR) *reinterpret_cast<float4*>(a.part_o + at * DR + d) = float4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
        }
    }
    __syncthreads();
  }
}

// A thread per output value.
__global__ void shared_join_kernel(const SharedArgs a, int D) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= static_cast<int64_t>(a.n_dec) * a.heads * D) return;
  const int d = static_cast<int>(i % D), head = static_cast<int>(i / D % a.heads), token = static_cast<int>(i / D / a.heads);
  const int4 m = a.meta[token];
  if (m.y <= 0) return;
  const int parts = parts_of(m.w, a.shared_slice, a.shared_parts) + parts_of(m.y - max(m.w, 0), a.own_slice, a.own_parts);
  const int64_t at = (static_cast<int64_t>(token) * a.heads + head) * (a.shared_parts + a.own_parts);
  float M = -INFINITY, L = 0.0f, O = 0.0f;
  for (int p = 0; p < parts; ++p) M = fmaxf(M, a.part_ml[2 * (at + p)]);
  for (int p = 0; p < parts; ++p) {
    const float f = fast_exp2(a.part_ml[2 * (at + p)] - M);
    L += f * a.part_ml[2 * (at + p) + 1];
    O += f * a.part_o[(at + p) * D + d];
  }
  a.out[m.x * a.out_stride + static_cast<int64_t>(head) * D + d] = static_cast<half_t>(O / L);
}

struct Plan {
  int shared_slice, shared_parts, own_slice, own_parts, tiles, own_tiles;
};

Plan plan_of(int n_dec, int n_groups, int max_members, int max_shared, int max_own, int heads, int kv_heads, int head_dim) {
  const int group = heads / kv_heads;
  Plan p{kStep * kWaves, 1, kStep * kWaves, 1, 1, (group + kRows - 1) / kRows};
  const auto cut = [](int64_t wgs, int keys, int* slice, int* parts) {
    const int least = kStep * kWaves;
    const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(1, wgs));
    *slice = std::max<int64_t>(least, ((keys + want - 1) / want + least - 1) / least * least);
    *parts = std::max(1, (keys + *slice - 1) / *slice);
  };
  p.tiles = std::max<int64_t>(1, (static_cast<int64_t>(max_members) * group + kRows - 1) / kRows);
  cut(static_cast<int64_t>(n_groups) * kv_heads * p.tiles, max_shared, &p.shared_slice, &p.shared_parts);
  cut(static_cast<int64_t>(n_dec) * kv_heads * p.own_tiles, max_own, &p.own_slice, &p.own_parts);
  return p;
}

}  // namespace
}  // namespace relay_hip

using namespace relay_hip;

extern "C" size_t rh_shared_prefix_workspace(int n_dec, int n_groups, int max_members, int max_shared, int max_own, int heads,
                                             int kv_heads, int head_dim) {
  if (n_dec <= 0 || n_groups < 0 || max_members < 0 || max_shared < 0 || max_own < 0 || kv_heads <= 0 || heads <= 0 ||
      heads % kv_heads || head_dim <= 0)
    return 0;
  const Plan p = plan_of(n_dec, n_groups, max_members, max_shared, max_own, heads, kv_heads, head_dim);
  return static_cast<size_t>(n_dec) * heads * (p.shared_parts + p.own_parts) * (head_dim + 2) * 4;
}

extern "C" int rh_shared_prefix_attention(const void* q, int64_t q_row_stride, const void* kpool, const void* vpool,
                                          const int* dec_meta, const int* groups, const int* tables, int n_dec,
                                          int n_groups, int max_members, int max_shared, int max_own, int heads,
                                          int kv_heads, int head_dim, int block_size, float scale, void* workspace,
                                          size_t workspace_bytes, void* out, int64_t out_row_stride, void* stream) {
  if (n_dec == 0) return 0;
  RH_REQUIRE(n_dec > 0 && n_groups >= 0 && max_members >= 0 && max_shared >= 0 && max_own >= 0,
             "shared prefix attention: bad sizes");
  RH_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "shared prefix attention: bad head counts");
  RH_REQUIRE(head_dim == 16 || head_dim == 32 || head_dim == 64 || head_dim == 128,
             "shared prefix attention: head_dim must be 16, 32, 64 or 128");
  RH_REQUIRE(block_size > 0, "shared prefix attention: bad block size");
  RH_REQUIRE(q && kpool && vpool && dec_meta && tables && out && (groups || n_groups == 0),
             "shared prefix attention: missing pointer");
  RH_REQUIRE(q_row_stride % 8 == 0 && out_row_stride >= static_cast<int64_t>(heads) * head_dim,
             "shared prefix attention: q rows must be 16-byte aligned and out rows hold heads * head_dim");
  RH_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kpool) | reinterpret_cast<uintptr_t>(vpool) |
              reinterpret_cast<uintptr_t>(dec_meta) | reinterpret_cast<uintptr_t>(groups)) % 16 == 0,
             "shared prefix attention: q, the pools, dec_meta and groups must be 16-byte aligned");
  const size_t need = rh_shared_prefix_workspace(n_dec, n_groups, max_members, max_shared, max_own, heads, kv_heads, head_dim);
  RH_REQUIRE(workspace_bytes >= need && (!need || (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0)),
             "shared prefix attention: needs a 16-byte aligned workspace of rh_shared_prefix_workspace bytes");
  const Plan p = plan_of(n_dec, n_groups, max_members, max_shared, max_own, heads, kv_heads, head_dim);
  SharedArgs a{};
  a.q = static_cast<const half_t*>(q);
  a.q_stride = q_row_stride;
  a.kpool = static_cast<const half_t*>(kpool);
  a.vpool = static_cast<const half_t*>(vpool);
  a.meta = reinterpret_cast<const int4*>(dec_meta);
  a.groups = reinterpret_cast<const int4*>(groups);
  a.tables = tables;
  a.n_dec = n_dec;
  a.n_groups = n_groups;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.group = heads / kv_heads;
  a.block = block_size;
  a.bs_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
  a.shared_slice = p.shared_slice;
  a.shared_parts = p.shared_parts;
  a.own_slice = p.own_slice;
  a.own_parts = p.own_parts;
  a.tiles = p.tiles;
  a.own_tiles = p.own_tiles;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + static_cast<size_t>(n_dec) * heads * (p.shared_parts + p.own_parts) * head_dim;
  a.out = static_cast<half_t*>(out);
  a.out_stride = out_row_stride;
  const int64_t shared_wgs = static_cast<int64_t>(n_groups) * kv_heads * p.shared_parts * p.tiles;
  const int64_t wgs = shared_wgs + static_cast<int64_t>(n_dec) * kv_heads * p.own_parts * p.own_tiles;
  const int64_t values = static_cast<int64_t>(n_dec) * heads * head_dim;
  RH_REQUIRE(wgs < (int64_t{1} << 31) && values < (int64_t{1} << 38), "shared prefix attention: too large");
  a.shared_wgs = static_cast<int>(shared_wgs);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(wgs)), dim3(kThreads), 0, s, a);
  };
  switch (head_dim) {
    case 16: RH_TRY_LAUNCH(launch(shared_attention_kernel<32, 16>)); break;
    case 32: RH_TRY_LAUNCH(launch(shared_attention_kernel<32, 32>)); break;
    case 64: RH_TRY_LAUNCH(launch(shared_attention_kernel<64, 64>)); break;
    default: RH_TRY_LAUNCH(launch(shared_attention_kernel<128, 128>));
  }
  RH_TRY_LAUNCH(hipLaunchKernelGGL(shared_join_kernel, dim3(static_cast<unsigned>((values + 255) / 256)), dim3(256), 0, s, a, head_dim));
  return 0;
}
