// Decode attention for sequences that share the blocks of a prefix (relay's prefix cache,
// block_manager.cpp): softmax(scale q K^T) V over each token's context, where the keys of the
// shared prefix are read once for all members of a group and not once for each.
//
// Per kv head the members' query heads form one matrix of members * G rows against the prefix's K
// and V; the keys behind the prefix are each token's own. A workgroup of four waves takes some rows
// and a slice of keys, and leaves (maximum, sum, O) of each row; a row's slices are joined by
// log-sum-exp. Softmax in the log2 domain, sums, maxima and O in fp32; the weights are rounded to fp16
// for the product with V, as in the other attention kernels: an MFMA operand of twice the width
// would double that product. Two ways through a slice:
//
//  - many rows (prefixes of more than 16 rows or 1024 keys, or of more than 12 rows of 128): 128 rows, 32 a
//    wave, on tiles of K and V that the waves share in LDS (attend_rows). 64 x 4 rows on 16,384 keys of
//    8 heads of 128 (17 GFLOP, 67 MB) take 41 us, the join of their slices 6. Bound by the chain of a
//    step (LDS reads, products, weights: no one of them taken out made it faster by over a tenth); a
//    ring of five tiles takes 5-10% longer.
//  - few rows (own keys, short prefixes): 16 rows, the waves on keys of their own, K straight into MFMA
//    operands (attend_few). Bound by memory: 64 x 1000 own keys, 8 kv heads of 128 (ragged, 164 MB) 34 us.
//
// One launch does both, prefixes first: the prefix's products run beside the own keys' loads. 64 members on
// 16,384 keys with up to 1000 of their own (231 MB, 18 GFLOP) take 60 us, the join 5.9. Prefix tiles staged
// through registers, whose reloads from scratch waited for every load in flight, took 107 in all, and
// workgroups of eight waves that do not share their tiles 244.
#include <algorithm>
#include <exception>
#include <string>
#include <type_traits>
#include <vector>

#include "../../include/relay_hip.h"
#include "common.h"
#include "lds_ring.h"

namespace relay_hip {
namespace {

constexpr int kStrip = 32;  // query rows of a wave: a strip
constexpr int kStep = 32;   // keys of a wave's step
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kLeast = kStep * kWaves;  // slices are multiples of as many keys
constexpr int kFew = 16;    // query rows of a workgroup whose waves take keys of their own
constexpr int kMerge = 8;   // slices whose values are loaded at once (attend_few)
constexpr int kRing = 4;    // 32-key tiles of K and V in LDS, where strips share them

struct SharedArgs {
  const half_t* q;
  int64_t q_stride;
  const half_t *kpool, *vpool;
  const int4* meta;    // per token: row, context, table offset, shared keys
  const int4* groups;  // first token, members, shared keys, table offset
  const int* tables;
  int n_dec, n_groups, heads, kv_heads, group, block, bs_shift;
  int shared_slice, shared_parts, own_slice, own_parts, tiles, own_tiles;  // tiles: row tiles of a group, of a token
  int shared_units, shared_wgs, own_units;  // workgroups on prefixes come first
  int each, pieces;  // attend_few: tokens of a row tile, row tiles of a token (one of the two is 1)
  Div by_tiles, by_own_tiles, by_shared_parts, by_own_parts, by_kv_heads;
  Div by_heads, by_group, by_pieces, by_shared_slice, by_own_slice;  // of rows and tiles of attend_few, of 128 keys
  float scale_log2;
  int* counters;  // per token and kv head, counter_step apart: slices that have come (zero between calls)
  int counter_step;
  float *part_o, *part_ml;
  half_t* out;
  int64_t out_stride;
};

// Slices (of so many 128 keys) of `keys` keys where the launch has room for `most`; the last takes what is left.
__device__ __forceinline__ int parts_of(int keys, const Div& slice, int most) {
  return keys <= 0 ? 0 : min(most, slice(static_cast<int>((keys + (kLeast - 1u)) / kLeast) + static_cast<int>(slice.d) - 1));
}

__device__ __forceinline__ float row_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_sum(float x) { return x + __shfl_xor(x, 32); }

// Swizzle of a key's 16-byte chunks in LDS rows of K and V (flash_prefill.hip's, by the same reads).
template <int D>
__device__ __forceinline__ int kswz(int key) {
  return D == 128 ? ((key & 3) << 2) | ((key >> 2) & 3) : D == 64 ? key & 7 : (key >> 2) & 3;
}

// A strip's state in one wave: lanes c and c + 32 hold row c.
template <int D>
struct Strip {
  float16v o[D / 32];
  float ref, l;  // the offset of the row's weights in the log2 domain (-inf: no key seen), this lane's share of their sum
};

// Weights are 2^kUp for the greatest score so far: as fp16 they then keep their 11 bits down to 2^-25 of it and end at 2^-36. (With 1
// for the greatest they end at 2^-25: one key that outweighs each of many others by that much, and the others were lost.)
constexpr float kUp = 11.0f;

// P = exp2(S scale - ref) with the row's running maximum less `up` as ref, and the sum. O and l are rescaled where a
// row of the wave has a new maximum: on fewer and fewer steps. (An offset that moved only before a
// weight could overflow fp16 took up to 5% less time, and doubled the noise of the weights' rounding:
// with a maximum as offset the greatest weight, which counts most, is a power of two.) A masked key's S is -inf.
template <int D>
__device__ __forceinline__ void weigh(Strip<D>& st, const float16v& s, half8 (&p)[2], float scale, float up) {
  float mx = s[0];
#pragma unroll
  for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
  mx = row_max(mx) * scale - up;
  if (__ballot(mx > st.ref) != 0) {
    const float ref = fmaxf(mx, st.ref), alpha = ref == -INFINITY ? 1.0f : fast_exp2(st.ref - ref);
    st.ref = ref;
    st.l *= alpha;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) st.o[i][e] *= alpha;
  }
  const float nref = st.ref == -INFINITY ? 0.0f : -st.ref;
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float x = fast_exp2(fmaf(s[e], scale, nref));
    sum += x;
    p[e >> 3][e & 7] = static_cast<half_t>(x);
  }
  st.l += sum;
}

// V^T operands of 32 keys whose rows begin at sv: a transposing read gives a lane rows kr .. kr + 3 of
// its column (S^T's key order).
template <int D>
__device__ __forceinline__ void read_v(half8 (&v)[2][D / 32], const half_t* sv) {
  const int lane = threadIdx.x & 63, hh = lane >> 5, i16 = lane & 15;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const int col = 32 * i + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
      const int kr = 16 * u + 4 * hh + (i16 >> 2);
      const half4 a = tr_read_b64(sv + kr * D + (((col >> 3) ^ kswz<D>(kr)) << 3) + (col & 7));
      const half4 b = tr_read_b64(sv + (kr + 8) * D + (((col >> 3) ^ kswz<D>(kr + 8)) << 3) + (col & 7));
      v[u][i] = half8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
}

// O^T += V^T P^T
template <int D>
__device__ __forceinline__ void add_pv(Strip<D>& st, const half8 (&v)[2][D / 32], const half8 (&p)[2]) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) st.o[i] = mfma32x32x16(v[u][i], p[u], st.o[i]);
}

// Only keys lo .. lim - 1 of the 32 from key0 on count. (The empty asm keeps the selects in the branch
// that calls this: as selects on every step they cost 100 registers.)
__device__ __forceinline__ void mask_keys(float16v& s, int key0, int lo, int lim) {
  asm volatile("");
  const int first = key0 + 4 * ((threadIdx.x & 63) >> 5), from = lo - first, to = lim - first;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int k = 8 * (e >> 2) + (e & 3);
    if (k < from || k >= to) s[e] = -INFINITY;
  }
}

// One fma a score, fma(S, scale, -ref), is off for the greatest key by the rounding error of ref: up to 4 where scores reach 2^27,
// and beyond by more than fp16's range. Waves whose queries could have such scores (on keys of 65504) round S scale to fp32
// first, as the few rows' path does, and weigh the greatest by 1.
constexpr float kFar = 134217728.0f;

__device__ __forceinline__ void scale_first(float16v& s, float scale) {
  asm volatile("");
#pragma unroll
  for (int e = 0; e < 16; ++e) s[e] = mul_rounded(s[e], scale);
}

__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 1 KB from global memory to LDS: lane l's 16 bytes at base + offset go to lds + 16 l. No output
// register; the ring's own waits order it before the reads (as lds_ring.h's buffer form, which
// reaches 2 GB from its base; a cache may be larger). Non-temporal, which leaves the L2 to the row tiles that
// run beside each other: 64 members on 16,384 keys with own keys 67.8 -> 64.7 us, small calls level.
__device__ __forceinline__ void global_to_lds(const half_t* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
               :
               : "v"(offset), "s"(base), "s"(lds)
               : "memory");
}

// A workgroup's share: rows of `members` tokens' G heads (row tiles tile, tile + step, ...) against keys
// begin .. end - 1 of a table.
struct Share {
  int first, members, kvh, begin, end, part, tile, step;
  const int* table;
};

typedef const __attribute__((address_space(4))) int* scalar_ints;  // uniform reads go through the scalar unit

// The block of a table's entry. Entries that hold none may be any negative number: they lead to block 0 and not outside the pools
// where a group is said to share more keys than its table has (the max is taken where an entry is used: at its load, a step ahead, it would wait for it).
__device__ __forceinline__ int block_at(int entry) { return max(entry, 0); }

// ---- many rows: the waves share tiles of K and V in LDS, 32 rows a wave ---------------------------
//
//   S^T[32 keys x 32 rows] = K[32 keys x D] * Q^T[D x 32 rows]          (MFMA 32x32x16)
//   O^T[D x 32 rows] += V^T[D x 32 keys] * P^T[32 keys x 32 rows]       (MFMA 32x32x16)
//
// with lanes c and c + 32 on row c. Tiles come by loads straight to LDS into a ring of kRing, three
// tiles ahead. D is the head size; 16 keys from a multiple of 16 on lie in one block.
template <int D>
__device__ __forceinline__ void attend_rows(const SharedArgs& a, Share g, char* smem) {
  constexpr int CH = D / 8;            // 16-byte chunks a row
  constexpr int MK = D / 16;           // QK products a step
  constexpr int DT = D / 32;           // 32-wide tiles of O^T
  constexpr int KEYS = kWave / CH;     // keys of a 1 KB piece
  constexpr int PER16 = 16 / KEYS;     // pieces of 16 keys
  constexpr int TILE = kStep * D;      // halves of a tile's K
  static_assert(KEYS <= 16, "a piece lies in one block");
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.group, bs = a.block, sh = a.bs_shift;
  const half_t* const ring = reinterpret_cast<const half_t*>(smem);
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_address(smem));
  const scalar_ints entries = (scalar_ints)(g.table);
  const half_t* const pool = w >= 2 ? a.vpool : a.kpool;
  const int n = (g.end - g.begin + kStep - 1) / kStep;

  for (; g.tile * kWaves * kStrip < g.members * G; g.tile += g.step) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // keeps what depends on it from being held across the loop over tiles
    const int c = lane & 31, hh = lane >> 5;
    // A wave brings half a tile's K or V, 16 keys of one table entry, which it looks up a tile ahead.
    int entry;
    const auto first16 = [&](int j) { return min(g.begin + j * kStep + 16 * (w & 1), (g.end - 1) & ~15); };
    const auto lookup = [&](int j) { entry = entries[first16(j) >> sh]; };
    uint32_t piece[PER16];  // a lane's offsets in 16 keys
    const auto pieces_to = [&](int last) {
#pragma unroll
      for (int i = 0; i < PER16; ++i) {
        const int at = i * KEYS + lane / CH;
        piece[i] = (min(at, last) * D + 8 * ((lane % CH) ^ kswz<D>(16 * (w & 1) + at))) * 2;
      }
    };
    pieces_to(15);
    const auto send = [&](int j, int slot) {
      const int key = first16(j);
      const half_t* const base = pool + ((static_cast<int64_t>(block_at(entry)) * a.kv_heads + g.kvh) * bs + (key & (bs - 1))) * D;
      if (g.end - key < 16) pieces_to(g.end - 1 - key);  // the last tile: past the end the last key again
#pragma unroll
      for (int i = 0; i < PER16; ++i)
        global_to_lds(base, piece[i], lds + (slot * 2 * TILE + (w >> 1) * TILE + (16 * (w & 1) + i * KEYS) * D) * 2);
    };
    lookup(0);
    for (int j = 0; j < kRing - 1; ++j)
      if (j < n) {
        send(j, j);
        lookup(j + 1);
      }

    const int r = (g.tile * kWaves + w) * kStrip + c;
    const bool on = r < g.members * G;
    const int token = g.first + (on ? r / G : 0), head = g.kvh * G + (on ? r % G : 0);
    const int4 m = a.meta[token];
    const int lim = on ? min(m.y, g.end) : g.end;  // the row sees the keys before this
    int all = lim;                                 // every row of the strip sees the keys before this
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = min(all, __shfl_xor(all, o));
    all = __builtin_amdgcn_readfirstlane(all);

    half8 qb[MK];
#pragma unroll
    for (int i = 0; i < MK; ++i) {
      if (on && m.y > 0) {
        qb[i] = load_half8(a.q + m.x * a.q_stride + static_cast<int64_t>(head) * D + 16 * i + 8 * hh);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) qb[i][e] = 0;
      }
    }
#pragma unroll
    for (int i = 0; i < MK; ++i) asm volatile("" : "+v"(qb[i]));  // q is here: the loop waits for its own loads alone
    Strip<D> st;
    st.ref = -INFINITY, st.l = 0.0f;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) st.o[i][e] = 0.0f;

    // Step j has S of tile j. It waits for tile j + 1 (one barrier, which also frees tile j - 1's
    // buffer to be sent for again), reads its K while tile j's weights are computed, and tile j's V
    // while the next S is: the LDS reads' latency lies under other work.
    // (Unrolled by the ring, so that a buffer's address is a constant beside the lane's.)
    half8 k[MK];
    const auto read_k = [&](int slot) {
      const half_t* const kt = ring + slot * 2 * TILE + c * D;
#pragma unroll
      for (int i = 0; i < MK; ++i) k[i] = *reinterpret_cast<const half8*>(kt + (((2 * i + hh) ^ kswz<D>(c)) << 3));
    };
    float16v s;
    const auto scores = [&] {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < MK; ++i) s = mfma32x32x16(k[i], qb[i], s);
    };
    wait_stages<PER16, kRing - 2>(min(n - 1, kRing - 2));
    ring_barrier();
    // The sum of a row's |q| says what scores it could have.
    float size = 0.0f;
#pragma unroll
    for (int i = 0; i < MK; ++i) {
      const uint4v bits = __builtin_bit_cast(uint4v, qb[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        size = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, bits[e] & 0x7fff7fffu), half2_t{1, 1}, size, false);
    }
    const bool far = __ballot(row_sum(size) * 65504.0f * a.scale_log2 >= kFar) != 0;
    const float by = far ? 1.0f : a.scale_log2, up = far ? 0.0f : kUp;
    const int plain = far ? 0 : all;  // the scores of steps up to here are left as they come
    const bool busy = (g.tile * kWaves + w) * kStrip < g.members * G;  // a wave without rows only brings tiles
    read_k(0);
    scores();
    const auto step = [&](int j, auto slot_tag) {
      constexpr int SLOT = decltype(slot_tag)::value;
      const bool more = j + 1 < n;
      if (more) wait_stages<PER16, kRing - 3>(min(n - 2 - j, kRing - 3));
      ring_barrier();
      if (j + kRing - 1 < n) {
        send(j + kRing - 1, (SLOT + kRing - 1) % kRing);
        lookup(j + kRing);
      }
      if (!busy) return;
      if (more) read_k((SLOT + 1) % kRing);
      __builtin_amdgcn_sched_barrier(0);
      const int k0 = g.begin + j * kStep;
      if (k0 + kStep > plain) {
        if (far) scale_first(s, a.scale_log2);
        if (k0 + kStep > all) mask_keys(s, k0, g.begin, lim);
      }
      half8 p[2], v[2][DT];
      weigh(st, s, p, by, up);
      read_v<D>(v, ring + SLOT * 2 * TILE + TILE);
      __builtin_amdgcn_sched_barrier(0);
      if (more) scores();
      add_pv(st, v, p);
    };
    static_assert(kRing == 4, "four steps a turn");
    for (int j = 0; j < n; j += kRing) {
      step(j, std::integral_constant<int, 0>{});
      if (j + 1 < n) step(j + 1, std::integral_constant<int, 1>{});
      if (j + 2 < n) step(j + 2, std::integral_constant<int, 2>{});
      if (j + 3 < n) step(j + 3, std::integral_constant<int, 3>{});
    }
    st.l = row_sum(st.l);
    __syncthreads();

    // Out through LDS, so that a row's values leave as whole lines (each wave has 32 rows of D floats
    // there; row c is rotated by 4 c: the 32 rows of one write would otherwise hit the same banks).
    float* const x = reinterpret_cast<float*>(smem) + w * kStrip * D;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<float4*>(x + c * D + ((32 * i + 2 * e + 4 * hh + 4 * c) & (D - 1))) =
            float4{st.o[i][e], st.o[i][e + 1], st.o[i][e + 2], st.o[i][e + 3]};
    const int64_t at = on && m.y > 0 ? (static_cast<int64_t>(token) * a.heads + head) * (a.shared_parts + a.own_parts) + g.part : -1;
    if (hh == 0 && at >= 0) reinterpret_cast<float2*>(a.part_ml)[at] = float2{st.ref, st.l};
    wave_fence();
    constexpr int LANES = D / 4, ROWS = kWave / LANES;  // lanes of a row, rows a store
#pragma unroll
    for (int i = 0; i < kStrip; i += ROWS) {
      const int row = i + lane / LANES, d = 4 * (lane % LANES);
      const int64_t to = __shfl(at, row);
      const float4 v = *reinterpret_cast<const float4*>(x + row * D + ((d + 4 * row) & (D - 1)));
      if (to >= 0) *reinterpret_cast<float4*>(a.part_o + to * D + d) = v;
    }
    __syncthreads();
  }
}

// ---- few rows: the waves take steps of 32 keys of their own -----------------------------------------
//
//   S^T[16 keys x 16 rows] = K[16 keys x D] * Q^T[D x 16 rows], twice     (MFMA 16x16x32)
//   O^T[D x 16 rows] += V^T[D x 32 keys] * P^T[32 keys x 16 rows]         (MFMA 16x16x32)
//
// with lane (c, g) on row c and keys 4 g .. 4 g + 3 of each 16. K goes straight into MFMA operands, V through a
// staging area of the wave in LDS, and the loads of the next step are in flight under this one's work,
// so that a workgroup alone on its CU, as at the end of a batch of ragged lengths, still streams. That holds up to head size
// 64. At 128 two steps' operands pass the 256 registers by 16 (by 26 where blocks are no power of two from 16 on), and what is
// spilled in the loop is stored and fetched behind waits for all loads: every second step waits for the loads it should overlap.
template <int D, int DR>
struct KvStep {
  half8 k[2][D / 32], v[kStep * (D / 8) / kWave];
};

// Two floats, coherent across the device's XCDs (as coherent_load).
__device__ __forceinline__ float2 coherent_load2(const float* p) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return __builtin_bit_cast(float2, v);
}

// Swizzle of a key's 16-byte chunks in the staging rows.
template <int D>
__device__ __forceinline__ int vswz(int key) {
  return D >= 64 ? ((key >> 2) & 3) << 1 : ((key >> 2) & 1) << 1;
}

template <int D, int DR, bool SCALAR, bool JOIN>
__device__ __forceinline__ void attend_few(const SharedArgs& a, Share sh, char* smem) {
  constexpr int CH = D / 8, KH = D / 32, DT = D / 16, VL = kStep * CH / kWave, VKEYS = kWave / CH;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.group, bs = a.block, bshift = a.bs_shift, begin = sh.begin, end = sh.end;
  const scalar_ints entries = (scalar_ints)(sh.table);
  half_t* const sv = reinterpret_cast<half_t*>(smem) + w * kStep * D;
  float* const s_ml = reinterpret_cast<float*>(smem + kWaves * kFew * D * 4);  // [wave][16 rows][max, sum]
  __shared__ int s_last[kFew], s_row[kFew];

  // A tile has the heads of whole tokens, or up to 16 of one token's.
  const int each = a.each, pieces = a.pieces;
  for (; pieces == 1 ? sh.tile * each < sh.members : sh.tile < sh.members * pieces; sh.tile += sh.step) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int c = lane & 15, g = lane >> 4;
    const int whole = a.by_pieces(sh.tile);
    const int token0 = sh.first + whole * each, head0 = (sh.tile - whole * pieces) * kFew;
    const int here = min(each, sh.first + sh.members - token0);  // tokens of the tile
    const int rows = here * min(G - head0, kFew);
    const auto token_of = [&](int row) { return token0 + (pieces == 1 ? a.by_group(row) : 0); };
    const auto head_of = [&](int row) { return sh.kvh * G + (pieces == 1 ? row - a.by_group(row) * G : head0 + row); };
    const auto row_any = [&](int j) -> unsigned {
      j = min(j, end - 1);
      return (static_cast<unsigned>(block_at(sh.table[bshift >= 0 ? j >> bshift : j / bs])) * a.kv_heads + sh.kvh) * bs +
             (bshift >= 0 ? j & (bs - 1) : j % bs);
    };
    // SCALAR: the table entries of the two 16-key runs of a step, looked up a step ahead. The first
    // run may begin before `begin`, whose slots may hold anything: rows are clamped at both ends.
    int entry[2];
    const auto run_of = [&](int k0, int t) { return min(k0 + 16 * t, (end - 1) & ~15); };
    const auto lookup = [&](int k0) {
      if (SCALAR) entry[0] = entries[run_of(k0, 0) >> bshift], entry[1] = entries[run_of(k0, 1) >> bshift];
    };
    const auto issue = [&](KvStep<D, DR>& st, int k0) {
      const auto row_of = [&](int t, int off) -> unsigned {
        const int r0 = run_of(k0, t);
        return (static_cast<unsigned>(block_at(entry[t])) * a.kv_heads + sh.kvh) * bs + (r0 & (bs - 1)) + min(max(off, begin - r0), end - 1 - r0);
      };
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const half_t* const at = a.kpool + static_cast<int64_t>(SCALAR ? row_of(t, c) : row_any(k0 + 16 * t + c)) * DR;
#pragma unroll
        for (int h = 0; h < KH; ++h) {
          if (DR == D || 32 * h + 8 * g < DR) {
            st.k[t][h] = load_half8(at + 32 * h + 8 * g);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) st.k[t][h][e] = 0;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int kl = VKEYS * i;  // first key of the load
        const half_t* const at = a.vpool + static_cast<int64_t>(SCALAR ? row_of(kl >> 4, (kl & 15) + lane / CH) : row_any(k0 + kl + lane / CH)) * DR;
        if (DR == D || 8 * (lane % CH) < DR) {
          // Own V is read once, by one workgroup: non-temporal (64 x 1000 own keys at head size 128 46 -> 39 us,
          // 45 x 700 beside 5 x 1504 33 -> 30; K too 44, 33).
          st.v[i] = __builtin_bit_cast(half8, __builtin_nontemporal_load(reinterpret_cast<const uint4v*>(at + 8 * (lane % CH))));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) st.v[i][e] = 0;
        }
      }
      lookup(k0 + kWaves * kStep);
    };

    const bool on = c < rows;
    const int token = token_of(on ? c : 0), head = head_of(on ? c : 0);
    int k0 = (SCALAR ? begin & ~15 : begin) + w * kStep;
    KvStep<D, DR> ahead[2];
    lookup(k0);
    if (k0 < end) issue(ahead[0], k0);
    const int4 m = a.meta[token];
    // For the join, a thread for each token of the tile: how many slices it has, and its row.
    int slices = 0;
    if (JOIN && static_cast<int>(threadIdx.x) < here) {
      const int4 mt = a.meta[token0 + threadIdx.x];
      s_row[threadIdx.x] = mt.x;
      if (mt.y > 0)
        slices = parts_of(mt.w, a.by_shared_slice, a.shared_parts) + parts_of(mt.y - max(mt.w, 0), a.by_own_slice, a.own_parts);
    }
    const int lim = on ? min(m.y, end) : end;
    half8 qb[KH];
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      if (on && m.y > 0 && (DR == D || 32 * h + 8 * g < DR)) {
        qb[h] = load_half8(a.q + m.x * a.q_stride + static_cast<int64_t>(head) * DR + 32 * h + 8 * g);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) qb[h][e] = 0;
      }
    }
    float ref = -INFINITY, l = 0.0f;
    float4v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};

    const auto compute = [&](const KvStep<D, DR>& st) {
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int kl = VKEYS * i + lane / CH;
        *reinterpret_cast<half8*>(sv + kl * D + (((lane % CH) ^ vswz<D>(kl)) << 3)) = st.v[i];
      }
      float x[8], mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float4v s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < KH; ++h) s = mfma16x16x32(st.k[t][h], qb[h], s);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = k0 + 16 * t + 4 * g + e;
          x[4 * t + e] = key >= begin && key < lim ? s[e] * a.scale_log2 : -INFINITY;
          mx = fmaxf(mx, x[4 * t + e]);
        }
      }
      mx = group4_max(mx);
      mx = fmaxf(ref, fabsf(mx) < 1048576.0f ? mx - kUp : mx);  // (2^20: past it kUp comes to be lost in rounding)
      const float base = mx == -INFINITY ? 0.0f : mx, alpha = fast_exp2(ref - base);
      ref = mx;
      half8 p;
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = fast_exp2(x[e] - base);
        sum += y;
        p[e] = static_cast<half_t>(y);
      }
      l = l * alpha + sum;
      wave_fence();
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        // A transposing read gives lane c of group g rows kr .. kr + 3 of column 16 i + c.
        const int col = 16 * i + 4 * (c & 3), kr = 4 * g + (c >> 2);
        const half4 lo = tr_read_b64(sv + kr * D + (((col >> 3) ^ vswz<D>(kr)) << 3) + (col & 7));
        const half4 hi = tr_read_b64(sv + (kr + 16) * D + (((col >> 3) ^ vswz<D>(kr + 16)) << 3) + (col & 7));
        float4v acc = o[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] *= alpha;
        o[i] = mfma16x16x32(half8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, p, acc);
      }
      wave_fence();
    };
    while (k0 < end) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (k0 < end) {
          if (k0 + kWaves * kStep < end) issue(ahead[1 - i], k0 + kWaves * kStep);
          __builtin_amdgcn_sched_barrier(0);  // the next step's loads before this one's arithmetic
          compute(ahead[i]);
          k0 += kWaves * kStep;
        }
      }
    }
    l = group4_sum(l);

    // The waves' rows meet in LDS (row c rotated by 4 c floats against bank conflicts).
    __syncthreads();
    float* const so = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) so[(w * kFew + c) * D + ((16 * i + 4 * g + 4 * c) & (D - 1)) + e] = o[i][e];
    if (g == 0) s_ml[2 * (w * kFew + c)] = ref, s_ml[2 * (w * kFew + c) + 1] = l;
    __syncthreads();
    const int most = a.shared_parts + a.own_parts;
    for (int i = threadIdx.x; i < rows * DR; i += kThreads) {
      const int row = i / DR, d = i % DR;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < kWaves; ++j) top = fmaxf(top, s_ml[2 * (j * kFew + row)]);
      const float base = top == -INFINITY ? 0.0f : top;
      float L = 0.0f, O = 0.0f;
#pragma unroll
      for (int j = 0; j < kWaves; ++j) {
        const float f = fast_exp2(s_ml[2 * (j * kFew + row)] - base);
        L += f * s_ml[2 * (j * kFew + row) + 1];
        O += f * so[(j * kFew + row) * D + ((d + 4 * row) & (D - 1))];
      }
      const int64_t at = (static_cast<int64_t>(token_of(row)) * a.heads + head_of(row)) * most + sh.part;
      if (JOIN) {
        coherent_store(a.part_o + at * DR + d, O);
        if (d == 0) coherent_store(a.part_ml + 2 * at, top), coherent_store(a.part_ml + 2 * at + 1, L);
      } else {
        a.part_o[at * DR + d] = O;  // an idle token's are never read
        if (d == 0) reinterpret_cast<float2*>(a.part_ml)[at] = float2{top, L};
      }
    }
    if constexpr (JOIN) {
      // The last workgroup of a token's slices to come joins them. Its own stores are done before the
      // barrier, so before it counts itself; the values travel by coherent stores and loads.
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < here) {
        int last = 0;
        if (slices) {
          int* const count = a.counters + (static_cast<int64_t>(token0 + threadIdx.x) * a.kv_heads + sh.kvh) * a.counter_step;
          if (__hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == pieces * slices - 1) {
            last = slices;
            __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
        }
        s_last[threadIdx.x] = last;
      }
      __syncthreads();
      // Two values a thread, slices' loads kMerge at a time.
      for (int i = threadIdx.x; i < here * G * (DR / 2); i += kThreads) {
        const int row = i / (DR / 2), t = pieces == 1 ? a.by_group(row) : 0, d = 2 * (i % (DR / 2)), hd = sh.kvh * G + row - t * G;
        const int parts = s_last[t];
        if (!parts) continue;
        const int64_t at = (static_cast<int64_t>(token0 + t) * a.heads + hd) * most;
        float M = -INFINITY, L = 0.0f, O0 = 0.0f, O1 = 0.0f;
        for (int p0 = 0; p0 < parts; p0 += kMerge) {
          float2 ml[kMerge], ov[kMerge];
          float top = M;
#pragma unroll
          for (int j = 0; j < kMerge; ++j) {
            if (p0 + j < parts) {
              ml[j] = coherent_load2(a.part_ml + 2 * (at + p0 + j));
              ov[j] = coherent_load2(a.part_o + (at + p0 + j) * DR + d);
            }
          }
#pragma unroll
          for (int j = 0; j < kMerge; ++j)
            if (p0 + j < parts) top = fmaxf(top, ml[j].x);
          const float base = top == -INFINITY ? 0.0f : top, keep = fast_exp2(M - base);
          L *= keep, O0 *= keep, O1 *= keep;
#pragma unroll
          for (int j = 0; j < kMerge; ++j) {
            if (p0 + j < parts) {
              const float f = fast_exp2(ml[j].x - base);
              L += f * ml[j].y;
              O0 += f * ov[j].x;
              O1 += f * ov[j].y;
            }
          }
          M = top;
        }
        half_t* const out = a.out + s_row[t] * a.out_stride + static_cast<int64_t>(hd) * DR + d;
        out[0] = static_cast<half_t>(O0 / L);
        out[1] = static_cast<half_t>(O1 / L);
      }
    }
    __syncthreads();
  }
}

// D: compute width, DR: head size of the rows (16 runs at width 32 with zeros behind). SCALAR: the
// block size is a power of two >= 16, so 16 keys from a multiple of 16 on lie in one block. ROWS: prefixes
// have many rows.
template <int D, int DR, bool SCALAR, bool ROWS>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(D > 64 ? 2 : 3, D > 64 ? 2 : 4))) void shared_attention_kernel(
    const SharedArgs a) {
  constexpr int FEW = kWaves * kFew * (D * 4 + 8), RING = ROWS ? kRing * 2 * kStep * D * 2 : 0;
  __shared__ __attribute__((aligned(16))) char smem[std::max(FEW, RING)];
  static_assert(kWaves * kStep * D * 2 <= FEW && (!ROWS || kWaves * kStrip * D * 4 <= RING), "staging and hand-over fit");

  // The arguments at once: the compiler loads them where they are used, one wait after another (32 members on 2048
  // keys 16.4 -> 16.15 us; in the join 16.15 -> 15.75).
  asm volatile("" : : "s"(a.q), "s"(a.tables), "s"(a.kv_heads), "s"(a.shared_slice), "s"(a.tiles), "s"(a.each), "s"(a.by_own_parts.m), "s"(a.by_shared_parts.m), "s"(a.by_kv_heads.m),
               "s"(a.by_own_slice.m), "s"(a.by_shared_slice.m), "s"(a.scale_log2), "s"(a.counters), "s"(a.part_o), "s"(a.out_stride));
  // Workgroups go round the 8 XCDs; the row tiles of one slice share an XCD, whose L2 then holds its K and V.
  const bool shared = blockIdx.x < static_cast<unsigned>(a.shared_wgs);
  int shared_units = a.shared_units, own_units = a.own_units;
  asm volatile("" : "+s"(shared_units), "+s"(own_units));  // both loaded with the rest, not one when it is known which
  int b = shared ? blockIdx.x : blockIdx.x - a.shared_wgs;
  Share g;
  g.step = shared ? a.tiles : a.own_tiles;
  const int over = shared ? a.by_tiles(b >> 3) : a.by_own_tiles(b >> 3);
  g.tile = (b >> 3) - over * g.step;
  b = over * 8 + (b & 7);
  if (b >= (shared ? shared_units : own_units)) return;
  if (shared) {
    const int head = a.by_shared_parts(b), group = a.by_kv_heads(head);
    g.part = b - head * a.shared_parts;
    g.kvh = head - group * a.kv_heads;
    const int4 rec = a.groups[group];
    const int parts = parts_of(rec.z, a.by_shared_slice, a.shared_parts);
    if (g.part >= parts) return;
    g.first = rec.x, g.members = rec.y, g.table = a.tables + rec.w;
    g.begin = g.part * a.shared_slice;
    g.end = g.part == parts - 1 ? rec.z : g.begin + a.shared_slice;
    if constexpr (ROWS) {
      attend_rows<D>(a, g, smem);
      return;
    }
  } else {
    const int head = a.by_own_parts(b);
    g.part = b - head * a.own_parts;
    g.first = a.by_kv_heads(head), g.members = 1;
    g.kvh = head - g.first * a.kv_heads;
    const int4 m = a.meta[g.first];
    const int from = max(m.w, 0), parts = parts_of(m.y - from, a.by_own_slice, a.own_parts);
    if (g.part >= parts) return;
    g.table = a.tables + m.z;
    g.begin = from + g.part * a.own_slice;
    g.end = g.part == parts - 1 ? m.y : g.begin + a.own_slice;
    g.part += parts_of(m.w, a.by_shared_slice, a.shared_parts);
  }
  attend_few<D, DR, SCALAR, !ROWS>(a, g, smem);
}

// Joins a row's slices, a lane for each value. LANES slices' maxima and sums come at once, one a lane, and
// kJoin slices' values.
constexpr int kJoin = 16;
template <int D>
__global__ __launch_bounds__(256) void shared_join_kernel(const SharedArgs a) {
  constexpr int LANES = D < kWave ? D : kWave;
  asm volatile("" : : "s"(a.meta), "s"(a.n_dec), "s"(a.shared_parts), "s"(a.by_heads.m), "s"(a.by_own_slice.m), "s"(a.by_shared_slice.m), "s"(a.part_o),
               "s"(a.out_stride));  // as above
  const int row = blockIdx.x * (256 / D) + threadIdx.x / D, d = threadIdx.x % D, lane = threadIdx.x % LANES;
  if (row >= a.n_dec * a.heads) return;
  const int token = a.by_heads(row), head = row - token * a.heads;
  const int4 m = a.meta[token];
  if (m.y <= 0) return;
  const int most = a.shared_parts + a.own_parts;
  const int parts = parts_of(m.w, a.by_shared_slice, a.shared_parts) + parts_of(m.y - max(m.w, 0), a.by_own_slice, a.own_parts);
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + static_cast<int64_t>(row) * most;
  const float* o = a.part_o + static_cast<int64_t>(row) * most * D + d;
  float M = -INFINITY, L = 0.0f, O = 0.0f;
  for (int p0 = 0; p0 < parts; p0 += LANES) {
    const int n = min(LANES, parts - p0);
    float v[kJoin];
#pragma unroll
    for (int j = 0; j < kJoin; ++j)
      if (j < n) v[j] = o[static_cast<int64_t>(p0 + j) * D];
    const float2 mine = lane < n ? ml[p0 + lane] : float2{-INFINITY, 0.0f};
    float top = mine.x;
#pragma unroll
    for (int e = LANES / 2; e > 0; e >>= 1) top = fmaxf(top, __shfl_xor(top, e));
    top = fmaxf(top, M);
    const float base = top == -INFINITY ? 0.0f : top;
    const float f = fast_exp2(mine.x - base), keep = fast_exp2(M - base);
    float l = f * mine.y;
#pragma unroll
    for (int e = LANES / 2; e > 0; e >>= 1) l += __shfl_xor(l, e);
    L = L * keep + l;
    O *= keep;
    M = top;
    for (int j0 = 0; j0 < n; j0 += kJoin) {
#pragma unroll
      for (int j = 0; j < kJoin; ++j)
        if (j0 + j < n) O += __shfl(f, j0 + j, LANES) * v[j];
#pragma unroll
      for (int j = 0; j < kJoin; ++j)
        if (j0 + kJoin + j < n) v[j] = o[static_cast<int64_t>(p0 + j0 + kJoin + j) * D];
    }
  }
  a.out[m.x * a.out_stride + static_cast<int64_t>(head) * D + d] = static_cast<half_t>(O / L);
}

template <int D, int DR>
int launch(const SharedArgs& a, bool rows, int64_t wgs, hipStream_t s) {
  const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(wgs)), dim3(kThreads), 0, s, a); };
  if constexpr (D == DR) {
    if (rows) {
      RH_TRY_LAUNCH(go(shared_attention_kernel<D, DR, true, true>));
      return 0;
    }
  }
  if (a.bs_shift >= 4) {
    RH_TRY_LAUNCH(go(shared_attention_kernel<D, DR, true, false>));
  } else {
    RH_TRY_LAUNCH(go(shared_attention_kernel<D, DR, false, false>));
  }
  return 0;
}

// The counters have a fixed place at the workspace's start, so that they stay zero between calls of any shape.
constexpr int kCounters = 65536;
constexpr int kMostKeys = 1 << 30;

struct Plan {
  bool rows;
  int shared_slice, shared_parts, own_slice, own_parts, tiles, own_tiles;
};

Plan plan_of(int n_dec, int n_groups, int max_members, int max_shared, int max_own, int heads, int kv_heads, int head_dim,
             int block) {
  const int group = heads / kv_heads;
  max_members = std::min(max_members, n_dec);  // a group has no more, whatever the caller allows for
  const int64_t rows = static_cast<int64_t>(max_members) * group;
  Plan p{};
  // Shared tiles come in pieces of up to 16 keys of one block, straight to LDS.
  const bool pieces = head_dim > 16 && block >= 16 && (block & (block - 1)) == 0;
  // Few rows on a short prefix are joined by the last workgroup that comes, which saves a launch; a long
  // one has more slices than one workgroup joins well, and many values take it long. Measured (us, so / as
  // many rows): 6 rows on 512 keys at head size 64 7.7 / 10.2, 15 there 9.4 / 10.4; 12 on 512 at head size
  // 128 12.4 / 12.6, 16 there 13.9 / 12.8; 8 on 4096 at 128 21 / 18; 24 on 1024 at 64 13.6 / 11.3.
  p.rows = pieces && (rows > kFew || rows * head_dim > 1536 || max_shared > 1024);
  const int each = std::max(1, kFew / group), pieces_of = (group + kFew - 1) / kFew;
  const int64_t tiles = p.rows ? (rows + kWaves * kStrip - 1) / (kWaves * kStrip) : (static_cast<int64_t>(max_members) + each - 1) / each * pieces_of;
  p.tiles = static_cast<int>(std::min<int64_t>(std::max<int64_t>(1, tiles), 1 << 20));
  p.own_tiles = pieces_of;
  const double held = 256.0 * (head_dim > 64 ? 2 : 3);  // workgroups that the card holds
  const int64_t own_units = static_cast<int64_t>(n_dec) * kv_heads * p.own_tiles;
  const int64_t shared_units = static_cast<int64_t>(n_groups) * kv_heads * p.tiles;
  const auto slice_of = [](int keys, int want) {
    return static_cast<int>((static_cast<int64_t>(keys) + static_cast<int64_t>(want) * kLeast - 1) / (static_cast<int64_t>(want) * kLeast)) * kLeast;
  };
  const auto put = [&](int keys, int size, int* slice, int* parts) {
    *slice = std::max(size, kLeast), *parts = size < kLeast ? 1 : (keys + size - 1) / size;
  };
  if (p.rows) {
    // Both kinds' slices together, by what the call then takes (us): a start and the steps of either; all of
    // them in the card's places, and half a last one; no less than their bytes; each slice's way through memory to
    // its join. (Own lengths spread below the largest.) Constants from timings of every cut of 30 shapes; the cut that the
    // rule takes is 1.5% from the best on average, 8% at worst. Two rules, each for its own kind alone, took 8%: 4 x 8 members
    // on 2000 keys with 300 of their own (32/8 heads of 128), 16 slices and 2 own 32 us, 8 and 1 23; 64 on 16,384
    // with 1000, 13 and 1 64 us, 32 and 1 86.
    const double step = head_dim > 64 ? 0.75 : 0.6, own_step = head_dim > 64 ? 1.2 : 0.75, spread = 0.72;
    const double bytes = (static_cast<double>(n_groups) * max_shared + spread * n_dec * max_own) * kv_heads * head_dim * 4;
    const double part = static_cast<double>(n_dec) * heads * head_dim * 8 / 1.9e6;
    double best = 0.0;
    for (const int want : {1, 2, 3, 4, 5, 6, 8, 10, 11, 13, 16, 19, 22, 26, 32, 43, 64}) {
      const int size = slice_of(max_shared, want), n = size < kLeast ? 1 : (max_shared + size - 1) / size;
      const double time = 4.8 + step * size / kStep;
      for (const int own_want : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
        const int own_size = slice_of(max_own, own_want), own_n = own_size < kLeast ? 1 : (max_own + own_size - 1) / own_size;
        const double own_time = 5.2 + own_step * std::min(own_size, max_own) / kLeast;
        const double own_mean = 5.2 + own_step * std::min<double>(own_size, spread * max_own) / kLeast;
        const double places = (static_cast<double>(shared_units) * n + static_cast<double>(own_units) * own_n) / held;
        const double work = (shared_units * n * time + 0.57 * own_units * own_n * own_mean) / held + (places > 1.0 ? 0.5 * own_time : 0.0);
        const double cost = std::max({time, own_time, work, bytes / 6.6e6}) + part * (n + own_n);
        if (best == 0.0 || cost < best) {
          best = cost;
          put(max_shared, size, &p.shared_slice, &p.shared_parts);
          put(max_own, own_size, &p.own_slice, &p.own_parts);
        }
        if (own_size <= kLeast) break;
      }
      if (size <= kLeast) break;
    }
    return p;
  }
  // Few rows: each kind by its own time, and what its slices cost the workgroup that joins them (us: a start of 5, a step of
  // 128 keys 1.5 at head size 128 and 0.8 below, in rounds of the card's places).
  const auto cut = [&](int64_t units, int keys, int64_t rows_joined, int* slice, int* parts) {
    const double part = 0.09 * std::max(1.0, std::min<int64_t>(rows_joined, kFew) * head_dim / 256.0);
    double best = 0.0;
    put(keys, 0, slice, parts);
    for (int want = 1; want <= 64; ++want) {
      const int size = slice_of(keys, want);
      if (size < kLeast) break;
      const int n = (keys + size - 1) / size;
      const double rounds = static_cast<double>(units) * n / held;  // a last one is rarely full
      const double cost = (5.0 + (head_dim > 64 ? 1.5 : 0.8) * size / kLeast) * (rounds <= 1.0 ? 1.0 : rounds + 0.5) + part * n;
      if (want == 1 || cost < best) best = cost, *slice = size, *parts = n;
      if (size == kLeast) break;
    }
  };
  cut(own_units, max_own, group, &p.own_slice, &p.own_parts);
  cut(shared_units, max_shared, rows, &p.shared_slice, &p.shared_parts);
  return p;
}

size_t bytes_of(const Plan& p, int n_dec, int heads, int head_dim) {
  return kCounters * 4 + static_cast<size_t>(n_dec) * heads * (p.shared_parts + p.own_parts) * (head_dim + 2) * 4;
}

}  // namespace
}  // namespace relay_hip

using namespace relay_hip;

extern "C" int rh_shared_prefix_pays(int n_dec, int max_shared, int max_own, int heads, int kv_heads, int head_dim) {
  // One token shares nothing.
  if (n_dec < 2 || max_shared <= 0 || max_own < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
  // The decode kernel reads each token's keys, once for each 16 query heads of a kv head (at head size 32 the caches hide
  // that); here a prefix is read once, but own keys take some 10% longer and most calls a second launch. So sharing pays where
  // the readings saved, less what own keys lose, pass a number of bytes, fewer where there are many workgroups. Measured (us,
  // decode / shared; members x shared + own; MB saved): 32/8 heads of 128, 4 x 4096 + 304 (50) 15.2 / 19.0, 16 x 1024 + 200 (63) 14.3 /
  // 15.5, 24 x 1024 + 100 (96) 21 / 16, 32 x 1024 + 300 (130) 28 / 20, 48 x 1024 + 4000 98 / 108 and 105 / 108 with 256 shared; 32/4 of 64, 32 x
  // 1024 + 300 (32) 10.3 / 13.1, 48 x 1024 + 1000 (49) 19 / 17, 48 x 4096 + 16,000 113 / 114; 9/3 of 64, 104 tokens on 672 + 13 (53) 18.3 / 11.2.
  // Of 1500 shapes with groups of three and more members the rule makes 33 slower, by 5% on average and 25% at worst, and leaves
  // 180 that sharing would make faster by 12% on average; of 460 with groups of two, which save half, 19 slower, 24% at worst.
  const int group = heads / kv_heads;
  const double pieces = head_dim >= 64 ? (group + 15) / 16 : 1, units = pieces * n_dec * kv_heads;
  const double saved = 4.0 * head_dim * kv_heads * pieces * ((n_dec - 1.0) * max_shared - 0.26 * (n_dec + 4.0) * max_own);
  if (saved > (units >= 192 ? 45e6 : 70e6)) return 1;
  // Few workgroups of wide kv heads merge their slices slowly there: 16/1 of 128, 2 x 2048 + 40 18.3 / 13.7, 2 x 4096 + 100 23 / 16,
  // 16 x 4096 + 100 23.5 / 18.3, but 16 x 1024 + 300 13.1 / 14.2, 64 x 512 + 100 13.6 / 15.3; 32/2, 16 x 2048 + 40 16.0 / 17.3.
  return head_dim == 128 && group * head_dim > 1024 && max_shared >= 2000 && units <= 24;
}

extern "C" int rh_shared_prefix_groups(const int* tokens, const int* tables, int n_dec, int block_size, int min_shared,
                                       int* dec_meta, int* groups, int* limits) {
  RH_REQUIRE(n_dec >= 0 && block_size > 0 && min_shared >= 0, "shared prefix groups: bad sizes");
  RH_REQUIRE(limits && (n_dec == 0 || (tokens && tables && dec_meta && groups)), "shared prefix groups: missing pointer");
  limits[0] = limits[1] = limits[2] = 0;
  try {
    // Tokens in the order of their tables' whole blocks; neighbours then share the most.
    std::vector<int> order(n_dec);
    for (int i = 0; i < n_dec; ++i) order[i] = i;
    const auto blocks = [&](int i) { return std::max(0, tokens[4 * i + 1]) / block_size; };
    const auto table = [&](int i) { return tables + tokens[4 * i + 2]; };
    std::stable_sort(order.begin(), order.end(), [&](int x, int y) {
      return std::lexicographical_compare(table(x), table(x) + blocks(x), table(y), table(y) + blocks(y));
    });
    std::vector<int> alike(n_dec, 0);  // whole blocks that a token shares with the one before it
    for (int i = 1; i < n_dec; ++i) {
      const int n = std::min(blocks(order[i - 1]), blocks(order[i]));
      alike[i] = static_cast<int>(std::mismatch(table(order[i]), table(order[i]) + n, table(order[i - 1])).first - table(order[i]));
    }
    // Runs of neighbours that save the most reads, (members - 1) * shared blocks each.
    std::vector<int64_t> saved(n_dec + 1, 0);
    std::vector<int> from(n_dec + 1, 0);
    const int least = std::max(1, (min_shared + block_size - 1) / block_size);
    for (int end = 1; end <= n_dec; ++end) {
      saved[end] = saved[end - 1];
      from[end] = end - 1;
      int common = INT32_MAX;
      for (int first = end - 2; first >= 0; --first) {
        common = std::min(common, alike[first + 1]);
        if (common < least) break;
        const int64_t with = saved[first] + static_cast<int64_t>(end - first - 1) * common;
        if (with > saved[end]) saved[end] = with, from[end] = first;
      }
    }
    std::vector<int> ends;
    for (int end = n_dec; end > 0; end = from[end]) ends.push_back(end);
    int n_groups = 0;
    for (std::size_t e = ends.size(); e-- > 0;) {
      const int end = ends[e], first = from[end], members = end - first;
      int common = members > 1 ? INT32_MAX : 0;
      for (int i = first + 1; i < end; ++i) common = std::min(common, alike[i]);
      const int shared = common * block_size;
      for (int i = first; i < end; ++i) {
        const int* t = tokens + 4 * order[i];
        const int meta[4] = {t[0], t[1], t[2], shared};
        std::copy(meta, meta + 4, dec_meta + 4 * i);
        limits[2] = std::max(limits[2], t[1] - shared);
      }
      if (members == 1) continue;
      const int record[4] = {first, members, shared, tokens[4 * order[first] + 2]};
      std::copy(record, record + 4, groups + 4 * n_groups++);
      limits[0] = std::max(limits[0], members);
      limits[1] = std::max(limits[1], shared);
    }
    return n_groups;
  } catch (const std::exception& e) {
    set_error(std::string("shared prefix groups: ") + e.what());
    return -1;
  }
}

extern "C" size_t rh_shared_prefix_workspace(int n_dec, int n_groups, int max_members, int max_shared, int max_own, int heads,
                                             int kv_heads, int head_dim) {
  if (n_dec <= 0 || n_groups < 0 || max_members < 0 || max_shared < 0 || max_own < 0 || max_shared > kMostKeys || max_own > kMostKeys || kv_heads <= 0 || heads <= 0 ||
      heads % kv_heads || head_dim <= 0)
    return 0;
  size_t most = 0;  // enough for any block size
  for (const int block : {1, 16})
    most = std::max(most, bytes_of(plan_of(n_dec, n_groups, max_members, max_shared, max_own, heads, kv_heads, head_dim, block), n_dec, heads, head_dim));
  return most;
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
  RH_REQUIRE(static_cast<int64_t>(n_dec) * kv_heads <= kCounters, "shared prefix attention: n_dec * kv_heads must be at most 65536");
  RH_REQUIRE(max_shared <= kMostKeys && max_own <= kMostKeys, "shared prefix attention: at most 2^30 keys");
  RH_REQUIRE(scale > 0.0f && scale * 1.4426950408889634f < INFINITY, "shared prefix attention: scale must be positive");
  RH_REQUIRE(q && kpool && vpool && dec_meta && tables && out && (groups || n_groups == 0),
             "shared prefix attention: missing pointer");
  RH_REQUIRE(q_row_stride % 8 == 0 && out_row_stride >= static_cast<int64_t>(heads) * head_dim,
             "shared prefix attention: q rows must be 16-byte aligned and out rows hold heads * head_dim");
  RH_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kpool) | reinterpret_cast<uintptr_t>(vpool) |
              reinterpret_cast<uintptr_t>(dec_meta) | reinterpret_cast<uintptr_t>(groups)) % 16 == 0,
             "shared prefix attention: q, the pools, dec_meta and groups must be 16-byte aligned");
  const Plan p = plan_of(n_dec, n_groups, max_members, max_shared, max_own, heads, kv_heads, head_dim, block_size);
  const size_t need = bytes_of(p, n_dec, heads, head_dim);
  RH_REQUIRE(workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
             "shared prefix attention: needs a 16-byte aligned workspace of rh_shared_prefix_workspace bytes");
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
  a.counters = static_cast<int*>(workspace);
  // In lines of their own while there is room: counts in one line are taken one after another.
  a.counter_step = std::min(32, kCounters / (n_dec * kv_heads));
  a.part_o = static_cast<float*>(workspace) + kCounters;
  a.part_ml = a.part_o + static_cast<size_t>(n_dec) * heads * (p.shared_parts + p.own_parts) * head_dim;
  a.out = static_cast<half_t*>(out);
  a.out_stride = out_row_stride;
  const int64_t shared_units = static_cast<int64_t>(n_groups) * kv_heads * p.shared_parts;
  const int64_t own_units = static_cast<int64_t>(n_dec) * kv_heads * p.own_parts;
  const int64_t shared_wgs = (shared_units + 7) / 8 * 8 * p.tiles, own_wgs = (own_units + 7) / 8 * 8 * p.own_tiles;
  const int64_t wgs = shared_wgs + own_wgs;
  RH_REQUIRE(wgs < (int64_t{1} << 31) && static_cast<int64_t>(n_dec) * heads < (int64_t{1} << 31), "shared prefix attention: too large");
  a.shared_units = static_cast<int>(shared_units);
  a.own_units = static_cast<int>(own_units);
  a.shared_wgs = static_cast<int>(shared_wgs);
  a.each = std::max(1, kFew / a.group);
  a.pieces = (a.group + kFew - 1) / kFew;
  a.by_tiles = div_by(p.tiles);
  a.by_own_tiles = div_by(p.own_tiles);
  a.by_shared_parts = div_by(p.shared_parts);
  a.by_own_parts = div_by(p.own_parts);
  a.by_kv_heads = div_by(kv_heads);
  a.by_shared_slice = div_by(p.shared_slice / kLeast);
  a.by_own_slice = div_by(p.own_slice / kLeast);
  a.by_group = div_by(a.group);
  a.by_pieces = div_by(a.pieces);
  a.by_heads = div_by(heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (head_dim) {
    case 16: if (int rc = launch<32, 16>(a, p.rows, wgs, s)) return rc; break;
    case 32: if (int rc = launch<32, 32>(a, p.rows, wgs, s)) return rc; break;
    case 64: if (int rc = launch<64, 64>(a, p.rows, wgs, s)) return rc; break;
    default: if (int rc = launch<128, 128>(a, p.rows, wgs, s)) return rc;
  }
  if (!p.rows) return 0;  // (as always at head size 16)
  const int64_t values = static_cast<int64_t>(n_dec) * heads * head_dim;
  const auto join = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((values + 255) / 256)), dim3(256), 0, s, a);
  };
  switch (head_dim) {
    case 32: RH_TRY_LAUNCH(join(shared_join_kernel<32>)); break;
    case 64: RH_TRY_LAUNCH(join(shared_join_kernel<64>)); break;
    default: RH_TRY_LAUNCH(join(shared_join_kernel<128>));
  }
  return 0;
}
