// The operators of a decode step that stays on the GPU, around its attention: block tables and
// slot maps from the request lengths, the norm of q and k per head with the rotation and the
// cache write, and penalties, biases, grammar masks and the greedy token on the logits. relay
// does the first and the last on the host (engine.cpp, sampler.cpp) and has no norm of q and k.
#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/relay_hip.h"
#include "common.h"

namespace relay_hip {
namespace {

// ---- block tables and slot maps --------------------------------------------------------------
//
// held = ceil(cached / B), want = ceil((cached + fresh) / B); sequence s takes want - held ids off the
// top of the free stack, behind those of the sequences before it, and has the rows row_off[s] ..
// row_off[s + 1] - 1. Two exclusive sums over the sequences, then one row after another by binary
// search. One workgroup does all of it: the sums are a chain of dependent steps, and a second
// launch costs more than the rows of a decode step.

constexpr int kTableThreads = 1024;
constexpr int kSumCap = (1 << 30) - 1;  // sums stop here, past every limit that they are compared with

struct StepArgs {
  const int *cached, *fresh, *shared, *group_seqs;
  int n_seqs, n_groups, block;
  int* tables;
  int stride;
  const int *free_blocks, *free_count;
  int max_rows;
  int *row_off, *last_row, *table_off, *pos, *seq, *slot;
  int4 *meta, *groups;
  int* totals;
};

__device__ __forceinline__ int capped_add(int a, int b) { return min(a + b, kSumCap); }
__device__ __forceinline__ int blocks_of(int keys, int block) { return (keys + block - 1) / block; }

struct Need {
  int rows, blocks;
};

// Inclusive sums over the workgroup and the workgroup's total.
__device__ Need block_scan(Need v, Need* waves, Need* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int r = __shfl_up(v.rows, o), b = __shfl_up(v.blocks, o);
    if (lane >= o) v.rows = capped_add(v.rows, r), v.blocks = capped_add(v.blocks, b);
  }
  if (lane == 63) waves[w] = v;
  __syncthreads();
  Need sum = {0, 0}, before = {0, 0};
  for (int i = 0; i < kTableThreads / 64; ++i) {
    if (i == w) before = sum;
    sum.rows = capped_add(sum.rows, waves[i].rows);
    sum.blocks = capped_add(sum.blocks, waves[i].blocks);
  }
  __syncthreads();
  *total = sum;
  return {capped_add(before.rows, v.rows), capped_add(before.blocks, v.blocks)};
}

// Row t of the step (a row past the last is idle: no slot, an empty context).
__device__ void fill_row(const StepArgs& a, int t, int total) {
  if (t >= total) {
    a.pos[t] = 0;
    a.seq[t] = 0;
    a.slot[t] = -1;
    a.meta[t] = int4{t, 0, 0, 0};
    return;
  }
  int lo = 0, hi = a.n_seqs;  // the last s with row_off[s] <= t that has rows
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.row_off[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  const int p = a.cached[lo] + t - a.row_off[lo];
  const int off = lo * a.stride;
  a.pos[t] = p;
  a.seq[t] = lo;
  a.slot[t] = a.tables[off + p / a.block] * a.block + p % a.block;
  a.meta[t] = int4{t, p + 1, off, a.shared ? a.shared[lo] : 0};
}

__global__ __launch_bounds__(kTableThreads) void step_tables_kernel(const StepArgs a) {
  __shared__ Need waves[kTableThreads / 64];
  __shared__ int s_bad;
  const int free = *a.free_count;
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  // The sums and checks of the whole step come first: a step that does not fit changes nothing.
  int bad = free < 0 ? RH_STEP_BAD_LENGTH : 0;
  Need all = {0, 0};
  for (int base = 0; base < a.n_seqs; base += kTableThreads) {
    const int s = base + threadIdx.x;
    Need n = {0, 0}, total;
    if (s < a.n_seqs) {
      const int c = a.cached[s], f = a.fresh[s];
      if (c < 0 || f < 0 || c > kSumCap || f > kSumCap - c || (a.shared && a.shared[s] < 0)) {
        bad |= RH_STEP_BAD_LENGTH;
      } else {
        const int held = blocks_of(c, a.block), want = blocks_of(c + f, a.block);
        if (want > a.stride) bad |= RH_STEP_TABLE_FULL;
        n = {f, want - held};
      }
    }
    block_scan(n, waves, &total);
    all.rows = capped_add(all.rows, total.rows);
    all.blocks = capped_add(all.blocks, total.blocks);
  }
  for (int g = threadIdx.x; g < a.n_groups; g += kTableThreads) {
    const int first = a.group_seqs[2 * g], count = a.group_seqs[2 * g + 1];
    if (first < 0 || count < 0 || first > a.n_seqs || count > a.n_seqs - first) bad |= RH_STEP_BAD_LENGTH;
  }
  if (all.rows > a.max_rows) bad |= RH_STEP_ROWS_FULL;
  if (all.blocks > free) bad |= RH_STEP_NO_BLOCKS;
  if (bad) atomicOr(&s_bad, bad);
  __syncthreads();
  const int status = s_bad;

  Need carry = {0, 0};
  for (int base = 0; base < a.n_seqs; base += kTableThreads) {
    const int s = base + threadIdx.x;
    Need n = {0, 0}, total;
    int held = 0;
    if (s < a.n_seqs && !status) {
      const int c = a.cached[s];
      held = blocks_of(c, a.block);
      n = {a.fresh[s], blocks_of(c + a.fresh[s], a.block) - held};
    }
    const Need upto = block_scan(n, waves, &total);
    if (s < a.n_seqs) {
      const int row = carry.rows + upto.rows - n.rows, first = carry.blocks + upto.blocks - n.blocks;
      a.row_off[s] = row;
      a.last_row[s] = n.rows ? row + n.rows - 1 : 0;
      a.table_off[s] = s * a.stride;
      for (int j = 0; j < n.blocks; ++j)
        a.tables[static_cast<int64_t>(s) * a.stride + held + j] = a.free_blocks[free - 1 - (first + j)];
    }
    carry.rows += total.rows;
    carry.blocks += total.blocks;
  }
  if (threadIdx.x == 0) a.row_off[a.n_seqs] = carry.rows;
  __syncthreads();
  for (int g = threadIdx.x; g < a.n_groups; g += kTableThreads) {
    int4 v = {0, 0, 0, 0};
    if (!status) {
      const int first = a.group_seqs[2 * g], count = a.group_seqs[2 * g + 1];
      v.x = a.row_off[first];
      v.y = a.row_off[first + count] - v.x;
      if (count) v.z = a.shared ? a.shared[first] : 0, v.w = first * a.stride;
    }
    a.groups[g] = v;
  }
  for (int t = threadIdx.x; t < a.max_rows; t += kTableThreads) fill_row(a, t, carry.rows);
  if (threadIdx.x == 0) {
    a.totals[0] = carry.rows;
    a.totals[1] = carry.blocks;
    a.totals[2] = free - carry.blocks;
    a.totals[3] = status;
  }
}

// ---- norm of q and k per head, rotation, cache write --------------------------------------------
//
// Per head x of q and k: y = w * x / sqrt(mean(x^2) + eps), then the pair (i, i + D/2) turns by pos *
// inv_freq[i]. A thread holds four consecutive pairs, a power of two of lanes a head, so the mean is a
// few shuffles. The angle is taken in turns with the product in double precision: at position
// 131,071 an fp32 product alone is off by up to 2^-8 radians, more than the fp16 results' rounding.

constexpr int kThreads = 256;

struct QkArgs {
  const float* qkv;
  int planes;
  const float* scale;
  int T;
  const float *bias, *q_norm, *k_norm;
  float eps;
  const float* inv_freq;
  const int *pos, *slot;
  half_t *kpool, *vpool, *q_out;
  float q_scale;
  int heads, kv_heads, D, block;
};

template <int LANES>
__global__ __launch_bounds__(kThreads) void qk_norm_kernel(const QkArgs a) {
  const int t = blockIdx.x, half = a.D / 2;
  const int h = blockIdx.y * (kThreads / LANES) + threadIdx.x / LANES, i = 4 * (threadIdx.x % LANES);
  const int slot = a.slot[t];
  if (slot < 0) return;  // an idle row
  const bool on = h < a.heads + 2 * a.kv_heads && i < half;
  const int n = h * a.D + i;
  const int64_t width = static_cast<int64_t>(a.heads + 2 * a.kv_heads) * a.D;
  float x[4] = {0, 0, 0, 0}, y[4] = {0, 0, 0, 0};
  if (on) {
    const int64_t plane = a.T * width, e = t * width + n;
    const float4 lo = merged4(a.qkv, a.planes, plane, e, a.scale ? a.scale + n : nullptr);
    const float4 hi = merged4(a.qkv, a.planes, plane, e + half, a.scale ? a.scale + n + half : nullptr);
    x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w;
    y[0] = hi.x, y[1] = hi.y, y[2] = hi.z, y[3] = hi.w;
    if (a.bias) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] += a.bias[n + j], y[j] += a.bias[n + j + half];
    }
  }
  const bool turned = h < a.heads + a.kv_heads;
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) ss += x[j] * x[j] + y[j] * y[j];
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
  if (!on) return;
  if (turned) {
    const float inv = 1.0f / sqrtf(ss / a.D + a.eps);
    const float* w = h < a.heads ? a.q_norm : a.k_norm;
    const double p = a.pos[t];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float u = x[j] * inv * w[i + j], v = y[j] * inv * w[i + j + half];
      const double turns = p * (static_cast<double>(a.inv_freq[i + j]) * 0.15915494309189535);
      float sn, cs;
      sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sn, &cs);
      x[j] = u * cs - v * sn;
      y[j] = v * cs + u * sn;
    }
  }
  half_t* dst;
  float f = 1.0f;
  if (h < a.heads) {
    dst = a.q_out + static_cast<int64_t>(t) * a.heads * a.D + n;
    f = a.q_scale;
  } else {
    dst = (turned ? a.kpool : a.vpool) +
          kv_row_offset(slot / a.block, a.kv_heads, (h - a.heads) % a.kv_heads, a.block, slot % a.block, a.D) + i;
  }
  half4 ox, oy;
#pragma unroll
  for (int j = 0; j < 4; ++j) ox[j] = static_cast<half_t>(x[j] * f), oy[j] = static_cast<half_t>(y[j] * f);
  *reinterpret_cast<half4*>(dst) = ox;
  *reinterpret_cast<half4*>(dst + half) = oy;
}

// ---- penalties, biases and masks on logits --------------------------------------------------------
//
// A workgroup takes a slice of consecutive logits of one row. Every logit of its slice is loaded first, 16
// bytes a lane; while they come it counts the row's history into an LDS word for each logit (bit 31:
// in the prompt; the rest: how often in the output; integer adds, so their order does not matter)
// and notes the last bias for each; then one pass over the registers. Slices begin where a row's
// address is a multiple of 16, so rows of odd vocabularies load and store 16 bytes too.

constexpr int kVec = 4;                                // 16-byte loads of a thread
constexpr int kSlice = 4 * kVec * kThreads;            // logits of a workgroup

struct LogitArgs {
  const float* in;
  int64_t ld;
  int rows, vocab, slices;
  const int* history;
  int64_t history_stride;
  const int *history_len, *prompt_len;
  const float *repetition, *frequency, *presence;
  const int* bias_tokens;
  const float* bias_values;
  int64_t bias_stride;
  const int* bias_len;
  const unsigned* masks;
  int64_t mask_stride;
  const int* mask_of;
  float* out;
  int64_t out_ld;
  int* next;
  int* counters;
  unsigned long long* best;
};

// A greater key for a greater logit, and at one logit for a lower token; 0: no logit above -inf.
__device__ __forceinline__ unsigned long long token_key(float x, int token) {
  if (!(x > -INFINITY)) return 0;
  const unsigned u = __float_as_uint(x + 0.0f);  // -0 counts as 0
  const unsigned k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return static_cast<unsigned long long>(k) << 32 | (0xffffffffu - static_cast<unsigned>(token));
}

__device__ __forceinline__ unsigned long long block_best(unsigned long long v, unsigned long long* waves) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor(v, o);
    v = w > v ? w : v;
  }
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  v = waves[0];
#pragma unroll
  for (int i = 1; i < kThreads / 64; ++i) v = waves[i] > v ? waves[i] : v;
  __syncthreads();
  return v;
}

// BIAS: there are biases. VEC: a row's logits and results lie alike to 16 bytes.
template <bool BIAS, bool VEC>
__global__ __launch_bounds__(kThreads) void process_logits_kernel(const LogitArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned s_seen[kSlice];
  __shared__ __attribute__((aligned(16))) int s_bias[BIAS ? kSlice : 4];
  __shared__ unsigned long long s_best[kThreads / 64];
  __shared__ int s_last;
  const int row = blockIdx.x / a.slices, part = blockIdx.x % a.slices;
  const float* in = a.in + row * a.ld;
  float* out = a.out + row * a.out_ld;
  // The slice's first logit; the first slice begins up to three before the row.
  const int v0 = part * kSlice - (VEC ? static_cast<int>(reinterpret_cast<uintptr_t>(in) / 4 % 4) : 0);
  const auto at = [&](int i) { return VEC ? 4 * (threadIdx.x + i * kThreads) : static_cast<int>(threadIdx.x) + 4 * i * kThreads; };
  float x[kVec][4];
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = v0 + at(i);
    if (VEC && v >= 0 && v + 3 < a.vocab) {
      const float4 f = *reinterpret_cast<const float4*>(in + v);
      x[i][0] = f.x, x[i][1] = f.y, x[i][2] = f.z, x[i][3] = f.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int u = v + (VEC ? e : e * kThreads);
        x[i][e] = u >= 0 && u < a.vocab ? in[u] : 0.0f;
      }
    }
  }
  const int mask_row = a.masks ? (a.mask_of ? a.mask_of[row] : row) : -1;
  const unsigned* mask = a.masks + (mask_row < 0 ? 0 : mask_row * a.mask_stride);
  unsigned lo[kVec], hi[kVec];  // the mask's words of a thread's four logits (VEC; else read one by one)
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    lo[i] = hi[i] = ~0u;
    const int v = v0 + at(i);
    if (VEC && mask_row >= 0 && v < a.vocab) {
      lo[i] = mask[max(v, 0) >> 5];
      hi[i] = mask[min(v + 3, a.vocab - 1) >> 5];
    }
  }
  const float rep = a.repetition ? a.repetition[row] : 1.0f;
  const float freq = a.frequency ? a.frequency[row] : 0.0f, pres = a.presence ? a.presence[row] : 0.0f;
  const int64_t bias_at = row * a.bias_stride;
  if (a.history || BIAS) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      reinterpret_cast<uint4v*>(s_seen)[threadIdx.x + i * kThreads] = uint4v{0, 0, 0, 0};
      if (BIAS) reinterpret_cast<uint4v*>(s_bias)[threadIdx.x + i * kThreads] = uint4v{0, 0, 0, 0};
    }
    __syncthreads();
    const unsigned n = static_cast<unsigned>(max(0, min(kSlice, a.vocab - v0)));
    // A token below 0 or past the vocabulary is outside every slice.
    const auto place = [&](int token) { return token < 0 ? ~0u : static_cast<unsigned>(token) - static_cast<unsigned>(v0); };
    if (a.history) {
      const int len = static_cast<int>(min(static_cast<int64_t>(max(a.history_len[row], 0)), a.history_stride));
      const int prompt = a.prompt_len ? a.prompt_len[row] : 0;
      const int* h = a.history + row * a.history_stride;
      constexpr int kAhead = 8;  // tokens of a thread in flight
      for (int j0 = threadIdx.x; j0 < len; j0 += kAhead * kThreads) {
        int token[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) token[i] = j0 + i * kThreads < len ? h[j0 + i * kThreads] : -1;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const unsigned p = place(token[i]);
          if (p < n) {
            if (j0 + i * kThreads < prompt)
              atomicOr(&s_seen[p], 0x80000000u);
            else
              atomicAdd(&s_seen[p], 1u);
          }
        }
      }
    }
    if (BIAS) {
      const int len = static_cast<int>(min(static_cast<int64_t>(max(a.bias_len[row], 0)), a.bias_stride));
      for (int j = threadIdx.x; j < len; j += kThreads) {
        const unsigned p = place(a.bias_tokens[bias_at + j]);
        if (p < n) atomicMax(&s_bias[p], j + 1);
      }
    }
    __syncthreads();
  }
  unsigned long long best = 0;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = v0 + at(i);
    unsigned seen4[4] = {0, 0, 0, 0};
    int bias4[4] = {0, 0, 0, 0};
    if (VEC) {
      const uint4v s = reinterpret_cast<const uint4v*>(s_seen)[threadIdx.x + i * kThreads];
      if (a.history) seen4[0] = s[0], seen4[1] = s[1], seen4[2] = s[2], seen4[3] = s[3];
      if (BIAS) {
        const uint4v b = reinterpret_cast<const uint4v*>(s_bias)[threadIdx.x + i * kThreads];
        bias4[0] = b[0], bias4[1] = b[1], bias4[2] = b[2], bias4[3] = b[3];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (a.history) seen4[e] = s_seen[at(i) + e * kThreads];
        if (BIAS) bias4[e] = s_bias[at(i) + e * kThreads];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int u = v + (VEC ? e : e * kThreads);
      float y = x[i][e];
      if (a.history) {
        if (const unsigned seen = seen4[e]) {
          // Each step rounded by itself, in the order of the formula.
          y = y > 0.0f ? y / rep : mul_rounded(y, rep);
          if (const unsigned count = seen & 0x7fffffffu) y = y - mul_rounded(freq, static_cast<float>(count)) - pres;
        }
      }
      if (BIAS)
        if (const int b = bias4[e]) y += a.bias_values[bias_at + b - 1];
      if (u >= 0 && u < a.vocab) {
        const unsigned word = !VEC ? (mask_row >= 0 ? mask[u >> 5] : ~0u) : u >> 5 == max(v, 0) >> 5 ? lo[i] : hi[i];
        if (!((word >> (u & 31)) & 1u)) y = -INFINITY;
        const unsigned long long k = token_key(y, u);
        best = k > best ? k : best;
      }
      x[i][e] = y;
    }
    if (VEC && v >= 0 && v + 3 < a.vocab) {
      *reinterpret_cast<float4*>(out + v) = float4{x[i][0], x[i][1], x[i][2], x[i][3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int u = v + (VEC ? e : e * kThreads);
        if (u >= 0 && u < a.vocab) out[u] = x[i][e];
      }
    }
  }
  if (!a.next) return;
  best = block_best(best, s_best);
  if (threadIdx.x == 0) {
    __hip_atomic_store(&a.best[static_cast<int64_t>(row) * a.slices + part], best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_s_waitcnt(0);
    const int prev = __hip_atomic_fetch_add(&a.counters[row], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = prev == a.slices - 1;
    if (s_last) __hip_atomic_store(&a.counters[row], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  // The row's last workgroup takes the best of all slices.
  best = 0;
  for (int p = threadIdx.x; p < a.slices; p += kThreads) {
    unsigned long long* const from = &a.best[static_cast<int64_t>(row) * a.slices + p];
    const unsigned long long k = __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(from, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // zero again, for calls of any shape
    best = k > best ? k : best;
  }
  best = block_best(best, s_best);
  if (threadIdx.x == 0) a.next[row] = best ? static_cast<int>(0xffffffffu - static_cast<unsigned>(best)) : -1;
}

// (A row may begin up to three logits into its first slice.)
int slices_of(int vocab) { return static_cast<int>((static_cast<int64_t>(vocab) + 3 + kSlice - 1) / kSlice); }

}  // namespace
}  // namespace relay_hip

using namespace relay_hip;

extern "C" {

int rh_step_tables(const int* cached, const int* fresh, const int* shared, int n_seqs, const int* group_seqs, int n_groups,
                   int block_size, int* tables, int table_stride, const int* free_blocks, const int* free_count,
                   int max_rows, int* row_off, int* last_row, int* table_off, int* pos, int* seq, int* slot,
                   int* dec_meta, int* groups, int* totals, void* stream) {
  RH_REQUIRE(n_seqs >= 0 && n_groups >= 0 && block_size > 0 && table_stride > 0 && max_rows >= 0,
             "step tables: bad sizes");
  RH_REQUIRE(max_rows < kSumCap && block_size < kSumCap && static_cast<int64_t>(n_seqs) * table_stride < (int64_t{1} << 31),
             "step tables: max_rows and block_size must be below 2^30 - 1 and n_seqs * table_stride below 2^31");
  RH_REQUIRE(free_count && row_off && totals &&
                 (n_seqs == 0 || (cached && fresh && tables && free_blocks && last_row && table_off)) &&
                 (n_groups == 0 || (group_seqs && groups)) && (max_rows == 0 || (pos && seq && slot && dec_meta)),
             "step tables: missing pointer");
  RH_REQUIRE((reinterpret_cast<uintptr_t>(dec_meta) | reinterpret_cast<uintptr_t>(groups)) % 16 == 0,
             "step tables: dec_meta and groups must be 16-byte aligned");
  const StepArgs a{cached, fresh, shared, group_seqs, n_seqs, n_groups, block_size, tables, table_stride, free_blocks,
                   free_count, max_rows, row_off, last_row, table_off, pos, seq, slot,
                   reinterpret_cast<int4*>(dec_meta), reinterpret_cast<int4*>(groups), totals};
  RH_TRY_LAUNCH(hipLaunchKernelGGL(step_tables_kernel, dim3(1), dim3(kTableThreads), 0, static_cast<hipStream_t>(stream), a));
  return 0;
}

int rh_qk_norm_to_cache(const float* qkv, int planes, const float* scale, int T, const float* bias, const float* q_norm,
                        const float* k_norm, float eps, const float* inv_freq, const int* pos, const int* slot,
                        void* kpool, void* vpool, void* q_out, float q_scale, int heads, int kv_heads, int head_dim,
                        int block_size, void* stream) {
  if (T == 0) return 0;
  RH_REQUIRE(T > 0 && heads > 0 && kv_heads > 0 && block_size > 0, "qk_norm: bad sizes");
  RH_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 512, "qk_norm: head_dim must be a multiple of 8, at most 512");
  RH_REQUIRE(planes >= 1 && planes <= kMaxMergeSplit, "qk_norm: planes must be in 1..8");
  RH_REQUIRE(qkv && q_norm && k_norm && inv_freq && pos && slot && kpool && vpool && q_out, "qk_norm: missing pointer");
  RH_REQUIRE(reinterpret_cast<uintptr_t>(qkv) % 16 == 0 &&
                 (reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(kpool) |
                  reinterpret_cast<uintptr_t>(vpool)) % 8 == 0,
             "qk_norm: qkv must be 16-byte aligned, q_out and the pools 8-byte");
  const QkArgs a{qkv, planes, scale, T, bias, q_norm, k_norm, eps, inv_freq, pos, slot, static_cast<half_t*>(kpool),
                 static_cast<half_t*>(vpool), static_cast<half_t*>(q_out), q_scale, heads, kv_heads, head_dim, block_size};
  const int total = heads + 2 * kv_heads;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const auto launch = [&](auto kernel, int lanes) {
    const int per = kThreads / lanes;
    hipLaunchKernelGGL(kernel, dim3(T, (total + per - 1) / per), dim3(kThreads), 0, s, a);
  };
  if (head_dim <= 32) {
    RH_TRY_LAUNCH(launch(qk_norm_kernel<4>, 4));
  } else if (head_dim <= 64) {
    RH_TRY_LAUNCH(launch(qk_norm_kernel<8>, 8));
  } else if (head_dim <= 128) {
    RH_TRY_LAUNCH(launch(qk_norm_kernel<16>, 16));
  } else if (head_dim <= 256) {
    RH_TRY_LAUNCH(launch(qk_norm_kernel<32>, 32));
  } else {
    RH_TRY_LAUNCH(launch(qk_norm_kernel<64>, 64));
  }
  return 0;
}

size_t rh_process_logits_workspace(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0) return 0;
  return (static_cast<size_t>(rows) + 1) / 2 * 8 + static_cast<size_t>(rows) * slices_of(vocab) * 8;
}

int rh_process_logits(const float* logits, int64_t ld, int rows, int vocab, const int* history, int64_t history_stride,
                      const int* history_len, const int* prompt_len, const float* repetition, const float* frequency,
                      const float* presence, const int* bias_tokens, const float* bias_values, int64_t bias_stride,
                      const int* bias_len, const uint32_t* masks, int64_t mask_stride, const int* mask_of, float* out,
                      int64_t out_ld, int* next, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows == 0) return 0;
  RH_REQUIRE(rows > 0 && vocab > 0 && ld >= vocab && out_ld >= vocab, "process_logits: bad sizes");
  RH_REQUIRE(logits && out, "process_logits: missing pointer");
  RH_REQUIRE(logits != out || ld == out_ld, "process_logits: in place needs one row stride");
  RH_REQUIRE(!history || (history_len && history_stride >= 0 && history_stride < kSumCap),
             "process_logits: a history needs its lengths and a stride below 2^30");
  RH_REQUIRE(history || !(prompt_len || repetition || frequency || presence), "process_logits: penalties need a history");
  RH_REQUIRE(!bias_tokens || (bias_values && bias_len && bias_stride >= 0 && bias_stride < kSumCap),
             "process_logits: biases need values, lengths and a stride below 2^30");
  RH_REQUIRE(!masks || mask_stride >= (static_cast<int64_t>(vocab) + 31) / 32, "process_logits: a mask row holds a bit for each token");
  const int slices = slices_of(vocab);
  RH_REQUIRE(static_cast<int64_t>(rows) * slices < (int64_t{1} << 31), "process_logits: too many rows");
  RH_REQUIRE(!next || (workspace && workspace_bytes >= rh_process_logits_workspace(rows, vocab) &&
                       reinterpret_cast<uintptr_t>(workspace) % 8 == 0),
             "process_logits: next needs an 8-byte aligned workspace of rh_process_logits_workspace bytes");
  LogitArgs a{logits, ld, rows, vocab, slices, history, history_stride, history_len, prompt_len, repetition, frequency,
              presence, bias_tokens, bias_values, bias_stride, bias_len, masks, mask_stride, mask_of, out, out_ld, next,
              static_cast<int*>(workspace), nullptr};
  if (next) a.best = reinterpret_cast<unsigned long long*>(a.counters + (rows + 1) / 2 * 2);
  // Every row lies alike in logits and out: equal strides, or both whole 16-byte steps.
  const bool vec = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(out)) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(logits) % 4 == 0 && (ld - out_ld) % 4 == 0;
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(rows * slices), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
  };
  if (bias_tokens) {
    RH_TRY_LAUNCH(vec ? go(process_logits_kernel<true, true>) : go(process_logits_kernel<true, false>));
  } else {
    RH_TRY_LAUNCH(vec ? go(process_logits_kernel<false, true>) : go(process_logits_kernel<false, false>));
  }
  return 0;
}

}  // extern "C"
