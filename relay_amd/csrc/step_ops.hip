// The operators of a decode step that stays on the GPU, around its attention: block tables and
// slot maps from the request lengths, the norm of q and k per head with the rotation and the
// cache write, and penalties, biases, grammar masks and the greedy token on the logits. relay
// does the first and the last on the host (engine.cpp, sampler.cpp) and has no norm of q and k.
#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "../../include/relay_hip.h"
#include "common.h"

namespace relay_hip {
namespace {

// ---- block tables and slot maps --------------------------------------------------------------
//
// held = ceil(cached / B), want = ceil((cached + fresh) / B); sequence s takes want - held ids off the
// top of the free stack, behind those of the sequences before it, and has the rows row_off[s] ..
// row_off[s + 1] - 1: two exclusive sums over the sequences, a chain of dependent steps that bounds the call.
// Up to kWideRows rows one workgroup takes them, a sequence a thread (more in several turns); where no
// sequence adds more than kOwnRows tokens, as in decoding, its thread writes its rows too, from what it
// has in registers (48 decoding sequences 3.9 us, with a search for each row's sequence 6). Larger steps take
// many workgroups that all make the sums (step_wide_kernel; 511 sequences of which 40 add a prompt, 26,500
// rows, 5.5 us), unless the stack's count lies in the totals: then one workgroup makes them, with the rows in a
// second launch past kOneLaunch of them (9.4 us; in one workgroup 58).

constexpr int kSumCap = (1 << 30) - 1;  // sums stop here, past every limit that they are compared with
constexpr int kOwnRows = 4;
constexpr int kWideRows = 512;           // 511 decoding sequences 5.3 us in one workgroup, 5.5 in two; 48 and a prompt of 512 6.5, 4.7
constexpr int kOneLaunch = 4096;
constexpr int kRowThreads = 256;
constexpr int kRowOffsets = 4096;        // sequences whose first rows a workgroup keeps in LDS

struct StepArgs {
  const int *cached, *fresh, *shared, *group_seqs;
  int n_seqs, n_groups, block;
  Div by_block;
  int* tables;
  int stride, row_keys;  // entries of a sequence's row of the tables, and keys that they hold
  const int *free_blocks, *free_count;
  int max_rows;
  int *row_off, *last_row, *table_off, *pos, *seq, *slot;
  int4 *meta, *groups;
  int* totals;
};

__device__ __forceinline__ int capped_add(int a, int b) { return min(a + b, kSumCap); }
__device__ __forceinline__ int blocks_of(int keys, const Div& block) { return block(keys + static_cast<int>(block.d) - 1); }

struct Need {
  int rows, blocks;
};

// Inclusive sums over the workgroup and the workgroup's total. `waves` holds an entry a wave, and is free
// again after the caller's next barrier.
template <int THREADS>
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
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) {
    if (i == w) before = sum;
    sum.rows = capped_add(sum.rows, waves[i].rows);
    sum.blocks = capped_add(sum.blocks, waves[i].blocks);
  }
  *total = sum;
  return {capped_add(before.rows, v.rows), capped_add(before.blocks, v.blocks)};
}

struct Length {
  int cached, shared, bad;
  Need need;
};

constexpr int kPastTable = 16;  // more shared keys than a row of the tables holds: attention would read past it

// The call's status: what is wrong with its lengths and its room, else with its shared keys.
__device__ __forceinline__ int status_of(int bad) { return bad & (kPastTable - 1) ? bad & (kPastTable - 1) : bad ? RH_STEP_BAD_LENGTH : 0; }

// What sequence s adds, or why it cannot.
__device__ __forceinline__ Length length_of(const StepArgs& a, int s) {
  Length n{a.cached[s], a.shared ? a.shared[s] : 0, 0, {0, 0}};
  const int f = a.fresh[s];
  if (n.shared > a.row_keys) n.bad = kPastTable;
  if (n.cached < 0 || f < 0 || n.cached > kSumCap || f > kSumCap - n.cached || n.shared < 0) {
    n.bad |= RH_STEP_BAD_LENGTH;
  } else {
    const int want = blocks_of(n.cached + f, a.by_block);
    if (want > a.stride) n.bad |= RH_STEP_TABLE_FULL;
    n.need = {f, want - blocks_of(n.cached, a.by_block)};
  }
  return n;
}

template <int THREADS>
__device__ __forceinline__ int bad_groups(const StepArgs& a) {
  int bad = 0;
  for (int g = threadIdx.x; g < a.n_groups; g += THREADS) {
    const int first = a.group_seqs[2 * g], count = a.group_seqs[2 * g + 1];
    if (first < 0 || count < 0 || first > a.n_seqs || count > a.n_seqs - first) bad = RH_STEP_BAD_LENGTH;
  }
  return bad;
}

__device__ __forceinline__ void put_totals(const StepArgs& a, Need all, int free, int status) {
  a.row_off[a.n_seqs] = all.rows;
  a.totals[0] = all.rows;
  a.totals[1] = all.blocks;
  a.totals[2] = free - all.blocks;
  a.totals[3] = status;
}

// Row t: position p of sequence s in block `id`.
__device__ __forceinline__ void put_row(const StepArgs& a, int t, int s, int p, int id, int shared) {
  a.pos[t] = p;
  a.seq[t] = s;
  a.slot[t] = id * a.block + p - a.by_block(p) * a.block;
  a.meta[t] = int4{t, p + 1, s * a.stride, shared};
}

// A row past the step's tokens: no slot, an empty context.
__device__ __forceinline__ void put_idle(const StepArgs& a, int t) {
  a.pos[t] = 0;
  a.seq[t] = 0;
  a.slot[t] = -1;
  a.meta[t] = int4{t, 0, 0, 0};
}

// Row t by search: its sequence is the last with row_off[s] <= t (one that has rows, as t < row_off[n_seqs]).
__device__ __forceinline__ void find_row(const StepArgs& a, const int* row_off, int t) {
  int lo = 0, hi = a.n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (row_off[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  const int p = a.cached[lo] + t - row_off[lo];
  put_row(a, t, lo, p, a.tables[lo * a.stride + a.by_block(p)], a.shared ? a.shared[lo] : 0);
}

// ROWS: the rows too.
template <int THREADS, bool ROWS>
__global__ __launch_bounds__(THREADS) void step_tables_kernel(const StepArgs a) {
  __shared__ Need waves[2][THREADS / 64];
  __shared__ int s_bad, s_most, s_taken[THREADS], s_held[THREADS];
  const int free = *a.free_count;
  if (threadIdx.x == 0) s_bad = 0, s_most = 0;
  // The sums and checks of the whole step come first: a step that does not fit changes nothing.
  int bad = free < 0 ? RH_STEP_BAD_LENGTH : 0, most = 0;
  Need all = {0, 0}, mine = {0, 0}, upto = {0, 0};  // mine, upto: of the last turn, the only one up to THREADS sequences
  int cached = 0, shared = 0;
  for (int base = 0, turn = 0; base < a.n_seqs; base += THREADS, turn ^= 1) {
    const int s = base + threadIdx.x;
    mine = {0, 0};
    if (s < a.n_seqs) {
      const Length n = length_of(a, s);
      cached = n.cached, shared = n.shared, mine = n.need;
      bad |= n.bad;
      most = max(most, mine.rows);
    }
    Need total;
    upto = block_scan<THREADS>(mine, waves[turn], &total);
    all.rows = capped_add(all.rows, total.rows);
    all.blocks = capped_add(all.blocks, total.blocks);
  }
  bad |= bad_groups<THREADS>(a);
  if (all.rows > a.max_rows) bad |= RH_STEP_ROWS_FULL;
  if (all.blocks > free) bad |= RH_STEP_NO_BLOCKS;
  if (a.n_seqs == 0) __syncthreads();  // (the scans' barriers follow s_bad's clearing)
  if (bad) atomicOr(&s_bad, bad);
  if (most > kOwnRows) s_most = 1;
  __syncthreads();
  const int status = status_of(s_bad);
  const bool own_rows = ROWS && !s_most;
  if (status) all = {0, 0};

  Need carry = {0, 0};
  for (int base = 0, turn = 0; base < a.n_seqs; base += THREADS, turn ^= 1) {
    const int s = base + threadIdx.x;
    if (a.n_seqs > THREADS) {
      mine = {0, 0};
      if (s < a.n_seqs && !status) {
        cached = a.cached[s];
        shared = a.shared ? a.shared[s] : 0;
        mine = {a.fresh[s], blocks_of(cached + a.fresh[s], a.by_block) - blocks_of(cached, a.by_block)};
      }
      Need total;
      upto = block_scan<THREADS>(mine, waves[turn], &total);
      upto.rows += carry.rows, upto.blocks += carry.blocks;
      carry.rows += total.rows, carry.blocks += total.blocks;
    }
    if (status) mine = upto = {0, 0};
    if (s < a.n_seqs) {
      const int row = upto.rows - mine.rows, first = upto.blocks - mine.blocks;
      a.row_off[s] = row;
      a.last_row[s] = mine.rows ? upto.rows - 1 : 0;
      a.table_off[s] = s * a.stride;
      const int held = blocks_of(cached, a.by_block);
      int* const table = a.tables + static_cast<int64_t>(s) * a.stride;
      s_taken[threadIdx.x] = first;
      s_held[threadIdx.x] = held;
      if (!s_most)
        for (int j = 0; j < mine.blocks; ++j) table[held + j] = a.free_blocks[free - 1 - (first + j)];
      if (own_rows) {
        for (int j = 0; j < mine.rows; ++j) {
          const int at = a.by_block(cached + j);
          put_row(a, row + j, s, cached + j, at < held ? table[at] : a.free_blocks[free - 1 - (first + at - held)], shared);
        }
      }
    }
    if (s_most) {
      // Prompts take many ids: a thread an id, which finds its sequence among this turn's.
      __syncthreads();
      const int count = min(THREADS, a.n_seqs - base), upto_here = a.n_seqs > THREADS ? carry.blocks : all.blocks;
      for (int k = s_taken[0] + threadIdx.x; k < upto_here; k += THREADS) {
        int lo = 0, hi = count;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (s_taken[mid] <= k)
            lo = mid;
          else
            hi = mid;
        }
        a.tables[static_cast<int64_t>(base + lo) * a.stride + s_held[lo] + k - s_taken[lo]] = a.free_blocks[free - 1 - k];
      }
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) put_totals(a, all, free, status);
  if (a.n_groups || (ROWS && !own_rows)) __syncthreads();  // row_off and the tables are read below
  for (int g = threadIdx.x; g < a.n_groups; g += THREADS) {
    int4 v = {0, 0, 0, 0};
    if (!status) {
      const int first = a.group_seqs[2 * g], count = a.group_seqs[2 * g + 1];
      v.x = a.row_off[first];
      v.y = a.row_off[first + count] - v.x;
      if (count) v.z = a.shared ? a.shared[first] : 0, v.w = first * a.stride;
    }
    a.groups[g] = v;
  }
  if (ROWS) {
    if (!own_rows)
      for (int t = threadIdx.x; t < all.rows; t += THREADS) find_row(a, a.row_off, t);
    for (int t = all.rows + threadIdx.x; t < a.max_rows; t += THREADS) put_idle(a, t);
  }
}

// The whole step in many workgroups, each of which takes the sums for itself (they read the same few KB), keeps
// every sequence's first row and first new id in LDS and then writes its rows; the first one writes what there is once
// a sequence. A row whose block is new reads its id from the stack, so nobody waits for the tables.
// Not where free_count is one of the totals, which the first may write before another has read it.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void step_wide_kernel(const StepArgs a) {
  __shared__ Need waves[2][THREADS / 64];
  __shared__ int s_bad, s_off[kRowOffsets], s_taken[kRowOffsets];
  const int free = *a.free_count;
  if (threadIdx.x == 0) s_bad = 0;
  int bad = free < 0 ? RH_STEP_BAD_LENGTH : 0;
  Need all = {0, 0};
  for (int base = 0, turn = 0; base < a.n_seqs; base += THREADS, turn ^= 1) {
    const int s = base + threadIdx.x;
    Need mine = {0, 0};
    if (s < a.n_seqs) {
      const Length n = length_of(a, s);
      bad |= n.bad;
      mine = n.need;
    }
    Need total;
    const Need upto = block_scan<THREADS>(mine, waves[turn], &total);
    if (s < a.n_seqs) {
      s_off[s] = capped_add(all.rows, upto.rows - mine.rows);
      s_taken[s] = capped_add(all.blocks, upto.blocks - mine.blocks);
    }
    all.rows = capped_add(all.rows, total.rows);
    all.blocks = capped_add(all.blocks, total.blocks);
  }
  bad |= bad_groups<THREADS>(a);
  if (all.rows > a.max_rows) bad |= RH_STEP_ROWS_FULL;
  if (all.blocks > free) bad |= RH_STEP_NO_BLOCKS;
  if (a.n_seqs == 0) __syncthreads();  // (the scans' barriers follow s_bad's clearing)
  if (bad) atomicOr(&s_bad, bad);
  __syncthreads();
  const int status = status_of(s_bad);
  if (status) all = {0, 0};
  const auto last_at = [&](const int* firsts, int k) {  // the last sequence that begins at or before k
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (firsts[mid] <= k)
        lo = mid;
      else
        hi = mid;
    }
    return lo;
  };
  const int t = blockIdx.x * THREADS + threadIdx.x;
  if (t < all.rows) {
    const int s = last_at(s_off, t), cached = a.cached[s], p = cached + t - s_off[s], at = a.by_block(p), held = blocks_of(cached, a.by_block);
    const int id = at < held ? a.tables[s * a.stride + at] : a.free_blocks[free - 1 - (s_taken[s] + at - held)];
    put_row(a, t, s, p, id, a.shared ? a.shared[s] : 0);
  } else if (t < a.max_rows) {
    put_idle(a, t);
  }
  for (int k = t; k < all.blocks; k += gridDim.x * THREADS) {
    const int s = last_at(s_taken, k);
    a.tables[s * a.stride + blocks_of(a.cached[s], a.by_block) + k - s_taken[s]] = a.free_blocks[free - 1 - k];
  }
  if (blockIdx.x) return;
  const auto off = [&](int s) { return status ? 0 : s < a.n_seqs ? s_off[s] : all.rows; };
  for (int s = threadIdx.x; s < a.n_seqs; s += THREADS) {
    a.row_off[s] = off(s);
    a.last_row[s] = off(s + 1) > off(s) ? off(s + 1) - 1 : 0;
    a.table_off[s] = s * a.stride;
  }
  for (int g = threadIdx.x; g < a.n_groups; g += THREADS) {
    int4 v = {0, 0, 0, 0};
    if (!status) {
      const int first = a.group_seqs[2 * g], count = a.group_seqs[2 * g + 1];
      v.x = off(first);
      v.y = off(first + count) - v.x;
      if (count) v.z = a.shared ? a.shared[first] : 0, v.w = first * a.stride;
    }
    a.groups[g] = v;
  }
  if (threadIdx.x == 0) put_totals(a, all, free, status);
}

__global__ __launch_bounds__(kRowThreads) void step_rows_kernel(const StepArgs a) {
  __shared__ int s_off[kRowOffsets];
  const int total = a.totals[0], t = blockIdx.x * kRowThreads + threadIdx.x;
  const bool in_lds = a.n_seqs <= kRowOffsets;
  if (in_lds) {
    for (int s = threadIdx.x; s < a.n_seqs; s += kRowThreads) s_off[s] = a.row_off[s];
    __syncthreads();
  }
  if (t >= a.max_rows) return;
  if (t >= total)
    put_idle(a, t);
  else if (in_lds)
    find_row(a, s_off, t);
  else
    find_row(a, a.row_off, t);
}

// ---- norm of q and k per head, rotation, cache write --------------------------------------------
//
// Per head x of q and k: y = w * x / sqrt(mean(x^2) + eps), then the pair (i, i + D/2) turns by pos *
// inv_freq[i]. A thread holds four consecutive pairs, a power of two of lanes a head, so the mean is a
// few shuffles. A wave takes HEADS sets of heads of one token, their loads together; the sines, most of
// the arithmetic, serve all of them. The angle is taken in turns with the product in double precision:
// at position 131,071 an fp32 product alone is off by up to 2^-8 radians, more than the fp16 results'
// rounding.

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
  Div by_block, by_sets;  // by_sets: sets of heads a token
};

// PLAIN: one plane and no scale, without the branches of up to 8 (2047 rows of 32/4 heads of 64 9.6 us, with them
// 10.8, one row 3.1 and 3.8; these figures and those below in a graph, call after call).
template <int LANES, int HEADS, bool PLAIN>
__global__ __launch_bounds__(kThreads) void qk_norm_kernel(const QkArgs a) {
  constexpr int PER = kWave / LANES;  // heads of a set
  // The arguments at once: the compiler loads them where they are used, one wait after another (2047 rows of 32/4
  // heads of 64 10.4 -> 9.6 us; the tables' and the logits' kernels gain nothing by it).
  asm volatile("" : : "s"(a.qkv), "s"(a.planes), "s"(a.scale), "s"(a.T), "s"(a.bias), "s"(a.q_norm), "s"(a.k_norm), "s"(a.eps), "s"(a.inv_freq),
               "s"(a.pos), "s"(a.slot), "s"(a.kpool), "s"(a.vpool), "s"(a.q_out), "s"(a.q_scale), "s"(a.heads), "s"(a.kv_heads), "s"(a.D),
               "s"(a.block), "s"(a.by_block.m), "s"(a.by_sets.m));
  const int unit = blockIdx.x * (kThreads / kWave) + (threadIdx.x >> 6);  // (token, HEADS sets)
  const int t = a.by_sets(unit), h0 = (unit - t * static_cast<int>(a.by_sets.d)) * (PER * HEADS) + (threadIdx.x & 63) / LANES, i = 4 * (threadIdx.x % LANES);
  if (t >= a.T) return;
  const int slot = a.slot[t];
  const double p = a.pos[t];
  if (slot < 0) return;  // an idle row
  const int block = a.by_block(slot);
  const int half = a.D / 2, total = a.heads + 2 * a.kv_heads;
  const int64_t width = static_cast<int64_t>(total) * a.D, plane = a.T * width;
  float x[HEADS][4], y[HEADS][4];
#pragma unroll
  for (int k = 0; k < HEADS; ++k) {
    const int h = h0 + k * PER, n = h * a.D + i;
    float4 lo = {0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
    if (PLAIN && h < total && i < half) {
      lo = *reinterpret_cast<const float4*>(a.qkv + t * width + n);
      hi = *reinterpret_cast<const float4*>(a.qkv + t * width + n + half);
    } else if (h < total && i < half) {
      lo = merged4(a.qkv, a.planes, plane, t * width + n, a.scale ? a.scale + n : nullptr);
      hi = merged4(a.qkv, a.planes, plane, t * width + n + half, a.scale ? a.scale + n + half : nullptr);
    }
    x[k][0] = lo.x, x[k][1] = lo.y, x[k][2] = lo.z, x[k][3] = lo.w;
    y[k][0] = hi.x, y[k][1] = hi.y, y[k][2] = hi.z, y[k][3] = hi.w;
  }
  float sn[4] = {}, cs[4] = {};
  if (i < half && h0 < a.heads + a.kv_heads) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double turns = p * (static_cast<double>(a.inv_freq[i + j]) * 0.15915494309189535);
      sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sn[j], &cs[j]);
    }
  }
#pragma unroll
  for (int k = 0; k < HEADS; ++k) {
    const int h = h0 + k * PER, n = h * a.D + i;
    const bool on = h < total && i < half;
    if (a.bias && on) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[k][j] += a.bias[n + j], y[k][j] += a.bias[n + j + half];
    }
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) ss += x[k][j] * x[k][j] + y[k][j] * y[k][j];
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
    if (!on) continue;
    const bool turned = h < a.heads + a.kv_heads;
    if (turned) {
      const float inv = 1.0f / sqrtf(ss / a.D + a.eps);
      const float* w = h < a.heads ? a.q_norm : a.k_norm;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float u = x[k][j] * inv * w[i + j], v = y[k][j] * inv * w[i + j + half];
        x[k][j] = u * cs[j] - v * sn[j];
        y[k][j] = v * cs[j] + u * sn[j];
      }
    }
    half_t* dst;
    float f = 1.0f;
    if (h < a.heads) {
      dst = a.q_out + static_cast<int64_t>(t) * a.heads * a.D + n;
      f = a.q_scale;
    } else {
      dst = (turned ? a.kpool : a.vpool) +
            kv_row_offset(block, a.kv_heads, h - a.heads - (turned ? 0 : a.kv_heads), a.block, slot - block * a.block, a.D) + i;
    }
    half4 ox, oy;
#pragma unroll
    for (int j = 0; j < 4; ++j) ox[j] = static_cast<half_t>(x[k][j] * f), oy[j] = static_cast<half_t>(y[k][j] * f);
    *reinterpret_cast<half4*>(dst) = ox;
    *reinterpret_cast<half4*>(dst + half) = oy;
  }
}

// ---- penalties, biases and masks on logits --------------------------------------------------------
//
// A workgroup takes a slice of consecutive logits of one row. While they come, 16 bytes a lane, it counts
// the row's history into an LDS word for each logit (bit 31: in the prompt; the rest: how often in the
// output; integer adds, so their order does not matter) and notes the last bias for each; then one pass
// over the registers. Slices begin where a row's address is a multiple of 16, so rows of odd
// vocabularies load and store 16 bytes too. The token: each slice posts its greatest (logit, -token)
// key, and the row's last workgroup takes the greatest of them.

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
  unsigned long long* records;  // per row: a count of slices, then their best keys
  int64_t record;               // words of a record
};

// A greater key for a greater logit, and at one logit for a lower token; 0: no logit above -inf.
__device__ __forceinline__ unsigned long long token_key(float x, int token) {
  if (!(x > -INFINITY)) return 0;
  const unsigned u = __float_as_uint(x + 0.0f);  // -0 counts as 0
  const unsigned k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return static_cast<unsigned long long>(k) << 32 | (0xffffffffu - static_cast<unsigned>(token));
}

template <int THREADS>
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
  for (int i = 1; i < THREADS / 64; ++i) v = waves[i] > v ? waves[i] : v;
  __syncthreads();
  return v;
}

// BIAS: there are biases. VEC: a row's logits and results lie alike to 16 bytes.
template <bool BIAS, bool VEC, int kVec, int THREADS>
__global__ __launch_bounds__(THREADS) void process_logits_kernel(const LogitArgs a) {
  // A word for each logit of the slice: first what the history says, then the last bias that names it
  // (an array of its own for these would halve the workgroups that a CU holds: 64 rows of 128,257
  // then 32 / 30 us).
  constexpr int kSlice = 4 * kVec * THREADS;
  __shared__ __attribute__((aligned(16))) unsigned s_word[kSlice];
  __shared__ unsigned long long s_best[THREADS / 64];
  __shared__ int s_last;
  // Workgroups go round the 8 XCDs; a row's go to one, whose L2 then serves its history (as many rows as come in
  // eights; 64 rows of 32,000 with histories of 8000 12.7 / 11.1 us, of 128,257 with 8000 27.0 / 26.2, with 100 level).
  int row = blockIdx.x / a.slices, part = blockIdx.x % a.slices;
  if (row < (a.rows & ~7)) {
    const int over = (blockIdx.x >> 3) / a.slices;
    row = 8 * over + (blockIdx.x & 7), part = (blockIdx.x >> 3) - over * a.slices;
  }
  const float* in = a.in + row * a.ld;
  float* out = a.out + row * a.out_ld;
  // The slice's first logit; the first slice begins up to three before the row.
  const int v0 = part * kSlice - (VEC ? static_cast<int>(reinterpret_cast<uintptr_t>(in) / 4 % 4) : 0);
  const auto at = [&](int i) { return VEC ? 4 * (threadIdx.x + i * THREADS) : static_cast<int>(threadIdx.x) + 4 * i * THREADS; };
  // The history in pieces of four tokens a thread (rows begin at any word), kAhead of them in flight and the first
  // before the logits: loads return in order, and the history is worked on while the logits come.
  constexpr int kAhead = 4;
  struct __attribute__((packed, aligned(4))) Four {
    int token[4];
  };
  const int len = a.history ? static_cast<int>(min(static_cast<int64_t>(max(a.history_len[row], 0)), a.history_stride)) : 0;
  const int prompt = a.prompt_len ? a.prompt_len[row] : 0;
  const int* h = a.history + row * a.history_stride;
  Four said[kAhead];
  const auto tokens_at = [&](int i, int j0) {  // piece i from token j0 on, the same for all threads
    const int j = j0 + 4 * static_cast<int>(threadIdx.x);
    if (j0 >= len) return;
    if (j + 3 < len) {
      said[i] = *reinterpret_cast<const Four*>(h + j);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) said[i].token[e] = j + e < len ? h[j + e] : -1;
    }
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) tokens_at(i, 4 * i * THREADS);
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
        const int u = v + (VEC ? e : e * THREADS);
        x[i][e] = u >= 0 && u < a.vocab ? in[u] : 0.0f;
      }
    }
  }
  const int64_t bias_at = row * a.bias_stride;
  const int biases = BIAS ? static_cast<int>(min(static_cast<int64_t>(max(a.bias_len[row], 0)), a.bias_stride)) : 0;
  int named = static_cast<int>(threadIdx.x) < biases ? a.bias_tokens[bias_at + threadIdx.x] : -1;
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
  const auto clear = [&] {
#pragma unroll
    for (int i = 0; i < kVec; ++i) reinterpret_cast<uint4v*>(s_word)[threadIdx.x + i * THREADS] = uint4v{0, 0, 0, 0};
    __syncthreads();
  };
  // A thread's words, laid out as its logits are.
  const auto words_of = [&](int i, unsigned (&w)[4]) {
    if (VEC) {
      const uint4v s = reinterpret_cast<const uint4v*>(s_word)[threadIdx.x + i * THREADS];
      w[0] = s[0], w[1] = s[1], w[2] = s[2], w[3] = s[3];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = s_word[at(i) + e * THREADS];
    }
  };
  // A token's place among the slice's from its first in the vocabulary on: n and more for any other token, one
  // below 0 or past the vocabulary too.
  const unsigned from = static_cast<unsigned>(max(v0, 0)), n = static_cast<unsigned>(max(0, min(v0 + kSlice, a.vocab) - max(v0, 0)));
  const auto place = [&](int token) { return static_cast<unsigned>(token) - from; };
  unsigned* const words = s_word + (max(v0, 0) - v0);
  if (len > 0) {
    const float rep = a.repetition ? a.repetition[row] : 1.0f;
    const float freq = a.frequency ? a.frequency[row] : 0.0f, pres = a.presence ? a.presence[row] : 0.0f;
    clear();
    for (int j0 = 0; j0 < len; j0 += 4 * kAhead * THREADS) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int j = j0 + 4 * i * THREADS;
        if (j >= len) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned p = place(said[i].token[e]);
          if (p < n) {
            if (j + 4 * static_cast<int>(threadIdx.x) + e < prompt)
              atomicOr(&words[p], 0x80000000u);
            else
              atomicAdd(&words[p], 1u);
          }
        }
        tokens_at(i, j + 4 * kAhead * THREADS);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      unsigned seen[4];
      words_of(i, seen);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (seen[e]) {
          // Each step rounded by itself, in the order of the formula.
          float y = x[i][e];
          y = y > 0.0f ? y / rep : mul_rounded(y, rep);
          if (const unsigned count = seen[e] & 0x7fffffffu) y = y - mul_rounded(freq, static_cast<float>(count)) - pres;
          x[i][e] = y;
        }
      }
    }
  }
  if (BIAS && biases > 0) {
    __syncthreads();  // the history's words have been read
    clear();
    for (int j = threadIdx.x; j < biases; j += THREADS) {
      const unsigned p = place(named);
      if (p < n) atomicMax(&words[p], static_cast<unsigned>(j + 1));
      named = j + THREADS < biases ? a.bias_tokens[bias_at + j + THREADS] : -1;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      unsigned by[4];
      words_of(i, by);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (by[e]) x[i][e] += a.bias_values[bias_at + by[e] - 1];
    }
  }
  unsigned long long best = 0;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = v0 + at(i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int u = v + (VEC ? e : e * THREADS);
      if (u >= 0 && u < a.vocab) {
        const unsigned word = !VEC ? (mask_row >= 0 ? mask[u >> 5] : ~0u) : u >> 5 == max(v, 0) >> 5 ? lo[i] : hi[i];
        if (!((word >> (u & 31)) & 1u)) x[i][e] = -INFINITY;
        const unsigned long long k = token_key(x[i][e], u);
        best = k > best ? k : best;
      }
    }
  }
  unsigned long long* const record = a.records + row * a.record;
  if (a.next) {
    best = block_best<THREADS>(best, s_best);
    if (threadIdx.x == 0) {
      __hip_atomic_store(&record[1 + part], best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __builtin_amdgcn_s_waitcnt(0);
      s_last = __hip_atomic_fetch_add(&record[0], 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.slices - 1ull;
    }
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = v0 + at(i);
    if (VEC && v >= 0 && v + 3 < a.vocab) {
      *reinterpret_cast<float4*>(out + v) = float4{x[i][0], x[i][1], x[i][2], x[i][3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int u = v + (VEC ? e : e * THREADS);
        if (u >= 0 && u < a.vocab) out[u] = x[i][e];
      }
    }
  }
  if (!a.next) return;
  __syncthreads();
  if (!s_last) return;
  // The row's last workgroup takes the best of all slices and leaves the record zero again, for calls of any shape.
  best = 0;
  for (int p = threadIdx.x; p <= a.slices; p += THREADS) {
    const unsigned long long k = __hip_atomic_load(&record[p], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(&record[p], 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (p) best = k > best ? k : best;
  }
  best = block_best<THREADS>(best, s_best);
  if (threadIdx.x == 0) a.next[row] = best ? static_cast<int>(0xffffffffu - static_cast<unsigned>(best)) : -1;
}

// Logits of a workgroup: one 16-byte load a thread while that makes few workgroups, else two. Each workgroup reads
// its row's whole history, so where that may be long it has twice the threads. Measured (us; histories of 2000, one / two /
// four loads of 256 threads): 1 x 32,000 7.2 / 8.0 / 10.0, 8 x 128,256 9.6 / 9.0 / 10.7, 48 x 32,000 10.5 / 9.9 / 12.3, 32 x
// 128,256 18.6 / 14.9 / 14.7. 256 / 512 threads: 64 x 128,257 with 100 18.9 / 19.8, with 4000 23.0 / 23.4, with 8000 and 300
// biases 27.6 / 26.2, with 16,000 31.3 / 28.1, 1 x 128,256 with 120,000 32 / 21; 1024 threads are slower by 1-15%.
int threads_of(int64_t history_stride) { return history_stride > 4096 ? 512 : 256; }
int slice_of(int rows, int vocab, int threads) {
  const int one = 4 * threads;
  return static_cast<int64_t>(rows) * ((vocab + one - 1) / one) <= 512 ? one : 2 * one;
}
// Slices of a row, which may begin up to three logits into its first one.
int slices_of(int vocab, int slice) { return static_cast<int>((static_cast<int64_t>(vocab) + 3 + slice - 1) / slice); }

// A row's record has 256-byte lines of its own: counts of several rows in one line are taken one after
// another, 10 ns each (with all counts side by side 64 rows of 128,257 logits took 37 us, with a line each 32; in records of a
// row's own without whole lines they are level with this).
int64_t record_words(int vocab, int slice) { return (1 + static_cast<int64_t>(slices_of(vocab, slice)) + 31) / 32 * 32; }

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
  const StepArgs a{cached, fresh, shared, group_seqs, n_seqs, n_groups, block_size, div_by(block_size), tables, table_stride,
                   static_cast<int>(std::min<int64_t>(static_cast<int64_t>(table_stride) * block_size, INT32_MAX)), free_blocks, free_count, max_rows, row_off, last_row, table_off, pos, seq, slot,
                   reinterpret_cast<int4*>(dec_meta), reinterpret_cast<int4*>(groups), totals};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const auto go = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, dim3(1), dim3(threads), 0, s, a); };
  const bool carried = free_count >= totals && free_count < totals + 4;
  if (max_rows > kWideRows && n_seqs <= kRowOffsets && !carried) {
    const auto wide = [&](auto kernel, int threads) {
      hipLaunchKernelGGL(kernel, dim3((max_rows - 1) / threads + 1), dim3(threads), 0, s, a);
    };
    // Measured (us, 256 / 512 / 1024 threads): 64 sequences and 8 prompts of 512 4.8 / 4.8 / 5.3, 511 and 40 of 700 6.5 / 5.5 /
    // 6.1, 2000 and 40 of 512 12.9 / 9.4 / 8.6 (now 8.2), 4000 21.5 / 14.3 / 12.4 (11.7).
    RH_TRY_LAUNCH(n_seqs <= 256    ? wide(step_wide_kernel<256>, 256)
                  : n_seqs <= 1024 ? wide(step_wide_kernel<512>, 512)
                                   : wide(step_wide_kernel<1024>, 1024));
  } else if (max_rows > kOneLaunch) {
    RH_TRY_LAUNCH(n_seqs <= 256 ? go(step_tables_kernel<256, false>, 256) : go(step_tables_kernel<1024, false>, 1024));
    RH_TRY_LAUNCH(hipLaunchKernelGGL(step_rows_kernel, dim3((max_rows + kRowThreads - 1) / kRowThreads), dim3(kRowThreads), 0, s, a));
  } else {
    RH_TRY_LAUNCH(n_seqs <= 256 && max_rows <= 1024 ? go(step_tables_kernel<256, true>, 256) : go(step_tables_kernel<1024, true>, 1024));
  }
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
                 static_cast<half_t*>(vpool), static_cast<half_t*>(q_out), q_scale, heads, kv_heads, head_dim, block_size, div_by(block_size), {}};
  const int total = heads + 2 * kv_heads;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const auto of_lanes = [&](auto lanes) -> int {
    constexpr int LANES = decltype(lanes)::value;
    const auto go = [&](auto kernel, int per_wave) -> int {
      const int64_t sets = (total + per_wave - 1) / per_wave, wgs = (T * sets + kThreads / kWave - 1) / (kThreads / kWave);
      RH_REQUIRE(T * sets + kThreads < (int64_t{1} << 31), "qk_norm: too many rows");
      QkArgs b = a;
      b.by_sets = div_by(static_cast<int>(sets));
      RH_TRY_LAUNCH(hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(wgs)), dim3(kThreads), 0, s, b));
      return 0;
    };
    constexpr int PER = kWave / LANES;
    // Two sets of heads a wave once that leaves enough waves. Measured (us, one / two; bound by latency
    // below, by memory above): 48 rows of 32/4 heads of 64 3.2 / 3.6, 256 3.6 / 3.7, 512 4.2 / 4.3, 2047 10.2 /
    // 9.6 (floor 6.1), 4096 of 32/8 heads of 128 37.5 / 32.5 (29); three to five sets are level.
    const bool many = static_cast<int64_t>(T) * total * LANES >= 150000;
    if (planes == 1 && !scale) return many ? go(qk_norm_kernel<LANES, 2, true>, 2 * PER) : go(qk_norm_kernel<LANES, 1, true>, PER);
    return many ? go(qk_norm_kernel<LANES, 2, false>, 2 * PER) : go(qk_norm_kernel<LANES, 1, false>, PER);
  };
  if (head_dim <= 32) return of_lanes(std::integral_constant<int, 4>{});
  if (head_dim <= 64) return of_lanes(std::integral_constant<int, 8>{});
  if (head_dim <= 128) return of_lanes(std::integral_constant<int, 16>{});
  if (head_dim <= 256) return of_lanes(std::integral_constant<int, 32>{});
  return of_lanes(std::integral_constant<int, 64>{});
}

size_t rh_process_logits_workspace(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0) return 0;
  return static_cast<size_t>(rows) * record_words(vocab, slice_of(rows, vocab, 256)) * 8;  // 512 threads have fewer slices
}

int rh_process_logits(const float* logits, int64_t ld, int rows, int vocab, const int* history, int64_t history_stride,
                      const int* history_len, const int* prompt_len, const float* repetition, const float* frequency,
                      const float* presence, const int* bias_tokens, const float* bias_values, int64_t bias_stride,
                      const int* bias_len, const uint32_t* masks, int64_t mask_stride, const int* mask_of, float* out,
                      int64_t out_ld, int* next, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows == 0) return 0;
  RH_REQUIRE(rows > 0 && vocab > 0 && vocab < kSumCap && ld >= vocab && out_ld >= vocab, "process_logits: bad sizes");
  RH_REQUIRE(logits && out, "process_logits: missing pointer");
  RH_REQUIRE(logits != out || ld == out_ld, "process_logits: in place needs one row stride");
  RH_REQUIRE(!history || (history_len && history_stride >= 0 && history_stride < kSumCap),
             "process_logits: a history needs its lengths and a stride below 2^30");
  RH_REQUIRE(history || !(prompt_len || repetition || frequency || presence), "process_logits: penalties need a history");
  RH_REQUIRE(!bias_tokens || (bias_values && bias_len && bias_stride >= 0 && bias_stride < kSumCap),
             "process_logits: biases need values, lengths and a stride below 2^30");
  RH_REQUIRE(!masks || mask_stride >= (static_cast<int64_t>(vocab) + 31) / 32, "process_logits: a mask row holds a bit for each token");
  const int threads = threads_of(history ? history_stride : 0), slice = slice_of(rows, vocab, threads), slices = slices_of(vocab, slice);
  RH_REQUIRE(static_cast<int64_t>(rows) * slices < (int64_t{1} << 31), "process_logits: too many rows");
  RH_REQUIRE(!next || (workspace && workspace_bytes >= rh_process_logits_workspace(rows, vocab) &&
                       reinterpret_cast<uintptr_t>(workspace) % 8 == 0),
             "process_logits: next needs an 8-byte aligned workspace of rh_process_logits_workspace bytes");
  const LogitArgs a{logits, ld, rows, vocab, slices, history, history_stride, history_len, prompt_len, repetition, frequency,
              presence, bias_tokens, bias_values, bias_stride, bias_len, masks, mask_stride, mask_of, out, out_ld, next,
              static_cast<unsigned long long*>(workspace), record_words(vocab, slice)};
  // Every row lies alike in logits and out: equal strides, or both whole 16-byte steps.
  const bool vec = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(out)) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(logits) % 4 == 0 && (ld - out_ld) % 4 == 0;
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(rows * slices), dim3(threads), 0, static_cast<hipStream_t>(stream), a);
  };
  const auto of_loads = [&](auto bias, auto aligned) {
    constexpr bool B = decltype(bias)::value, V = decltype(aligned)::value;
    const bool one = slice == 4 * threads;
    if (threads == 512)
      one ? go(process_logits_kernel<B, V, 1, 512>) : go(process_logits_kernel<B, V, 2, 512>);
    else
      one ? go(process_logits_kernel<B, V, 1, 256>) : go(process_logits_kernel<B, V, 2, 256>);
  };
  if (bias_tokens) {
    RH_TRY_LAUNCH(vec ? of_loads(std::true_type{}, std::true_type{}) : of_loads(std::true_type{}, std::false_type{}));
  } else {
    RH_TRY_LAUNCH(vec ? of_loads(std::false_type{}, std::true_type{}) : of_loads(std::false_type{}, std::false_type{}));
  }
  return 0;
}

}  // extern "C"
