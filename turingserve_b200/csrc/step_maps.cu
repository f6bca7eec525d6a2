// A step's maps out of its requests' lengths and the page tables that stay on the GPU.
//
// Request b has row r[b] of the tables (-1: a row that only pads the batch), start[b] tokens in the cache and brings q[b]:
//   q_start = 0, q[0], q[0] + q[1], ...      seq_lens[b] = start[b] + q[b]  (0 for padding)
//   token i of request b:  token_request = b, position p = start[b] + i,
//                          slot[g] = tables[g, r, p / page] * page + p % page  (-1 for padding)
//   block_tables[g, b, i] = tables[g, r, i] for i < ceil(seq_lens[b] / page), else 0, the page that nobody owns
// after `updates` (group, row, index, page) have gone into the tables; of updates of the same place the last one holds.
//
// One block a request (several where tables are wide or portions long), which sums the lengths before its own, puts its row's updates in
// place and writes its tokens and its table rows; one more block puts the others in place, of rows that are not in the step.
// Only the update that holds in the end is ever written, so blocks that write the same place write the same value.  One launch
// whatever the step: 8 requests of 2,048 tokens are bound by its latency (2.2 us in a graph, of which a launch is most); 129 requests
// with two tables of 2,048 entries and a portion of 1,920 tokens move 3 MB (4.9 us).  The kernel does not let kernels behind it start early: they
// may read the maps before they wait.
#include "common.cuh"

namespace {

constexpr int THREADS = 256, UPDATES = 512, ROWS_HELD = 1024;

struct MapArgs {
  const int* requests;                 // [3][B]: table row, tokens before, tokens brought
  const int4* updates;                 // [U]
  int* tables;                         // [G][R][P]
  int *q_start, *seq_lens, *token_request, *positions, *slots, *block_tables;
  long long slots_g, tables_g;         // elements between the groups of slots and of block_tables
  int B, T, U, G, R, P, W, page;
};

__global__ void __launch_bounds__(THREADS) step_maps_kernel(const MapArgs a) {
  pdl_wait();
  const int b = blockIdx.x, tid = threadIdx.x;
  const bool extra = b == a.B;
  if (extra && blockIdx.y > 0) return;
  __shared__ int sums[THREADS / 32];
  __shared__ int4 up_s[UPDATES];
  __shared__ int rows_s[ROWS_HELD];
  if (extra)
    for (int i = tid; i < min(a.B, ROWS_HELD); i += THREADS) rows_s[i] = a.requests[i];
  const int upto = extra ? a.B : b;
  int mine = 0;
  for (int i = tid; i < upto; i += THREADS) mine += max(0, a.requests[2 * a.B + i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if ((tid & 31) == 0) sums[tid >> 5] = mine;
  const int row = extra ? -1 : a.requests[b], start = extra ? 0 : a.requests[a.B + b], n = extra ? 0 : max(0, a.requests[2 * a.B + b]);
  const bool real = row >= 0 && row < a.R;
  __shared__ int segments, doubt;
  if (tid == 0) segments = doubt = 0;
  auto fetch = [&](int base, int count) {
    __syncthreads();
    for (int i = tid; i < count; i += THREADS) up_s[i] = a.updates[base + i];
    __syncthreads();
  };
  // Which updates this block puts in place: its row's; the extra block those of rows that no request has.
  auto mine_too = [&](const int4& up) {
    if (up.x < 0 || up.x >= a.G || up.y < 0 || up.y >= a.R || up.z < 0 || up.z >= a.P) return false;
    if (!extra) return up.y == row;
    bool owned = false;
    const int here = min(a.B, ROWS_HELD);
#pragma unroll 8
    for (int i = 0; i < here; ++i) owned |= rows_s[i] == up.y;
    for (int i = here; i < a.B; ++i) owned |= a.requests[i] == up.y;
    return !owned;
  };
  // One place twice?  Not if a row's updates stand next to each other, in ascending order; only otherwise every one is held against those
  // behind it (120 of one row: 12 us of 16).
  if (!extra)
    for (int base = 0; base < a.U; base += UPDATES) {
      const int count = min(UPDATES, a.U - base);
      fetch(base, count);
      for (int i = tid; i < count; i += THREADS) {
        const int4 up = up_s[i];
        if (up.y != row) continue;
        const int4 prev = i > 0 ? up_s[i - 1] : (base > 0 ? a.updates[base - 1] : make_int4(0, -2, 0, 0));
        if (prev.y != row) atomicAdd(&segments, 1);
        else if (prev.x > up.x || (prev.x == up.x && prev.z >= up.z)) doubt = 1;
      }
    }
  for (int base = 0; base < a.U; base += UPDATES) {
    const int count = min(UPDATES, a.U - base);
    if (extra || a.U > UPDATES) fetch(base, count);
    else __syncthreads();
    const bool look = extra || doubt || segments > 1;
    for (int i = tid; i < count; i += THREADS) {
      const int4 up = up_s[i];
      if (!mine_too(up)) continue;
      bool holds = true;                                           // no later one of the same place
      if (look) {
#pragma unroll 4
        for (int w = i + 1; w < count; ++w) holds = holds && (up_s[w].x != up.x || up_s[w].y != up.y || up_s[w].z != up.z);
        for (int w = base + count; w < a.U && holds; ++w) {
          const int4 later = a.updates[w];
          holds = later.x != up.x || later.y != up.y || later.z != up.z;
        }
      }
      if (holds) a.tables[((size_t)up.x * a.R + up.y) * a.P + up.z] = up.w;
    }
  }
  __syncthreads();
  int first = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) first += sums[i];
  if (extra) {                                                     // tokens that no request brings: none, where the lengths add up
    if (tid == 0) a.q_start[0] = 0;
    for (int t = first + tid; t < a.T; t += THREADS) {
      a.token_request[t] = 0;
      a.positions[t] = 0;
      for (int g = 0; g < a.G; ++g) a.slots[g * a.slots_g + t] = -1;
    }
    return;
  }
  const int len = real ? start + n : 0, live = min(len > 0 ? (len + a.page - 1) / a.page : 0, a.P);
  if (tid == 0 && blockIdx.y == 0) {
    a.q_start[b + 1] = first + n;
    a.seq_lens[b] = len;
  }
  const int at = blockIdx.y * THREADS + tid, step = gridDim.y * THREADS, tokens = min(n, a.T - first);
  for (int g = 0; g < a.G; ++g) {
    const int* tab = a.tables + ((size_t)g * a.R + (real ? row : 0)) * a.P;
    int* bt = a.block_tables + g * a.tables_g + (size_t)b * a.W;
    for (int i0 = at; i0 < a.W; i0 += 4 * step) {                  // four entries at a time on their way
      int v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = i0 + u * step < live ? tab[i0 + u * step] : 0;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + u * step < a.W) bt[i0 + u * step] = v[u];
    }
    int* slots = a.slots + g * a.slots_g + first;
    for (int i0 = at; i0 < tokens; i0 += 4 * step) {
      int v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int p = start + i0 + u * step, lp = p / a.page;
        const bool there = i0 + u * step < tokens && real && p >= 0 && lp < a.P;
        v[u] = there ? tab[lp] * a.page + p % a.page : -1;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + u * step < tokens) slots[i0 + u * step] = v[u];
    }
  }
  for (int i = at; i < tokens; i += step) {
    a.token_request[first + i] = b;
    a.positions[first + i] = start + i;
  }
}

}  // namespace

struct MapCall {
  const int *requests, *updates;
  int *tables, *q_start, *seq_lens, *token_request, *positions, *slots, *block_tables;
  long long slots_g, tables_g;
  int B, T, U, G, R, P, W, page;
};

TS_API int ts_step_maps_record() { return (int)sizeof(MapCall); }

// (the arguments as one record: see kv_write_q8.cu)
TS_API int ts_step_maps(const void* record, void* stream) {
  const MapCall& c = *(const MapCall*)record;
  const int B = c.B, T = c.T, U = c.U, G = c.G, R = c.R, P = c.P, W = c.W, page = c.page;
  if (B < 0 || T < 0 || U < 0 || G < 0 || R <= 0 || P <= 0 || W < 0 || page <= 0)
    TS_REFUSE(TS_ERR_SHAPE, "ts_step_maps: B=%d T=%d U=%d G=%d R=%d P=%d W=%d page=%d", B, T, U, G, R, P, W, page);
  if (((uintptr_t)c.updates & 15) != 0) TS_REFUSE(TS_ERR_ALIGN, "ts_step_maps: updates must be 16-byte aligned");
  MapArgs a = {c.requests, (const int4*)c.updates, c.tables, c.q_start, c.seq_lens, c.token_request, c.positions, c.slots, c.block_tables,
               c.slots_g, c.tables_g, B, T, U, G, R, P, W, page};
  // blocks a request: one for every 1,024 entries of its tables, or tokens, at most (one block a request with two tables of 2,048
  // entries: 24 us for 129 requests)
  const long long most = (long long)W * G > T - B ? (long long)W * G : T - B;
  const int parts = most <= 1024 ? 1 : (most >= 8192 ? 8 : (int)((most + 1023) / 1024));
  ts_launch(step_maps_kernel, dim3(B + 1, parts), dim3(THREADS), 0, (cudaStream_t)stream, a);
  TS_LAUNCH_CHECK();
}
