// The tables of a serving step, built on the GPU from the requests' new lengths: pages of the paged cache taken from a stack
// of free ones and entered in the block table, and for every token of the step its request, position and cache slot; and
// the way back (finished requests, rejected drafts).
//
//   start = exclusive sum of new[b];  need_b = max(0, min(ceil((lens_b + new_b) / bs), W) - held_b)
//   off   = exclusive sum of need;    page i of all needed ones = free[count - 1 - i], while i < count
//   token t of request b: position lens_b + t - start_b, slot table[b][position / bs] * bs + position % bs, -1 without a page
//   trim: lens_b = min(lens_b, keep_b); the R pages behind ceil(lens_b / bs) go back, page i to free[count + R - 1 - i]
//
// Latency is all there is (a decode step moves 25 KB), so a call is one launch: every workgroup reads all requests and forms
// both sums for itself in LDS; a token's page comes from the table where the request held it and from the stack where it
// is new, so nothing waits for the table's new entries. lens, held and the count change only after every workgroup
// has read them: the one that arrives last at a counter in the pool's state writes them (and clears the counter).
#include "spmla_common.h"
#include "spmla_quant.h"

namespace spmla {
namespace pages {

constexpr int MAXM = 8192;            // requests (two sums of them in LDS)
constexpr int TPB = 1024;

struct Pool {
  int* lens; int* held; int* table; long long t_st; int W;
  int* free; int P; int* state;       // state: free pages, pages missing in the last step, arrivals
  int bs;
};

__device__ inline int sat_add(int a, int b) {       // both >= 0
  const uint32_t s = (uint32_t)a + (uint32_t)b;
  return s > 0x7fffffffu ? 0x7fffffff : (int)s;
}
__device__ inline int pages_of(int tokens, int bs, int W) {
  const int n = tokens / bs + (tokens % bs != 0);
  return n < W ? n : W;
}

// Exclusive sums (saturating) of v[0..M) in place, the total behind them; blockDim.x a multiple of 64.
__device__ inline void scan(int* v, int M, int* part) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, nw = blockDim.x >> 6;
  int base = 0;
  for (int at = 0; at < M; at += blockDim.x) {
    const int x = at + tid < M ? v[at + tid] : 0;
    int s = x;                                      // (wave_incl_scan with sums that saturate)
    s = sat_add(s, __builtin_amdgcn_update_dpp(0, s, 0x111, 0xf, 0xf, false));
    s = sat_add(s, __builtin_amdgcn_update_dpp(0, s, 0x112, 0xf, 0xf, false));
    s = sat_add(s, __builtin_amdgcn_update_dpp(0, s, 0x114, 0xf, 0xf, false));
    s = sat_add(s, __builtin_amdgcn_update_dpp(0, s, 0x118, 0xf, 0xf, false));
    s = sat_add(s, __builtin_amdgcn_update_dpp(0, s, 0x142, 0xa, 0xf, false));
    s = sat_add(s, __builtin_amdgcn_update_dpp(0, s, 0x143, 0xc, 0xf, false));
    int ex = __shfl_up(s, 1);                       // (not s - x: the sums stay ascending where they saturate)
    ex = lane ? ex : 0;
    if (lane == 63) part[w] = s;
    __syncthreads();
    int before = base, all = base;
    for (int i = 0; i < nw; ++i) {
      if (i == w) before = all;
      all = sat_add(all, part[i]);
    }
    if (at + tid < M) v[at + tid] = sat_add(before, ex);
    base = all;
    __syncthreads();
  }
  if (tid == 0) v[M] = base;
  __syncthreads();
}

// The last b with v[b] <= x (v ascending, v[0] = 0, x < v[M]).
__device__ inline int find(const int* v, int M, int x) {
  int lo = 0, hi = M;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Whether this workgroup is the last to have read the pool (its counter is cleared then).
__device__ inline bool last_reader(int* state) {
  __shared__ int last;
  __syncthreads();                                  // every thread's reads are done
  if (gridDim.x == 1) return true;
  if (threadIdx.x == 0) {
    last = __hip_atomic_fetch_add(state + 2, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    if (last) __hip_atomic_store(state + 2, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return last;
}

__device__ inline int clamp0(int x, int hi) { return x < 0 ? 0 : x > hi ? hi : x; }

__global__ void __launch_bounds__(TPB) step_kernel(const int* fresh, int M, Pool p, int n, int* start, int* req, long long* positions,
                                                   long long* slots) {
  extern __shared__ int lds[];
  int* st = lds;                                    // [M + 1] sums of the new tokens
  int* off = lds + M + 1;                           // [M + 1] sums of the needed pages
  int* lens = lds + 2 * M + 2;                      // [M] lengths and pages before the step
  int* helds = lds + 3 * M + 2;
  int* part = lds + 4 * M + 2;
  const int tid = threadIdx.x, G = gridDim.x;
  for (int b = tid; b < M; b += blockDim.x) {
    const int x = clamp0(fresh[b], 0x7fffffff), len = clamp0(p.lens[b], 0x7fffffff), held = clamp0(p.held[b], p.W);
    const int want = pages_of(sat_add(len, x), p.bs, p.W);
    st[b] = x;
    off[b] = want > held ? want - held : 0;
    lens[b] = len;
    helds[b] = held;
  }
  const int count = clamp0(p.state[0], p.P);
  __syncthreads();
  scan(st, M, part);
  scan(off, M, part);
  const int total = off[M], got = total < count ? total : count;

  const int at0 = blockIdx.x * blockDim.x + tid, step = G * blockDim.x;
  for (int t = at0; t < n; t += step) {
    int b = M - 1;
    long long pos = 0, slot = -1;
    if (t < st[M]) {
      b = find(st, M, t);
      const int len = lens[b], held = helds[b];
      pos = (long long)len + (t - st[b]);
      const uint32_t c = (uint32_t)pos / (uint32_t)p.bs;           // (two lengths below 2^31: 32 bits without a sign)
      int page = -1;
      if (c < (uint32_t)held) {
        page = p.table[b * p.t_st + c];
      } else if (c < (uint32_t)p.W) {
        const int i = (int)c - held;                // of the pages that the request takes
        if (i < off[b + 1] - off[b] && i < got - off[b]) page = p.free[count - 1 - (off[b] + i)];
      }
      if (page >= 0) slot = (long long)page * p.bs + (uint32_t)pos % (uint32_t)p.bs;
    }
    req[t] = b;
    positions[t] = pos;
    slots[t] = slot;
  }
  for (int i = at0; i < got; i += step) {
    const int b = find(off, M, i), c = helds[b] + (i - off[b]);
    p.table[b * p.t_st + c] = p.free[count - 1 - i];
  }
  for (int b = at0; b <= M; b += step) start[b] = st[b];

  if (!last_reader(p.state)) return;
  for (int b = tid; b < M; b += blockDim.x) {
    const int need = off[b + 1] - off[b], left = got - off[b];
    p.lens[b] = sat_add(lens[b], st[b + 1] - st[b]);
    p.held[b] = helds[b] + (left < need ? clamp0(left, need) : need);
  }
  if (tid == 0) {
    p.state[0] = count - got;
    p.state[1] = total - got;
  }
}

__global__ void __launch_bounds__(TPB) trim_kernel(const int* keep, int M, Pool p) {
  extern __shared__ int lds[];
  int* off = lds;                                   // [M + 1] sums of the pages that go back
  int* lefts = lds + M + 1;                         // [M] pages that stay
  int* part = lds + 2 * M + 1;
  const int tid = threadIdx.x, G = gridDim.x;
  auto left_of = [&](int b, int& len) {             // pages that request b keeps
    len = clamp0(p.lens[b], 0x7fffffff);
    const int k = clamp0(keep[b], 0x7fffffff);
    len = k < len ? k : len;
    const int held = clamp0(p.held[b], p.W), want = pages_of(len, p.bs, p.W);
    return want < held ? want : held;
  };
  for (int b = tid; b < M; b += blockDim.x) {
    int len;
    const int left = left_of(b, len);
    off[b] = clamp0(p.held[b], p.W) - left;
    lefts[b] = left;
  }
  const int count = clamp0(p.state[0], p.P);
  __syncthreads();
  scan(off, M, part);
  const int R = off[M];
  const int at0 = blockIdx.x * blockDim.x + tid, step = G * blockDim.x;
  for (int i = at0; i < R; i += step) {
    const int b = find(off, M, i);
    int* e = p.table + b * p.t_st + lefts[b] + (i - off[b]);
    const long long to = (long long)count + R - 1 - i;
    if (to < p.P) p.free[to] = *e;                  // (a pool whose pages are all its own has room)
    *e = -1;
  }
  if (!last_reader(p.state)) return;
  for (int b = tid; b < M; b += blockDim.x) {
    int len;
    const int left = left_of(b, len);
    p.lens[b] = len;
    p.held[b] = left;
  }
  if (tid == 0) p.state[0] = clamp0(sat_add(count, R), p.P);
}

int check(const int* in, int M, const Pool& p) {
  if (M <= 0 || p.W < 0 || p.P < 0 || p.bs <= 0 || (M > 1 && p.t_st < p.W)) return SPMLA_EARG;
  if (!in || !p.lens || !p.held || !p.state || (p.W && !p.table) || (p.P && !p.free)) return SPMLA_EARG;
  if (M > MAXM) return SPMLA_ELIMIT;
  return SPMLA_OK;
}
int threads_of(long long work) { return work <= 256 ? 256 : TPB; }
constexpr int most_lds(int per) { return (per * MAXM + 2 + TPB / 64) * 4; }

}  // namespace pages
}  // namespace spmla

using namespace spmla;
using namespace spmla::pages;

extern "C" {

int spmla_page_step(const int* fresh, int M, int* lens, int* held, int* table, long long table_st, int W, int* free, int P,
                    int* state, int block_size, int n, int* start, int* req, long long* positions, long long* slots, void* stream) {
  const Pool p{lens, held, table, table_st, W, free, P, state, block_size};
  if (const int rc = check(fresh, M, p)) return rc;
  if (n < 0 || !start || (n && (!req || !positions || !slots))) return SPMLA_EARG;
  static DynLds attr;
  static Launcher go;
  if (const int rc = attr.ensure((const void*)step_kernel, most_lds(4))) return rc;
  const int tpb = threads_of(n > M ? n : M);
  int G = (n + tpb - 1) / tpb;
  G = G < 1 ? 1 : G > 64 ? 64 : G;
  return go((const void*)step_kernel, dim3((unsigned)G), tpb, (4 * M + 2 + TPB / 64) * 4, (hipStream_t)stream, fresh, M, p, n, start, req,
            positions, slots);
}

int spmla_page_trim(const int* keep, int M, int* lens, int* held, int* table, long long table_st, int W, int* free, int P, int* state,
                    int block_size, void* stream) {
  const Pool p{lens, held, table, table_st, W, free, P, state, block_size};
  if (const int rc = check(keep, M, p)) return rc;
  static DynLds attr;
  static Launcher go;
  if (const int rc = attr.ensure((const void*)trim_kernel, most_lds(2))) return rc;
  const long long most = (long long)M * W;                       // pages that may go back
  const int tpb = threads_of(most / 8 > M ? most / 8 : M);
  int G = (int)((most + 32 * TPB - 1) / (32 * TPB) < 32 ? (most + 32 * TPB - 1) / (32 * TPB) : 32);
  G = G < 1 ? 1 : G;
  return go((const void*)trim_kernel, dim3((unsigned)G), tpb, (2 * M + 1 + TPB / 64) * 4, (hipStream_t)stream, keep, M, p);
}

}  // extern "C"
