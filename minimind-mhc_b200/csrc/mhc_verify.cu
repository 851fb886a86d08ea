// Verification of drafted tokens against the target's probabilities.
//
// A sequence's drafted tokens are a tree whose parents come before their children, so one
// walk over the rows in their order settles it: a row whose parent is the last kept node
// is tested, every other one is passed over.
//
//   kept  if u mass q(x) < rest(x)       then rest = p of that node, mass = 1
//   else  rest = max(rest - mass q, 0), mass = sum of rest
//
// rest is not stored: after any number of refused children of one node
//   rest = max(p - A q, 0),   A = the sum of the masses so far,
// since what one refusal has taken to 0 the next ones leave there.  A refusal is
// therefore one pass over a row of p and of q, and the probabilities of all tests are two
// numbers for every row, fetched at once before the walk.  The next token is the first
// whose cumulative sum of rest passes u sum(rest): the last pass leaves the sum of every
// warp's piece of the vocabulary, so only one warp reads its piece again.
//
// Whole numbers come out, so the sums are fp64 (fp32 ones would move the borders by 1e-7 and
// with them a token of every few thousand draws); inputs are read as they are.
//
// A cluster of up to eight blocks owns a sequence, each block a piece of the vocabulary
// of neighbouring tokens; the blocks take the same walk and exchange one sum a pass through
// distributed shared memory, added up in the same order by each.
//
// Measured: 32 sequences with trees of up to 32 rows, 100,003 tokens: 29 us, of which a pass over
// both rows takes 4.6 (26 MB for all sequences, HBM or L2) and the slowest sequence has three; a
// chain of six over 6400 tokens 8 us: launch, two chains of loads (rows, then their probabilities)
// and one pass.  The trees without a draft take 30 us (every element is held against the refused
// tokens), with 16-bit probabilities 25 where fp32 ones that L2 holds take 24.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mhc_b200.h"
#include "mhc_device.cuh"
#include "mhc_dispatch.cuh"
#include "mhc_kernels.h"

namespace mhc {
namespace verify {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_NODES = 1024;
constexpr int MAX_CLUSTER = 8;
constexpr int AT_ONCE = 8;  // elements that a lane has under way

struct Args {
  const int64_t *tokens;
  const int32_t *parents, *cu;
  int batch, T;
  const void *target, *draft;
  int64_t ts, ds;
  int V;
  const float *random;
  int32_t *path, *kept;
  int64_t *next;
};

struct Shared {
  int parent[MAX_NODES], token[MAX_NODES], way[MAX_NODES], refused[MAX_NODES];
  float p[MAX_NODES], q[MAX_NODES], u[MAX_NODES];
  double warp_sum[WARPS];
  double total[2][MAX_CLUSTER];  // of every block of the cluster; two passes' apart
};

// an entry of a row as it counts: NaN and what is negative are 0
template <typename T>
__device__ __forceinline__ float entry(const T *row, int64_t i) { return fmaxf(to_f(row[i]), 0.f); }

struct Rest {  // what the rest of a node is made of
  double gone;   // A
  int refused;   // without a draft: how many tokens are left out
};
template <typename T>
__device__ __forceinline__ double rest_of(const Shared &sh, float p, float q, int x, bool drawn, const Rest &r) {
  if (drawn) return fmax(__dsub_rn((double)p, __dmul_rn(r.gone, (double)q)), 0.0);
  for (int i = 0; i < r.refused; ++i)
    if (sh.refused[i] == x) return 0.0;
  return (double)p;
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 2) verify_kernel(const Args a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ Shared sh;
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int start = min(max(a.cu[b], 0), a.T), rows = max(min(max(a.cu[b + 1], 0), a.T) - start, 0);
  const int n = min(rows, MAX_NODES);
  const T *target = static_cast<const T *>(a.target), *draft = static_cast<const T *>(a.draft);
  const bool drawn = draft != nullptr;

  for (int j = tid; j < n; j += THREADS) {
    const int parent = a.parents[start + j];
    const int64_t x = a.tokens[start + j];
    const bool ok = j > 0 && parent >= 0 && parent < j && x >= 0 && x < a.V;
    sh.parent[j] = ok ? parent : -1;
    sh.token[j] = ok ? (int)x : -1;
    sh.u[j] = a.random[start + j];
    sh.p[j] = ok ? entry(target + (int64_t)(start + parent) * a.ts, x) : 0.f;
    sh.q[j] = ok && drawn ? entry(draft + (int64_t)(start + parent) * a.ds, x) : 1.f;
  }
  if (tid == 0) sh.way[0] = 0;
  cluster.sync();  // every block runs: its memory may be written to

  // this warp's piece of the vocabulary
  const int64_t pieces = (int64_t)blocks * WARPS, piece = (a.V + pieces - 1) / pieces;
  const int64_t lo = min(piece * (rank * WARPS + warp), (int64_t)a.V), hi = min(lo + piece, (int64_t)a.V);

  int cur = 0, kept = n > 0 ? 1 : 0, passes = 0;
  Rest r{0.0, 0};
  double mass = 1.0;

  // the sum of the rest over the whole row; the warps' sums stay in shared memory
  auto sum_rest = [&]() -> double {
    const T *prow = target + (int64_t)(start + cur) * a.ts;
    const T *qrow = drawn && r.gone != 0.0 ? draft + (int64_t)(start + cur) * a.ds : nullptr;
    double part[2] = {0.0, 0.0};
    for (int64_t i0 = lo + lane; i0 < hi; i0 += 32 * AT_ONCE) {
      float p[AT_ONCE], q[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int64_t at = i0 + 32 * i;
        p[i] = at < hi ? entry(prow, at) : 0.f;
        q[i] = qrow && at < hi ? entry(qrow, at) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) part[i & 1] += rest_of<T>(sh, p[i], q[i], (int)(i0 + 32 * i), drawn, r);
    }
    double s = part[0] + part[1];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sh.warp_sum[warp] = s;
    __syncthreads();
    const int buffer = passes++ & 1;
    if (tid < blocks) {
      double t = 0.0;
      for (int w = 0; w < WARPS; ++w) t += sh.warp_sum[w];
      *cluster.map_shared_rank(&sh.total[buffer][rank], tid) = t;
    }
    cluster.sync();
    double all = 0.0;
    for (int i = 0; i < blocks; ++i) all += sh.total[buffer][i];
    return all;
  };

  // a warp looks at 32 rows at a time
  for (int j0 = 0; j0 < n; j0 += 32) {
    int from = j0;
    while (true) {
      const int j = j0 + lane;
      const unsigned asked = __ballot_sync(0xffffffffu, j >= from && j > cur && j < n && sh.parent[j] == cur);
      if (!asked) break;
      const int x = j0 + __ffs(asked) - 1;  // the first child that has not been tested
      from = x + 1;
      const double left = rest_of<T>(sh, sh.p[x], sh.q[x], sh.token[x], drawn, r);
      const bool take = __dmul_rn(__dmul_rn((double)sh.u[x], mass), (double)sh.q[x]) < left;
      if (take) {
        cur = x;
        if (tid == 0) sh.way[kept] = x;
        ++kept;
        r = Rest{0.0, 0};
        mass = 1.0;
      } else if (drawn) {
        r.gone += mass;
        mass = sum_rest();
      } else {
        // (only numbers of 1 and more refuse what has more than the mass; below 0 a token that the row does not hold would pass)
        mass = fmax(mass - left, 0.0);
        __syncthreads();
        if (tid == 0) sh.refused[r.refused] = sh.token[x];
        ++r.refused;
        __syncthreads();
      }
    }
  }

  int64_t next = -1;
  bool mine = rank == 0;
  if (n > 0) {
    double all = drawn && r.gone != 0.0 ? mass : sum_rest();
    if (!(all > 0.0 && all < (double)INFINITY) && (r.gone != 0.0 || r.refused)) {
      r = Rest{0.0, 0};
      all = sum_rest();
    }
    if (all > 0.0 && all < (double)INFINITY) {
      const double goal = (double)sh.u[0] * all;
      const double *totals = sh.total[(passes - 1) & 1];
      // the first block, then its first warp, whose cumulative sum passes the goal; where rounding (or a number that is
      // not below 1) leaves none, the last one that has anything
      double before = 0.0, at = 0.0;
      int chosen = -1, last = 0;
      for (int i = 0; i < blocks; ++i) {
        if (!(totals[i] > 0.0)) continue;
        last = i;
        if (chosen < 0 && at + totals[i] > goal) {
          chosen = i;
          before = at;
        }
        at += totals[i];
      }
      bool tail = chosen < 0;  // the last token with anything left
      if (tail) chosen = last;
      mine = rank == chosen;
      if (mine) {
        int w_at = -1, w_last = 0;
        double w_before = before;
        at = before;
        for (int w = 0; w < WARPS; ++w) {
          if (!(sh.warp_sum[w] > 0.0)) continue;
          w_last = w;
          if (!tail && w_at < 0 && at + sh.warp_sum[w] > goal) {
            w_at = w;
            w_before = at;
          }
          at += sh.warp_sum[w];
        }
        if (w_at < 0) {
          tail = true;
          w_at = w_last;
        }
        if (warp == w_at) {
          const T *prow = target + (int64_t)(start + cur) * a.ts;
          const T *qrow = drawn && r.gone != 0.0 ? draft + (int64_t)(start + cur) * a.ds : nullptr;
          auto at_token = [&](int64_t i) {
            return rest_of<T>(sh, entry(prow, i), qrow ? entry(qrow, i) : 0.f, (int)i, drawn, r);
          };
          // a lane's sum of neighbouring tokens, then the tokens of the lane whose sums pass the goal, one each
          const int64_t each = (hi - lo + 31) / 32, mine_lo = min(lo + lane * each, hi), mine_hi = min(mine_lo + each, hi);
          double sum = 0.0;
          for (int64_t i0 = mine_lo; i0 < mine_hi; i0 += AT_ONCE) {
            float p[AT_ONCE], q[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
              p[i] = i0 + i < mine_hi ? entry(prow, i0 + i) : 0.f;
              q[i] = qrow && i0 + i < mine_hi ? entry(qrow, i0 + i) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) sum += rest_of<T>(sh, p[i], q[i], (int)(i0 + i), drawn, r);
          }
          auto up_to = [&](double v) {  // the sum of the lanes up to this one
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double up = __shfl_up_sync(0xffffffffu, v, o);
              if (lane >= o) v += up;
            }
            return v;
          };
          const double inc = up_to(sum);
          const unsigned some = __ballot_sync(0xffffffffu, sum > 0.0);
          const unsigned past = __ballot_sync(0xffffffffu, !tail && sum > 0.0 && w_before + inc > goal);
          tail = tail || !past;
          const int owner = past ? __ffs(past) - 1 : 31 - __clz(some);
          double so_far = w_before + __shfl_sync(0xffffffffu, inc - sum, owner);
          const int64_t from = min(lo + owner * each, hi), to = min(from + each, hi);
          int64_t positive = from;
          for (int64_t i0 = from; i0 < to && next < 0; i0 += 32) {
            const int64_t i = i0 + lane;
            const double v = i < to ? at_token(i) : 0.0, upto = up_to(v);
            const unsigned any = __ballot_sync(0xffffffffu, v > 0.0);
            const unsigned beyond = __ballot_sync(0xffffffffu, !tail && v > 0.0 && so_far + upto > goal);
            if (any) positive = i0 + 31 - __clz(any);
            if (beyond) next = i0 + __ffs(beyond) - 1;
            so_far += __shfl_sync(0xffffffffu, upto, 31);
          }
          if (next < 0) next = positive;
          if (lane == 0) a.next[b] = next;
        }
      }
    } else if (rank == 0 && tid == 0) {
      a.next[b] = -1;
    }
  } else if (rank == 0 && tid == 0) {
    a.next[b] = -1;
  }

  __syncthreads();  // `way` is complete
  if (rank == 0) {
    if (tid == 0) a.kept[b] = kept;
    for (int j = tid; j < rows; j += THREADS) a.path[start + j] = j < kept ? sh.way[j] : -1;
    if (b == 0)
      for (int64_t t = tid; t < a.T; t += THREADS)
        if (t < a.cu[0] || t >= a.cu[a.batch]) a.path[t] = -1;
  }
  cluster.sync();  // no block leaves while another may still write to its memory
}

}  // namespace verify
}  // namespace mhc

using namespace mhc;

extern "C" int mhc_verify_drafts(const int64_t *tokens, const int32_t *parents, const int32_t *cu_tokens, int batch, int64_t T,
                                 const void *target, int64_t target_stride, const void *draft, int64_t draft_stride, int dtype,
                                 int64_t V, const float *random, int32_t *path, int32_t *kept, int64_t *next, void *stream) {
  const char *who = "mhc_verify_drafts";
  clear_error();
  if (dtype != MHC_F32 && dtype != MHC_BF16 && dtype != MHC_F16) return fail(MHC_ERR_DTYPE, "%s: bad dtype code %d", who, dtype);
  if (batch < 0 || batch > 0x7fffffff / verify::MAX_CLUSTER || T < 0 || T > 0x7fffffff || V < 1 || V > 0x7fffffff - 4096)
    return fail(MHC_ERR_SHAPE, "%s: %d sequences, %lld rows, %lld tokens", who, batch, (long long)T, (long long)V);
  if (T > 1 && (target_stride < V || (draft && draft_stride < V)))
    return fail(MHC_ERR_SHAPE, "%s: rows %lld and %lld apart hold %lld tokens", who, (long long)target_stride, (long long)draft_stride, (long long)V);
  if ((batch > 0 && (!cu_tokens || !kept || !next)) || (T > 0 && (!tokens || !parents || !target || !random || !path)))
    return fail(MHC_ERR_NULL, "%s: required pointer is NULL", who);
  const size_t es = dtype == MHC_F32 ? 4 : 2;
  if ((uintptr_t)tokens % 8 || (uintptr_t)parents % 4 || (uintptr_t)cu_tokens % 4 || (uintptr_t)target % es || (uintptr_t)draft % es ||
      (uintptr_t)random % 4 || (uintptr_t)path % 4 || (uintptr_t)kept % 4 || (uintptr_t)next % 8)
    return fail(MHC_ERR_ALIGN, "%s: a pointer is not aligned to its elements", who);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (batch == 0) return T == 0 ? MHC_OK : cuda_status(cudaMemsetAsync(path, 0xff, (size_t)T * 4, st), who);
  verify::Args a{tokens, parents, cu_tokens, batch, (int)T, target, draft, target_stride, draft_stride, (int)V, random, path, kept, next};
  int blocks = 1;
  while (blocks < verify::MAX_CLUSTER && V > (int64_t)blocks * 4096) blocks *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)batch * blocks);
  cfg.blockDim = dim3(verify::THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(with_dtype(dtype, [&](auto tag) -> cudaError_t {
                       using T_ = decltype(tag);
                       return cudaLaunchKernelEx(&cfg, verify::verify_kernel<T_>, a);
                     }),
                     who);
}
