// The global gradient norm over many tensors, and clipping by it:
//   norm = sqrt(sum over all tensors of x^2),   x *= c,  c = min(1, max_norm / (norm + 1e-6))
// (torch.nn.utils.clip_grad_norm_'s formula; a NaN norm makes c NaN, as there).
// Memory-bound: one read for the norm, one read and one write for the scaling. The tensors'
// addresses travel in the kernel arguments, 160 to a launch, so nothing is staged in device memory and
// a captured call replays what it was given. A workgroup takes one chunk of one tensor; squares
// are summed in f64 (a sum of 3e8 small squares loses the small ones in f32), the chunks' sums in a fixed
// order, so the norm has the same bits from call to call. Measured: 480 f32 tensors of up to 4 M elements (2.0 GB)
// norm 407 us = 4.9 TB/s, scaling 775 us = 5.2 TB/s of reads and writes, a large copy's rate (4.9); 150 bf16 tensors at
// odd offsets (113 MB) 21 + 4 + 37 us; 21 small ones 4.3 + 4.7 us, the launches.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "common.h"
#include "overlap.h"

namespace {

constexpr int PER_LAUNCH = 160;
constexpr int CHUNK_MIN = 4096, CHUNK_MAX = 65536;
constexpr int FEW = 1024;       // up to so many chunk sums, every scaling workgroup adds them itself
constexpr double EPS = 1e-6;

struct Table {
  void* ptr[PER_LAUNCH];
  long long n[PER_LAUNCH];
  int first[PER_LAUNCH + 1];    // first chunk of each tensor in this launch
  int count, chunk, part0, bf16[(PER_LAUNCH + 31) / 32];
};

struct Piece { char* p; long long lo, hi; bool b16; };   // elements [lo, hi) of the tensor at p

NRSE_DEV Piece piece_of(const Table& t, int blk) {
  int lo = 0, hi = t.count;     // first[lo] <= blk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= blk) lo = mid;
    else hi = mid;
  }
  const long long a = (long long)(blk - t.first[lo]) * t.chunk;
  return Piece{(char*)t.ptr[lo], a, min(a + t.chunk, t.n[lo]), (bool)((t.bf16[lo >> 5] >> (lo & 31)) & 1)};
}

NRSE_DEV double sq(float x) { return (double)x * (double)x; }

// sum over the block, the same order every time
NRSE_DEV double block_sum(double a) {
  __shared__ double red[4];
  a = wave_sum_d(a);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// f(first element, 16 bytes) over a piece's aligned middle, s(element) over its ragged ends (a tensor
// may start anywhere its type may)
template <typename T, typename V, typename S>
NRSE_DEV void over(const Piece& pc, V vec, S one) {
  constexpr int W = 16 / (int)sizeof(T);
  T* const p = (T*)pc.p;
  const long long mis = (long long)(((uintptr_t)(p + pc.lo) & 15) / sizeof(T));
  const long long a = min(pc.hi, pc.lo + (mis ? W - mis : 0));
  const long long nv = (pc.hi - a) / W;
  for (long long i = pc.lo + threadIdx.x; i < a; i += 256) one(p + i);
  uint4* const q = reinterpret_cast<uint4*>(p + a);
  long long i = threadIdx.x;
  for (; i + 768 < nv; i += 1024) {   // four loads in flight
    uint4 u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = ldg(q + i + 256 * j);
#pragma unroll
    for (int j = 0; j < 4; ++j) vec(q + i + 256 * j, u[j]);
  }
  for (; i < nv; i += 256) vec(q + i, ldg(q + i));
  for (long long k = a + nv * W + threadIdx.x; k < pc.hi; k += 256) one(p + k);
}

__global__ __launch_bounds__(256) void norm_kernel(const Table t, double* __restrict__ part) {
  const Piece pc = piece_of(t, blockIdx.x);
  double s = 0.0;
  if (pc.b16) {
    over<bf16_t>(
        pc,
        [&](const uint4*, uint4 u) {
          const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) s += sq(__uint_as_float(w[e] << 16)) + sq(__uint_as_float(w[e] & 0xffff0000u));
        },
        [&](const bf16_t* x) { s += sq(bf2f(*x)); });
  } else {
    over<float>(
        pc,
        [&](const uint4*, uint4 u) {
          s += sq(__uint_as_float(u.x)) + sq(__uint_as_float(u.y)) + sq(__uint_as_float(u.z)) + sq(__uint_as_float(u.w));
        },
        [&](const float* x) { s += sq(*x); });
  }
  s = block_sum(s);
  if (threadIdx.x == 0) part[t.part0 + blockIdx.x] = s;
}

NRSE_DEV double parts_sum(const double* __restrict__ part, int n) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) s += part[i];
  return block_sum(s);
}

// (a sum of up to 30000 chunks by one workgroup: 1024 threads, four loads each in flight)
__global__ __launch_bounds__(1024) void finish_kernel(const double* __restrict__ part, int n, float* __restrict__ norm,
                                                      double* __restrict__ exact) {
  __shared__ double red[16];
  double a = 0.0;
  for (int i = threadIdx.x; i < n; i += 4096) {
    double v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = part[min(i + 1024 * k, n - 1)];
#pragma unroll
    for (int k = 0; k < 4; ++k) a += i + 1024 * k < n ? v[k] : 0.0;
  }
  a = wave_sum_d(a);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int k = 0; k < 16; ++k) s += red[k];
    s = sqrt(s);
    *norm = (float)s;
    if (exact) *exact = s;
  }
}

// few: `part` holds that many chunk sums, to be added here (and by the first workgroup written as the
// norm); 0: it holds the norm
__global__ __launch_bounds__(256) void scale_kernel(const Table t, const double* __restrict__ part, int few,
                                                    float* __restrict__ norm, double max_norm) {
  const double v = few ? sqrt(parts_sum(part, few)) : *part;
  if (few && norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
  const double c64 = max_norm / (v + EPS);
  if (c64 >= 1.0) return;   // nothing to clip: nothing is written
  const float c = (float)c64;
  const Piece pc = piece_of(t, blockIdx.x);
  if (pc.b16) {
    over<bf16_t>(
        pc,
        [&](uint4* q, uint4 u) {
          unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = (unsigned)f2bf(__uint_as_float(w[e] << 16) * c) |
                   ((unsigned)f2bf(__uint_as_float(w[e] & 0xffff0000u) * c) << 16);
          *q = make_uint4(w[0], w[1], w[2], w[3]);
        },
        [&](bf16_t* x) { *x = f2bf(bf2f(*x) * c); });
  } else {
    over<float>(
        pc,
        [&](uint4* q, uint4 u) {
          *q = make_uint4(__float_as_uint(__uint_as_float(u.x) * c), __float_as_uint(__uint_as_float(u.y) * c),
                          __float_as_uint(__uint_as_float(u.z) * c), __float_as_uint(__uint_as_float(u.w) * c));
        },
        [&](float* x) { *x *= c; });
  }
}

struct Plan { long long total, chunks; int chunk; };

int es_of(int dtype) { return dtype == NRSE_BF16 ? 2 : 4; }

// chunks of about total / 2048 elements: enough workgroups for the chip, no more sums than are useful
int make_plan(const char* fn, const void* const* ptrs, const long long* numel, const int* dtypes, int count, Plan& pl) {
  NRSE_REQUIRE(count >= 0 && (count == 0 || (ptrs && numel && dtypes)), "%s: bad list", fn);
  pl = Plan{0, 0, CHUNK_MIN};
  for (int i = 0; i < count; ++i) {
    NRSE_REQUIRE(numel[i] >= 0 && (numel[i] == 0 || ptrs[i]), "%s: tensor %d: null or negative size", fn, i);
    NRSE_REQUIRE(dtypes[i] == NRSE_BF16 || dtypes[i] == NRSE_F32, "%s: tensor %d: dtype %d (bf16 and f32 only)", fn, i,
                 dtypes[i]);
    NRSE_REQUIRE(((uintptr_t)ptrs[i] & (es_of(dtypes[i]) - 1)) == 0, "%s: tensor %d: address not a multiple of its type",
                 fn, i);
    pl.total += numel[i];
  }
  const long long want = (pl.total / 2048 + 4095) / 4096 * 4096;
  pl.chunk = (int)(want < CHUNK_MIN ? CHUNK_MIN : want > CHUNK_MAX ? CHUNK_MAX : want);
  for (int i = 0; i < count; ++i) pl.chunks += (numel[i] + pl.chunk - 1) / pl.chunk;
  NRSE_REQUIRE(pl.chunks < (1LL << 30), "%s: %lld chunks", fn, pl.chunks);
  return NRSE_OK;
}

// norm and part are written while tensors are read: in none of them, and apart
int check_scratch(const char* fn, const void* const* ptrs, const long long* numel, const int* dtypes, int count, const Plan& pl,
                  const float* norm, const double* part) {
  using nrse_overlap::flat;
  NRSE_REQUIRE(norm && part, "%s: norm or part is null", fn);
  const auto n = flat("norm", norm, sizeof(float)), w = flat("part", part, (pl.chunks + 1) * (long long)sizeof(double));
  NRSE_REQUIRE(!meet(n, w), "%s: norm and part overlap", fn);
  for (int i = 0; i < count; ++i) {
    const auto t = flat("", ptrs[i], numel[i] * es_of(dtypes[i]));
    NRSE_REQUIRE(!meet(t, n) && !meet(t, w), "%s: tensor %d and norm or part overlap", fn, i);
  }
  return NRSE_OK;
}

template <typename F>
void launches(const void* const* ptrs, const long long* numel, const int* dtypes, int count, const Plan& pl, bool backwards,
              F launch) {
  // tables in order of the list, or from its end: what the norm read last may still be in the last-level
  // cache when the scaling begins
  int part0 = backwards ? (int)pl.chunks : 0;
  for (int at = 0; at < count;) {
    Table t;
    t.count = 0;
    t.chunk = pl.chunk;
    int blocks = 0;
    for (int& b : t.bf16) b = 0;
    while (at < count && t.count < PER_LAUNCH) {
      const int i = backwards ? count - 1 - at : at;
      ++at;
      if (numel[i] == 0) continue;
      const int k = t.count++;
      t.ptr[k] = const_cast<void*>(ptrs[i]);
      t.n[k] = numel[i];
      t.first[k] = blocks;
      if (dtypes[i] == NRSE_BF16) t.bf16[k >> 5] |= (int)(1u << (k & 31));
      blocks += (int)((numel[i] + pl.chunk - 1) / pl.chunk);
    }
    t.first[t.count] = blocks;
    if (!blocks) continue;
    t.part0 = part0;
    part0 += blocks;
    launch(t, blocks);
  }
}

int run_norm(const char* fn, const void* const* ptrs, const long long* numel, const int* dtypes, int count, const Plan& pl,
             double* part, hipStream_t st) {
  launches(ptrs, numel, dtypes, count, pl, false, [&](const Table& t, int blocks) {
    hipLaunchKernelGGL(norm_kernel, dim3(blocks), dim3(256), 0, st, t, part);
  });
  return nrse_check_launch(fn);
}

}  // namespace

extern "C" long long nrse_grad_norm_workspace(const void* const* ptrs, const long long* numel, const int* dtypes, int count) {
  Plan pl;
  if (const int rc = make_plan("nrse_grad_norm_workspace", ptrs, numel, dtypes, count, pl)) return rc;
  return pl.chunks + 1;
}

extern "C" int nrse_grad_norm(const void* const* ptrs, const long long* numel, const int* dtypes, int count, float* norm,
                              double* part, void* stream) {
  const char* fn = "nrse_grad_norm";
  Plan pl;
  if (const int rc = make_plan(fn, ptrs, numel, dtypes, count, pl)) return rc;
  if (const int rc = check_scratch(fn, ptrs, numel, dtypes, count, pl, norm, part)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (const int rc = run_norm(fn, ptrs, numel, dtypes, count, pl, part, st)) return rc;
  hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(1024), 0, st, part, (int)pl.chunks, norm, nullptr);
  return nrse_check_launch(fn);
}

extern "C" int nrse_clip_grad_norm(const void* const* ptrs, const long long* numel, const int* dtypes, int count,
                                   double max_norm, float* norm, double* part, void* stream) {
  const char* fn = "nrse_clip_grad_norm";
  Plan pl;
  if (const int rc = make_plan(fn, ptrs, numel, dtypes, count, pl)) return rc;
  NRSE_REQUIRE(norm && part, "%s: norm or part is null", fn);
  NRSE_REQUIRE(max_norm >= 0.0, "%s: max_norm %g", fn, max_norm);
  if (const int rc = check_scratch(fn, ptrs, numel, dtypes, count, pl, norm, part)) return rc;
  // two tensors that share an element would scale it twice, in any order
  try {
    std::vector<std::pair<uintptr_t, uintptr_t>> span;
    span.reserve(count);
    for (int i = 0; i < count; ++i)
      if (numel[i]) span.emplace_back((uintptr_t)ptrs[i], (uintptr_t)ptrs[i] + numel[i] * es_of(dtypes[i]));
    std::sort(span.begin(), span.end());
    for (size_t i = 1; i < span.size(); ++i)
      NRSE_REQUIRE(span[i - 1].second <= span[i].first, "%s: two of the tensors overlap", fn);
  } catch (const std::bad_alloc&) {
    nrse_set_error("%s: out of host memory", fn);
    return NRSE_ERR_ARG;
  }
  const hipStream_t st = (hipStream_t)stream;
  if (const int rc = run_norm(fn, ptrs, numel, dtypes, count, pl, part, st)) return rc;
  const int few = pl.chunks > 0 && pl.chunks <= FEW ? (int)pl.chunks : 0;
  double* const exact = part + pl.chunks;
  if (!few) hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(1024), 0, st, part, (int)pl.chunks, norm, exact);
  bool first = true;
  launches(ptrs, numel, dtypes, count, pl, true, [&](const Table& t, int blocks) {
    hipLaunchKernelGGL(scale_kernel, dim3(blocks), dim3(256), 0, st, t, few ? part : exact, few, first ? norm : nullptr,
                       max_norm);
    first = false;
  });
  return nrse_check_launch(fn);
}
