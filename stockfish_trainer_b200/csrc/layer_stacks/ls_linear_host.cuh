// Host side of the linear layer: how a product is cut into tiles and pieces,
// what its operands need, and the launches.
#pragma once

#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "ls_gemm.cuh"
#include "ls_host.cuh"
#include "ls_linear.cuh"

namespace nnue_ls {
namespace {

// ---- tensor maps -------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static std::atomic<void*> fn{nullptr};
  void* f = fn.load(std::memory_order_acquire);
  if (!f) {
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) !=
            cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      return nullptr;
    fn.store(f, std::memory_order_release);
  }
  return reinterpret_cast<EncodeTiled>(f);
}

// An operand in the products' layout: [planes][outer][inner] 16-bit values,
// inner contiguous.  base and ld * 2 are multiples of 16 bytes.
struct Operand {
  const void* base;
  int64_t inner, outer, ld;
  bool mn_major;  // inner runs along m or n rather than k
};

int make_map(CUtensorMap* map, const Operand& o, int planes, bool is_f16, int bk, int tile_rows) {
  EncodeTiled fn = encode_tiled();
  if (!fn) return fail(NNUE_LS_ERR_CUDA, "gemm: the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[3] = {(cuuint64_t)o.inner, (cuuint64_t)o.outer, (cuuint64_t)planes};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)o.ld * 2 * (cuuint64_t)o.outer};
  const cuuint32_t box[3] = {(cuuint32_t)(o.mn_major ? 64 : bk), (cuuint32_t)(o.mn_major ? bk : tile_rows), 1};
  const cuuint32_t one[3] = {1, 1, 1};
  auto encode = [&] {
    return fn(map, is_f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
              const_cast<void*>(o.base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              o.mn_major || bk == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  int dev = 0;
  if (r == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess)
    r = encode();  // the first call on this thread: it had no context yet
  return r == CUDA_SUCCESS ? NNUE_LS_OK : fail(NNUE_LS_ERR_CUDA, "gemm: the driver refused a tensor map (%d)", (int)r);
}

// ---- tiles ---------------------------------------------------------------------
struct TilePlan {
  int cg, bn, splits, k_blocks;
  int64_t m_tiles, n_tiles;
  size_t partial_bytes(int64_t M, int64_t N) const { return splits > 1 ? align256((size_t)splits * M * N * 4) : 0; }
};

// Estimates the clocks of each way to cut C = A B^T and takes the least.  The
// figures are fits to measured times of single products on B200: a k block
// (64 values, fp32 32) costs a part for A's tile and its copies and a part per
// column, an item its epilogue and drain, a pair of blocks its later start,
// pieces their joining pass (a launch, and their bytes at 3500 per clock).
// Fitted to results of 128 and more columns; narrower ones were not measured.
// Against the fits' own predecessor, which counted products and L2 bytes only:
// fp32 65536 x 1040 x 256 forward 201 instead of 253 us, 24 x 1040 x 1040 bf16
// 11.4 instead of 14.5 us.
TilePlan find_tiles(int64_t M, int64_t N, int64_t K, int planes) {
  const int64_t k_blocks = ceil_div(K, planes == 1 ? 64 : 32);
  TilePlan best{};
  double best_cost = 0;
  for (int cg = 1; cg <= 2; ++cg) {
    const int max_bn = planes == 3 && cg == 1 ? 128 : 256;
    const double block0 = planes == 1 ? (cg == 1 ? 330 : 370) : (cg == 1 ? 970 : 1600);
    const double block1 = planes == 1 ? (cg == 1 ? 1.92 : 1.3) : (cg == 1 ? 3.7 : 2.0);
    const int64_t m_tiles = ceil_div(M, kTileM * cg), least = ceil_div(N, max_bn);
    const int workers = kNumSMs / cg;
    int last_bn = 0;
    for (int i = 0; i < 8; ++i) {
      // the fewest column tiles and a few more; as many as occupy the SMs, and half of that
      const int64_t nt = i < 6 ? least + i : std::max(least, workers / m_tiles / (i - 5));
      const int bn = (int)(ceil_div(ceil_div(N, nt), 16) * 16);
      if (bn == last_bn) continue;
      last_bn = bn;
      const int64_t n_tiles = ceil_div(N, bn), tiles = m_tiles * n_tiles;
      const double block = block0 + block1 * std::max(bn, 48);
      const double item = planes == 1 ? 1000 + 14.0 * bn : 2000 + 10.0 * bn;
      for (int fill = 0; fill <= 4; ++fill) {  // pieces that fill this many rounds of the SMs
        int64_t splits = fill == 0 ? 1 : workers * fill / tiles;
        splits = std::min<int64_t>(std::min<int64_t>(splits, k_blocks), 256);
        if (splits < 1 || (fill && splits < 2)) continue;
        const double rounds = (double)ceil_div(tiles * splits, workers), per = (double)ceil_div(k_blocks, splits);
        double cost = (cg == 2 ? 3600 : 0) + rounds * (per * block + item) + 5.0 * std::min<int64_t>(tiles, workers);
        if (splits > 1) cost += 8000 + splits * (double)M * N * 8 / 3500;
        if (best.cg == 0 || cost < best_cost) {
          best_cost = cost;
          best = TilePlan{cg, bn, (int)splits, (int)k_blocks, m_tiles, n_tiles};
        }
      }
    }
  }
  return best;
}

// The plan of a shape, kept for the next call with it: the search takes a few
// microseconds, and a call asks for its workspace's size first.
TilePlan plan_tiles(int64_t M, int64_t N, int64_t K, int planes) {
  struct Entry {
    int64_t M = 0, N = 0, K = 0;
    TilePlan plan{};
  };
  static thread_local Entry kept[32];
  Entry& e = kept[(uint64_t)(M * 31 + N * 7 + K) % 32];
  if (e.M != M || e.N != N || e.K != K) e = Entry{M, N, K, find_tiles(M, N, K, planes)};
  return e.plan;
}

template <typename T, int CG>
int launch_gemm_cg(const CUtensorMap& a, const CUtensorMap& b, const GemmParams& p, cudaStream_t s) {
  using S = GemmShape<sizeof(T) == 4 ? 3 : 1, CG>;
  if (int rc = allow_shared<gemm_kernel<T, CG>>("gemm", S::kSmem)) return rc;
  const int64_t items = (int64_t)p.m_tiles * p.n_tiles * p.splits;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(items, kNumSMs / CG) * CG));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = CG;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  cfg.numAttrs = CG == 1 ? 0 : 1;
  count_launch();
  const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_kernel<T, CG>, a, b, p);
  return e == cudaSuccess ? NNUE_LS_OK : fail(NNUE_LS_ERR_CUDA, "gemm: %s", cudaGetErrorString(e));
}

// C[M, N] = A B^T over K with the epilogue e; partial as sized by the plan.
template <typename T>
int launch_gemm(const Operand& a, const Operand& b, int64_t M, int64_t N, const TilePlan& t, EpilogueParams e,
                void* partial, cudaStream_t s) {
  constexpr int planes = sizeof(T) == 4 ? 3 : 1;
  constexpr int bk = planes == 1 ? 64 : 32;
  constexpr bool is_f16 = std::is_same<T, f16>::value;
  GemmParams p;
  CUtensorMap map_a, map_b;
  if (int rc = make_map(&map_a, a, planes, is_f16, bk, kTileM)) return rc;
  if (int rc = make_map(&map_b, b, planes, is_f16, bk, t.bn / t.cg)) return rc;
  p.M = M;
  p.N = N;
  p.k_blocks = t.k_blocks;
  p.splits = t.splits;
  p.m_tiles = (int32_t)t.m_tiles;
  p.n_tiles = (int32_t)t.n_tiles;
  p.bn = t.bn;
  p.a_mn = a.mn_major;
  p.b_mn = b.mn_major;
  // kind::f16 instruction descriptor: fp32 sums; type of A and B; their majors; N / 8; M / 16
  const uint32_t type = is_f16 ? 0 : 1;
  p.idesc = 1u << 4 | type << 7 | type << 10 | (uint32_t)a.mn_major << 15 | (uint32_t)b.mn_major << 16 |
            (uint32_t)(t.bn / 8) << 17 | (uint32_t)(kTileM * t.cg / 16) << 24;
  p.partial = static_cast<float*>(partial);
  p.wait_limit_ns = wait_limit_ns();
  p.items = p.wait_limit_ns ? t.m_tiles * t.n_tiles * t.splits : 0;
  constexpr int64_t V = 16 / sizeof(T);
  auto aligned = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  e.vec = N % V == 0 && aligned(e.out) && aligned(e.act_grad) && aligned(e.residual) && (!e.residual || e.ldr % V == 0);
  p.e = e;
  if (int rc = t.cg == 1 ? launch_gemm_cg<T, 1>(map_a, map_b, p, s) : launch_gemm_cg<T, 2>(map_a, map_b, p, s)) return rc;
  if (t.splits > 1) {
    const int64_t total = e.vec ? M * N / 4 : M * N;
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(total, 256), kNumSMs * 16);
    count_launch();
    if (e.vec) join_kernel<T, true><<<grid, 256, 0, s>>>(p.partial, t.splits, M, N, e);
    else join_kernel<T, false><<<grid, 256, 0, s>>>(p.partial, t.splits, M, N, e);
  }
  return check_launch("gemm");
}

// ---- operands ----------------------------------------------------------------
// fp32 values are always brought into planes; 16-bit ones only when a row
// starts off a 16-byte boundary, where TMA cannot copy it.
template <typename T>
bool needs_pack(const void* p, int64_t ld, int64_t rows) {
  return sizeof(T) == 4 || reinterpret_cast<uintptr_t>(p) % 16 != 0 || (ld % 8 != 0 && rows > 1);
}
constexpr int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }
template <typename T>
size_t pack_bytes(int64_t rows, int64_t cols) {
  return align256((size_t)rows * round8(cols) * (sizeof(T) == 4 ? 6 : 2));
}

// Matrices that still have to be packed before a product, in one launch.
template <typename T>
struct Packer {
  PackJobs jobs{};
  int count = 0;

  // The matrix as an operand; packed into `buffer` where it cannot be read as it lies.
  Operand operand(const void* p, int64_t ld, int64_t rows, int64_t cols, bool mn_major, void* buffer) {
    if (!needs_pack<T>(p, ld, rows)) return Operand{p, cols, rows, round8(ld), mn_major};
    const bool vec = reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % (16 / (int64_t)sizeof(T)) == 0;
    jobs.job[count++] = PackJob{p, buffer, ld, rows, cols, round8(cols), vec};
    return Operand{buffer, cols, rows, round8(cols), mn_major};
  }
  void launch(cudaStream_t s) {
    if (count == 0) return;
    int64_t total = 0;
    for (int i = 0; i < 2; ++i) {
      if (i < count) total += jobs.job[i].rows * (jobs.job[i].ldo / 8);
      jobs.end[i] = total;
    }
    count_launch();
    pack_kernel<T><<<(unsigned)std::min<int64_t>(ceil_div(total, 256), kNumSMs * 16), 256, 0, s>>>(jobs);
  }
};

// ---- forward -------------------------------------------------------------------
// Up to 4 rows (fp32: 8, where the other way packs its operands first) go to the
// kernel without tiles.  1040 x 1040 bf16: 2.7 us for one row, 6.9 for 4, 10.9
// for 8; on tiles 10.1 for any of them.  1040 x 256 fp32: 2.7 us for one row,
// 6.3 for 8, 16.4 for 16; on tiles 14.6 in three launches.
template <typename T>
bool few_rows(const nnue_ls_linear& a) {
  return a.rows <= (sizeof(T) == 4 ? 8 : 4);
}

template <typename T, int MT>
void launch_few_rows(const nnue_ls_linear& a, const EpilogueParams& e, cudaStream_t s) {
  constexpr int64_t V = 16 / sizeof(T);
  auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool vec = a.inputs % V == 0 && (a.ldx % V == 0 || a.rows == 1) && (a.ldw % V == 0 || a.outputs == 1) &&
                   aligned(a.x) && aligned(a.weight);
  const T *x = static_cast<const T*>(a.x), *w = static_cast<const T*>(a.weight);
  const unsigned grid = (unsigned)ceil_div(a.outputs, 8);
  count_launch();
  if (vec) few_rows_kernel<T, MT, true><<<grid, 256, 0, s>>>(x, a.ldx, w, a.ldw, (int)a.rows, a.outputs, a.inputs, e);
  else few_rows_kernel<T, MT, false><<<grid, 256, 0, s>>>(x, a.ldx, w, a.ldw, (int)a.rows, a.outputs, a.inputs, e);
}

struct ForwardPlan {
  TilePlan tiles;
  size_t x, w, partial, total;
};

template <typename T>
ForwardPlan plan_forward(const nnue_ls_linear& a) {
  ForwardPlan p{};
  if (few_rows<T>(a)) return p;
  p.tiles = plan_tiles(a.rows, a.outputs, a.inputs, sizeof(T) == 4 ? 3 : 1);
  p.x = !a.x_packed && needs_pack<T>(a.x, a.ldx, a.rows) ? pack_bytes<T>(a.rows, a.inputs) : 0;
  p.w = !a.weight_packed && needs_pack<T>(a.weight, a.ldw, a.outputs) ? pack_bytes<T>(a.outputs, a.inputs) : 0;
  p.partial = p.tiles.partial_bytes(a.rows, a.outputs);
  p.total = p.x + p.w + p.partial;
  return p;
}

}  // namespace

template <typename T>
size_t linear_packed_bytes(const nnue_ls_linear& a, bool weight) {
  if (few_rows<T>(a)) return 0;
  if (weight) return needs_pack<T>(a.weight, a.ldw, a.outputs) ? pack_bytes<T>(a.outputs, a.inputs) : 0;
  return needs_pack<T>(a.x, a.ldx, a.rows) ? pack_bytes<T>(a.rows, a.inputs) : 0;
}

template <typename T>
size_t linear_forward_bytes(const nnue_ls_linear& a) {
  return plan_forward<T>(a).total;
}

template <typename T>
int linear_forward(const nnue_ls_linear& a, char* ws, cudaStream_t s) {
  EpilogueParams e{a.bias, a.residual, a.out, a.act_grad, a.ldr, a.activation, a.bias_dtype == NNUE_LS_F32, false};
  if (few_rows<T>(a)) {
    if (a.rows == 1) launch_few_rows<T, 1>(a, e, s);
    else if (a.rows <= 4) launch_few_rows<T, 4>(a, e, s);
    else if constexpr (sizeof(T) == 4) launch_few_rows<T, 8>(a, e, s);
    return check_launch("linear_forward");
  }
  const ForwardPlan p = plan_forward<T>(a);
  Packer<T> pack;
  const Operand x = pack.operand(a.x, a.ldx, a.rows, a.inputs, false, a.x_packed ? a.x_packed : ws);
  const Operand w =
      pack.operand(a.weight, a.ldw, a.outputs, a.inputs, false, a.weight_packed ? a.weight_packed : ws + p.x);
  pack.launch(s);
  return launch_gemm<T>(x, w, a.rows, a.outputs, p.tiles, e, ws + p.x + p.w, s);
}

// ---- backward --------------------------------------------------------------------
namespace {

struct BackwardPlan {
  TilePlan dx, dw;
  int64_t parts, rows_per_part;  // the bias sum's row ranges
  bool dz_written;
  int tx, v;                     // dz pass: threads along a row, columns per thread
  size_t dz, x, w, bias, partial, total;
};

template <typename T>
BackwardPlan plan_backward(const nnue_ls_linear& a) {
  BackwardPlan p{};
  const int planes = sizeof(T) == 4 ? 3 : 1;
  const bool products = a.rows > 0 && (a.grad_x || a.grad_weight);  // without rows there is nothing to cut into tiles
  if (products && a.grad_x) {
    p.dx = plan_tiles(a.rows, a.inputs, a.outputs, planes);
    p.w = !a.weight_packed && needs_pack<T>(a.weight, a.ldw, a.outputs) ? pack_bytes<T>(a.outputs, a.inputs) : 0;
    p.partial = p.dx.partial_bytes(a.rows, a.inputs);
  }
  if (products && a.grad_weight) {
    p.dw = plan_tiles(a.outputs, a.inputs, a.rows, planes);
    p.x = !a.x_packed && needs_pack<T>(a.x, a.ldx, a.rows) ? pack_bytes<T>(a.rows, a.inputs) : 0;
    p.partial = std::max(p.partial, p.dw.partial_bytes(a.outputs, a.inputs));
  }
  p.dz_written = products && (a.activation != NNUE_LS_ACT_NONE || needs_pack<T>(a.grad_out, a.ldg, a.rows));
  p.dz = p.dz_written ? pack_bytes<T>(a.rows, a.outputs) : 0;
  constexpr int64_t V = 16 / sizeof(T);
  auto aligned = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  p.v = a.outputs % V == 0 && a.ldg % V == 0 && aligned(a.grad_out) && aligned(a.act_grad) ? (int)V : 1;
  const int64_t groups = ceil_div(a.outputs, p.v);
  // no more than 32 groups across, spread evenly: 130 groups are five times 26, not four times 32 and one of 2
  const int64_t wide = ceil_div(groups, 32);
  p.tx = (int)ceil_div(groups, wide);
  const int64_t high = 256 / p.tx;
  // up to 8 rows per thread one block takes them all, which saves the launch that adds the parts (64 x 100 fp32:
  // 4.7 us, against 4.3 and 1.7; a whole training call 126 us of the host's time, against 140.  With 16 rows per
  // thread, 300 x 104 bf16: 9.9 us, against 5.3 and 1.3)
  p.parts = a.rows <= high * 8 ? 1 : std::min(ceil_div(a.rows, high * 4), ceil_div(kNumSMs * 8, wide));
  p.rows_per_part = std::max<int64_t>(1, ceil_div(a.rows, p.parts));
  p.bias = a.grad_bias && p.parts > 1 ? align256((size_t)p.parts * a.outputs * 4) : 0;
  p.total = p.dz + p.x + p.w + p.bias + p.partial;
  return p;
}

}  // namespace

template <typename T>
size_t linear_backward_bytes(const nnue_ls_linear& a) {
  return plan_backward<T>(a).total;
}

template <typename T>
int linear_backward(const nnue_ls_linear& a, char* ws, cudaStream_t s) {
  const BackwardPlan p = plan_backward<T>(a);
  using Code = typename Derivative<T>::Code;
  char *dz = ws, *x = dz + p.dz, *w = x + p.x, *bias = w + p.w, *partial = bias + p.bias;
  Operand d{a.grad_out, a.outputs, a.rows, round8(a.ldg), false};
  if (p.dz_written || a.grad_bias) {
    const T* g = static_cast<const T*>(a.grad_out);
    const Code* ag = a.activation == NNUE_LS_ACT_NONE ? nullptr : static_cast<const Code*>(a.act_grad);
    const int64_t ldo = round8(a.outputs);
    void* out = p.dz_written ? dz : nullptr;
    float* sums = p.bias ? reinterpret_cast<float*>(bias) : nullptr;
    const dim3 grid((unsigned)ceil_div(ceil_div(a.outputs, p.v), p.tx), (unsigned)p.parts);
    count_launch();
    const bool bias_f32 = a.bias_dtype == NNUE_LS_F32;
    const auto kernel = p.v > 1 ? dz_kernel<T, 16 / sizeof(T)> : dz_kernel<T, 1>;
    kernel<<<grid, 256, 0, s>>>(g, a.ldg, ag, out, ldo, sums, sums ? nullptr : a.grad_bias, bias_f32, a.rows, a.outputs,
                                p.rows_per_part, p.tx);
    if (p.dz_written) d = Operand{dz, a.outputs, a.rows, ldo, false};
    if (sums) {
      count_launch();
      column_total_kernel<T><<<(unsigned)ceil_div(a.outputs, 32), dim3(32, 8), 0, s>>>(
          sums, p.parts, a.outputs, a.grad_bias, bias_f32);
    }
  }
  if (a.rows == 0) {
    if (a.grad_weight &&
        cudaMemsetAsync(a.grad_weight, 0, (size_t)a.outputs * a.inputs * sizeof(T), s) != cudaSuccess)
      return check_launch("linear_backward");
    return check_launch("linear_backward");
  }
  // what the forward left packed is read from there
  Packer<T> pack;
  Operand bw{}, bx{};
  if (a.grad_x)
    bw = a.weight_packed ? Operand{a.weight_packed, a.inputs, a.outputs, round8(a.inputs), true}
                         : pack.operand(a.weight, a.ldw, a.outputs, a.inputs, true, w);
  if (a.grad_weight)
    bx = a.x_packed ? Operand{a.x_packed, a.inputs, a.rows, round8(a.inputs), true}
                    : pack.operand(a.x, a.ldx, a.rows, a.inputs, true, x);
  pack.launch(s);
  EpilogueParams e{};
  if (a.grad_x) {  // dx = dz W: k runs over the outputs
    e.out = a.grad_x;
    if (int rc = launch_gemm<T>(d, bw, a.rows, a.inputs, p.dx, e, partial, s)) return rc;
  }
  if (a.grad_weight) {  // dW = dz^T x: k runs over the rows
    e.out = a.grad_weight;
    d.mn_major = true;
    if (int rc = launch_gemm<T>(d, bx, a.outputs, a.inputs, p.dw, e, partial, s)) return rc;
  }
  return check_launch("linear_backward");
}

template <typename T>
cudaError_t linear_device_errors(unsigned* flags, bool clear) {
  return read_device_errors(flags, clear);
}

}  // namespace nnue_ls
