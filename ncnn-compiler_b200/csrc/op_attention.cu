// Attention of one sequence's tokens to another's (an encoder's states) on device arrays (ncnn_b200_op_cross_attention):
//   o[b][i][h] = sum_j softmax_j(scale * q[b][i][h] . k[b][j][h']) v[b][j][h']
// over the keys j < kv_lens[b] with key_mask[b][j] != 0; h' = h / (heads / kv_heads).  A sequence without such a key has
// zeros for its result.  What lies at keys that take no part is never used, NaN or infinity as it may be.
#include <cmath>

#include "op_attention.h"


#include "attend_f32.cuh"
#include "attend_few.cuh"
#include "tc_attend.cuh"
#include "tc_attend_short.cuh"

namespace nb {
namespace {

// What ncnn_b200_op_test_hooks asked for.
struct {
  std::atomic<int> stall{0}, registers{0};
  std::atomic<unsigned long long> wait_ns{0};
} g_hooks;

// The devices that calls on the tensor cores went to (as bits).
std::atomic<uint64_t> g_waited_on{0};

void will_wait_on(int device) {
  const uint64_t bit = 1ull << (device & 63);
  if (!(g_waited_on.load(std::memory_order_relaxed) & bit)) g_waited_on.fetch_or(bit, std::memory_order_relaxed);
}

// ------------------------------------------------------------------ tensor cores
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static const EncodeTiledFn fn = [] {
    cudaDriverEntryPointQueryResult query;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &query) != cudaSuccess || query != cudaDriverEntryPointSuccess) f = nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// [sequence][head][row][component] as TMA sees it, boxes of 128 rows (results: 32) of 64 components.  An axis that all heads or sequences
// share (stride 0) has one entry: `step` says what to multiply its index with.
bool encode_rows(CUtensorMap* map, bool half, const void* base, int d, long long rows, long long row, int heads, long long head, int batch,
                 long long seq, int* step, int box_rows = kAttRows) {
  const int head_extent = head == 0 ? 1 : heads, batch_extent = seq == 0 ? 1 : batch;
  if (step != nullptr) {
    step[0] = head == 0 ? 0 : 1;
    step[1] = seq == 0 ? 0 : 1;
  }
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(head_extent), static_cast<cuuint64_t>(batch_extent)};
  // an axis of one entry is never stepped over: any valid stride will do
  const cuuint64_t any = (static_cast<cuuint64_t>(d) * 2 + 15) / 16 * 16;
  const cuuint64_t strides[3] = {rows == 1 ? any : static_cast<cuuint64_t>(row) * 2, head_extent == 1 ? any : static_cast<cuuint64_t>(head) * 2,
                                 batch_extent == 1 ? any : static_cast<cuuint64_t>(seq) * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1}, ones[4] = {1, 1, 1, 1};
  return encode_tiled()(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box,
                        ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether `count` elements of `size` bytes can be moved at a time: starts, and strides of the axes that are stepped over.
bool rows_of(const AttendParams& p, int count, int size) {
  auto ok = [&](const void* base, std::initializer_list<std::pair<long long, long long>> axes) {
    if (reinterpret_cast<uintptr_t>(base) % (count * size) != 0) return false;
    for (const auto& a : axes)
      if (a.second > 1 && a.first % count != 0) return false;
    return true;
  };
  return p.d % count == 0 && ok(p.q, {{p.q_batch, p.batch}, {p.q_row, p.lq}, {p.q_head, p.heads}}) &&
         ok(p.k, {{p.k_batch, p.batch}, {p.k_row, p.lk}, {p.k_head, p.kv_heads}}) &&
         ok(p.v, {{p.v_batch, p.batch}, {p.v_row, p.lk}, {p.v_head, p.kv_heads}}) &&
         ok(p.o, {{p.o_batch, p.batch}, {p.o_row, p.lq}, {p.o_head, p.heads}});
}

// Dynamic shared memory above 48 KB is granted to a kernel once per device.  `registers`: what the kernel's roles share out
// between them; compiled for fewer, their setmaxnreg would wait for ever.
template <class K>
cudaError_t grant_smem(K kernel, int bytes, int device, std::atomic<uint64_t>* granted, int registers = 0) {
  const uint64_t bit = 1ull << (device & 63);
  const int as_if = registers > 0 ? g_hooks.registers.load(std::memory_order_relaxed) : 0;
  if (as_if != 0 && as_if != registers) return cudaErrorInvalidKernelImage;
  if (device < 64 && (granted->load(std::memory_order_acquire) & bit)) return cudaSuccess;
  if (registers > 0) {
    cudaFuncAttributes a{};
    if (const cudaError_t e = cudaFuncGetAttributes(&a, kernel); e != cudaSuccess) return e;
    if (a.numRegs != registers) return cudaErrorInvalidKernelImage;
  }
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && device < 64) granted->fetch_or(bit, std::memory_order_acq_rel);
  return e;
}

struct TcMaps {
  alignas(64) CUtensorMap q, k, v, o;
};

bool fill_tc(const AttendParams& a, bool half, TcAttendParams* p, TcMaps* m) {
  p->a = a;
  p->scale_log2 = a.scale * 1.44269504088896340736f;
  p->wait_ns = kTcWaitLimitNs;
  p->stall = g_hooks.stall.load(std::memory_order_relaxed);
  if (const unsigned long long ns = g_hooks.wait_ns.load(std::memory_order_relaxed); ns != 0) p->wait_ns = ns;
  return encode_rows(&m->q, half, a.q, a.d, a.lq, a.q_row, a.heads, a.q_head, a.batch, a.q_batch, p->q_step) &&
         encode_rows(&m->k, half, a.k, a.d, a.lk, a.k_row, a.kv_heads, a.k_head, a.batch, a.k_batch, p->k_step) &&
         encode_rows(&m->v, half, a.v, a.d, a.lk, a.v_row, a.kv_heads, a.v_head, a.batch, a.v_batch, p->v_step) &&
         encode_rows(&m->o, half, a.o, a.d, a.lq, a.o_row, a.heads, a.o_head, a.batch, a.o_batch, nullptr, 32);
}

// A launch that did not happen because of the kernel itself.
int refused_kernel(cudaError_t e) {
  cudaGetLastError();
  return op_fail(NCNN_B200_STATUS_RUNTIME, std::string("op_cross_attention: the kernel was not granted its registers and shared memory: ") + cudaGetErrorString(e));
}
int no_maps() { return op_fail(NCNN_B200_STATUS_RUNTIME, "op_cross_attention: the tensor maps could not be made"); }

template <class T, int D>
int launch_short(const AttendParams& a, int device, int sms, cudaStream_t st) {
  using Shape = TcShortShape<D>;
  TcShortParams p{};
  TcMaps m;
  if (!fill_tc(a, std::is_same<T, __half>::value, &p.t, &m)) return no_maps();
  static std::atomic<uint64_t> granted{0};
  if (const cudaError_t e = grant_smem(tc_attend_short_kernel<T, D>, Shape::kSmem, device, &granted, Shape::kRegsLaunch); e != cudaSuccess) return refused_kernel(e);
  p.row_tiles = (a.lq + kAttRows - 1) / kAttRows;
  p.tiles = p.row_tiles * a.heads * a.batch;
  will_wait_on(device);
  return op_launched("op_cross_attention",
                     op_launch(tc_attend_short_kernel<T, D>, dim3(std::min(sms, p.tiles)), Shape::kThreads, Shape::kSmem, st, 0, p, m.q, m.k, m.v, m.o));
}

template <class T, int D, int TILES>
int launch_tc(const AttendParams& a, int device, cudaStream_t st) {
  using Shape = TcAttendShape<D, TILES>;
  TcAttendParams p{};
  TcMaps m;
  if (!fill_tc(a, std::is_same<T, __half>::value, &p, &m)) return no_maps();
  static std::atomic<uint64_t> granted{0};
  const int registers = Shape::kShareRegs ? Shape::kRegsLaunch : 0;
  if (const cudaError_t e = grant_smem(tc_attend_kernel<T, D, TILES>, Shape::kSmem, device, &granted, registers); e != cudaSuccess) return refused_kernel(e);
  const dim3 grid((a.lq + kAttRows * TILES - 1) / (kAttRows * TILES), a.heads, a.batch);
  will_wait_on(device);
  return op_launched("op_cross_attention", op_launch(tc_attend_kernel<T, D, TILES>, grid, Shape::kThreads, Shape::kSmem, st, 0, p, m.q, m.k, m.v, m.o));
}

template <class T>
int attend_tc(const AttendParams& a, int device, int sms, cudaStream_t st) {
  // Two tiles to a CTA, whose MMAs and softmaxes take turns, or one, and two CTAs to an SM (heads above 128: one).  Device times, bf16,
  // two and one: 2048 queries over 2048 keys, 16 heads of 128 37 and 40 us (of 64: 30 and 32); 4096 over 4096, 40 heads of 128 360 and
  // 363; but 4096 over 4096, 10 heads of 128 118 and 114, and grids that do not fill the device: 1024 over 1024, 10 heads of 64
  // 16.8 and 14.3, 300 over 3000, 16 heads of 128 44 and 38.  Full grids decide.
  const bool two = a.lq > kAttRows;
  const long long tiles = static_cast<long long>((a.lq + kAttRows - 1) / kAttRows) * a.heads * a.batch;
  // one block of keys and a tile for every SM: 4096 queries over 77 keys (8 sequences, 10 heads of 64) 28.6 us of device time, 57 with
  // a CTA to two tiles
  if (a.lk <= kAttRows && a.d <= 128 && tiles >= sms && tiles < (1 << 30))
    return a.d <= 64 ? launch_short<T, 64>(a, device, sms, st) : launch_short<T, 128>(a, device, sms, st);
  if (a.d <= 64) return two ? launch_tc<T, 64, 2>(a, device, st) : launch_tc<T, 64, 1>(a, device, st);
  if (a.d <= 128) return two ? launch_tc<T, 128, 2>(a, device, st) : launch_tc<T, 128, 1>(a, device, st);
  return a.d <= 192 ? launch_tc<T, 192, 1>(a, device, st) : launch_tc<T, 256, 1>(a, device, st);
}

template <class T, int D, int WARPS, int STAGES, int BLOCKS>
int launch_few(const AttendParams& a, int device, int ranks, cudaStream_t st) {
  FewParams p{};
  p.a = a;
  p.scale_log2 = a.scale * 1.44269504088896340736f;
  const int shared = a.heads / a.kv_heads;
  p.row_tiles = (a.lq * shared + kFewRows - 1) / kFewRows;
  constexpr int smem = sizeof(FewShared<T, D, WARPS, STAGES>);
  static std::atomic<uint64_t> granted{0};
  const auto kernel = k_attend_few<T, D, WARPS, STAGES, BLOCKS>;
  if (const cudaError_t e = grant_smem(kernel, smem, device, &granted); e != cudaSuccess) return refused_kernel(e);
  if (ranks > 8)
    if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); e != cudaSuccess) return refused_kernel(e);
  return op_launched("op_cross_attention", op_launch(kernel, dim3(ranks, a.kv_heads * p.row_tiles, a.batch), WARPS * 32, smem, st, ranks, p));
}

// Whether a call is one of few queries.  At most two tiles of 16 to a key head always are.  So are up to 160 tiles over 512 keys or
// more where the tensor-core kernel, which gives a head's 128 queries to one CTA from the first key to the last, would use less
// than half of the SMs.  Device times, bf16, this kernel and that one: 8 heads of 64 (128) of 64 queries over 4096 keys 12 (16) us
// against 46 (49), of 128 queries 16 (24) against 47 (49), of 256 over 8192 keys (128 tiles) 46 (74) against 104 (108); 32 heads
// of 64 queries over 1024 keys (128 tiles) 10.6 (15.3) against 14.2 (15.4).
bool few_queries(const AttendParams& p, int sms) {
  const long long rows = static_cast<long long>(p.lq) * (p.heads / p.kv_heads), row_tiles = (rows + kFewRows - 1) / kFewRows;
  if (p.kv_heads * row_tiles > 65535) return false;
  const long long ctas = static_cast<long long>(p.batch) * p.heads * ((p.lq + kAttRows - 1) / kAttRows);
  return rows <= 2 * kFewRows || (p.batch * p.kv_heads * row_tiles <= 160 && p.lk >= 512 && 2 * ctas <= sms);
}

template <class T>
int attend_few(const AttendParams& a, int device, int sms, cudaStream_t st) {
  const long long rows = static_cast<long long>(a.lq) * (a.heads / a.kv_heads);
  const long long tiles = static_cast<long long>(a.batch) * a.kv_heads * ((rows + kFewRows - 1) / kFewRows);
  // Few tiles (a cluster of 8 to each leaves SMs idle): CTAs of 8 warps with deep rings, one to an SM, up to 16 to a tile while
  // each of their warps has two tiles of keys.  4 tiles of 20000 keys: 24.6 us, against 28.7 with CTAs of 4 warps.
  if (a.d <= 128 && tiles * 8 < sms && a.lk >= 4096) {
    int ranks = 8;
    while (ranks < 16 && tiles * ranks * 2 <= sms && a.lk >= ranks * 512) ranks *= 2;
    return a.d <= 64 ? launch_few<T, 64, 8, 6, 1>(a, device, ranks, st) : launch_few<T, 128, 8, 3, 1>(a, device, ranks, st);
  }
  // Otherwise CTAs of 4 warps, two (heads of 64: three) to an SM, and as many to a tile as the device holds at once: a CTA costs
  // some 3 us of its own (512 tiles of 2048 keys: 103 us with one to a tile, 115 with two, 120 with four; 64 tiles of 8192: 72,
  // 45, 38 and 49 us with 1, 2, 4 and 8).  Sequences of different lengths even out over four times as many (512 tiles of
  // ragged lengths: 129, 113, 119 us).
  const long long most = (a.lens != nullptr ? 8ll : 2ll) * sms;
  int ranks = 1;
  while (ranks < 8 && tiles * ranks * 2 <= most && a.lk > ranks * 64) ranks *= 2;
  if (a.d <= 64) return launch_few<T, 64, 4, 4, 3>(a, device, ranks, st);
  return a.d <= 128 ? launch_few<T, 128, 4, 3, 2>(a, device, ranks, st) : launch_few<T, 256, 4, 3, 1>(a, device, ranks, st);
}

// ------------------------------------------------------------------ CUDA cores
template <class T, int D, int ROWS, bool WIDE>
cudaError_t launch_split(F32Params& p, int sms, cudaStream_t st) {
  const AttendParams& a = p.a;
  const long long rows = static_cast<long long>(a.lq) * (a.heads / a.kv_heads);
  p.row_tiles = static_cast<int>((rows + ROWS - 1) / ROWS);
  const long long tiles = static_cast<long long>(a.batch) * a.kv_heads * p.row_tiles;
  // enough CTAs to a tile to fill the device twice over, while each of their warps has eight keys
  int ranks = 1;
  while (ranks < 8 && tiles * ranks * 2 <= 4ll * sms && a.lk > ranks * kSplitWarps * 8) ranks *= 2;
  return op_launch(k_attend_split<T, D, ROWS, WIDE>, dim3(ranks, a.kv_heads * p.row_tiles, a.batch), kSplitWarps * 32, 0, st, ranks, p);
}

template <class T, int D, int TM, int KEYS, int THREADS, bool WIDE>
cudaError_t launch_tile(F32Params p, int device, int sms, cudaStream_t st) {
  using Shape = TileShape<D, TM, KEYS, THREADS>;
  static std::atomic<uint64_t> granted{0};
  auto kernel = k_attend_tile<T, D, TM, KEYS, THREADS, WIDE>;
  if (const cudaError_t e = grant_smem(kernel, Shape::kSmem, device, &granted); e != cudaSuccess) return e;
  const long long rows = static_cast<long long>(p.a.lq) * (p.a.heads / p.a.kv_heads);
  const long long row_tiles = (rows + Shape::kRows - 1) / Shape::kRows, tiles = row_tiles * p.a.kv_heads * p.a.batch;
  // CTAs to a tile: what the device holds at once, while each has a block of keys; no more than the blocks are dealt evenly to
  const long long blocks = (p.a.lk + KEYS - 1) / KEYS, most = std::max<long long>(1, std::min<long long>({kF32Ranks, Shape::kBlocksPerSm * sms / tiles, blocks}));
  const long long deal = (blocks + most - 1) / most;  // blocks of the busiest CTA
  p.ranks = static_cast<int>((blocks + deal - 1) / std::max<long long>(1, deal));
  p.ranks = std::max(p.ranks, 1);
  return op_launch(kernel, dim3(static_cast<unsigned>(row_tiles * p.ranks), p.a.kv_heads, p.a.batch), THREADS, Shape::kSmem, st, p.ranks, p);
}

template <class T, bool WIDE>
cudaError_t attend_f32(const AttendParams& a, int device, int sms, cudaStream_t st) {
  F32Params p{};
  p.a = a;
  p.scale_log2 = a.scale * 1.44269504088896340736f;
  const long long rows = static_cast<long long>(a.lq) * (a.heads / a.kv_heads);
  // Up to 16 rows to a key head in tiles of a few rows over split keys, more in tiles of 64 or 128 rows.  Device times of split and
  // tiled keys over 4096 keys, one key head of 128: 23 and 135 us with 16 rows, 23 and 136 with 48; eight: 81 and 136 with 16, 106
  // and 136 with 24, 148 and 137 with 48; 64 key heads of 64 over 1024 keys: 35 and 42 with 8, 57 and 42 with 16, 92 and 43 with 17.
  // (The crossing lies at 8 rows where key heads fill the device and above 48 where there are few: 16 is between them.)
  if (rows <= 16 && a.kv_heads * rows <= 65535) {
    if (rows == 1) {
      if (a.d <= 64) return launch_split<T, 64, 1, WIDE>(p, sms, st);
      if (a.d <= 128) return launch_split<T, 128, 1, WIDE>(p, sms, st);
      return launch_split<T, 256, 1, WIDE>(p, sms, st);
    }
    if (a.d <= 64) return launch_split<T, 64, 4, WIDE>(p, sms, st);
    if (a.d <= 128) return launch_split<T, 128, 4, WIDE>(p, sms, st);
    return launch_split<T, 256, 2, WIDE>(p, sms, st);
  }
  if (a.d <= 64) {
    // 128 rows to a tile where those fill the device
    if (a.batch * static_cast<long long>(a.kv_heads) * ((rows + 127) / 128) >= 2 * sms) return launch_tile<T, 64, 8, 64, 256, WIDE>(p, device, sms, st);
    return launch_tile<T, 64, 4, 64, 256, WIDE>(p, device, sms, st);
  }
  if (a.d <= 128) return launch_tile<T, 128, 4, 64, 512, WIDE>(p, device, sms, st);
  return launch_tile<T, 256, 4, 32, 512, WIDE>(p, device, sms, st);
}

// Every stride an axis of more than one entry is stepped with has to be a stride that TMA takes: positive and below 2^40 bytes.
bool tma_strides(const AttendParams& p) {
  auto ok = [](long long stride, long long extent, bool shared) { return extent == 1 || ((stride > 0 || (shared && stride == 0)) && stride < (1ll << 38)); };
  return ok(p.q_batch, p.batch, true) && ok(p.q_row, p.lq, false) && ok(p.q_head, p.heads, true) && ok(p.k_batch, p.batch, true) &&
         ok(p.k_row, p.lk, false) && ok(p.k_head, p.kv_heads, true) && ok(p.v_batch, p.batch, true) && ok(p.v_row, p.lk, false) &&
         ok(p.v_head, p.kv_heads, true) && ok(p.o_batch, p.batch, false) && ok(p.o_row, p.lq, false) && ok(p.o_head, p.heads, false);
}

}  // namespace
}  // namespace nb

extern "C" int ncnn_b200_op_test_hooks(int32_t stall, uint64_t wait_ns, int32_t registers) {
  nb::g_hooks.stall.store(stall != 0 ? 1 : 0);
  nb::g_hooks.wait_ns.store(wait_ns);
  nb::g_hooks.registers.store(registers);
  return NCNN_B200_STATUS_SUCCESS;
}

extern "C" int ncnn_b200_op_check_status(void) {
  using namespace nb;
  return op_guarded("op_check_status", [&]() -> int {
    // The kernels count for ever, and each thread remembers what it has been told: no thread takes an answer from another, and no
    // count is lost between being read and being cleared.
    static thread_local unsigned told[64] = {};
    bool ran_out = false;
    auto failed = [] { return op_fail(NCNN_B200_STATUS_RUNTIME, std::string("op_check_status: ") + cudaGetErrorString(cudaGetLastError())); };
    if (cudaDeviceSynchronize() != cudaSuccess) return failed();
    const uint64_t devices = g_waited_on.load();
    for (int d = 0; d < 64; ++d) {
      if (!(devices >> d & 1u)) continue;
      DeviceGuard guard(d);
      unsigned count = 0;
      if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(&count, g_attend_gave_up, sizeof count) != cudaSuccess) return failed();
      ran_out = ran_out || count != told[d];
      told[d] = count;
    }
    return !ran_out ? NCNN_B200_STATUS_SUCCESS
                    : op_fail(NCNN_B200_STATUS_TIMEOUT, "op_check_status: a wait inside an operator's kernel ran out; its result is not valid");
  });
}

extern "C" int ncnn_b200_op_cross_attention(const void* q, const void* k, const void* v, void* o, int32_t type, int64_t batch, int64_t lq,
                                            int64_t lk, int32_t heads, int32_t kv_heads, int32_t head_dim, const int64_t* strides,
                                            const int32_t* kv_lens, const uint8_t* key_mask, float scale, void* stream) {
  using namespace nb;
  static const char* kOp = "op_cross_attention";
  return op_guarded(kOp, [&]() -> int {
    if (!op_type_ok(type)) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_cross_attention: unknown element type");
    if (batch < 0 || lq < 0 || lk < 0 || batch > 65535 || lq > (1 << 30) || lk > (1 << 30) || heads <= 0 || heads > 65535 || kv_heads <= 0 ||
        heads % kv_heads != 0 || head_dim <= 0 || head_dim > 256)
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE,
                     "op_cross_attention: batch 0 to 65535, lengths 0 to 2^30, heads a multiple of kv_heads up to 65535, head_dim 1 to 256");
    // (the kernels' exponentials are powers of two: scale / ln 2 has to be a number, too)
    if (!(scale >= 0.0f) || std::isinf(scale * 1.44269504088896340736f))
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_cross_attention: scale must not be negative, and scale / ln 2 finite");
    if (batch == 0 || lq == 0) return NCNN_B200_STATUS_SUCCESS;
    if (q == nullptr || o == nullptr || (lk > 0 && (k == nullptr || v == nullptr)))
      return op_fail(NCNN_B200_STATUS_NULL_POINTER, "op_cross_attention: NULL argument");
    const int size = op_elem_bytes(type);
    if (!op_starts(q, size) || !op_starts(k, size) || !op_starts(v, size) || !op_starts(o, size) || !op_starts(kv_lens, 4))
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_cross_attention: an array does not start at a multiple of its elements' size");
    if (o == q || o == k || o == v) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_cross_attention: the result must not lie over an input");
    AttendParams p{};
    p.q = q;
    p.k = k;
    p.v = v;
    p.o = o;
    p.batch = static_cast<int>(batch);
    p.lq = static_cast<int>(lq);
    p.lk = static_cast<int>(lk);
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.d = head_dim;
    p.lens = kv_lens;
    p.mask = key_mask;
    p.scale = scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(head_dim)) : scale;
    if (strides != nullptr) {
      for (int i = 0; i < 12; ++i)
        if (strides[i] < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_cross_attention: a stride is negative");
      std::tie(p.q_batch, p.q_row, p.q_head) = std::make_tuple(strides[0], strides[1], strides[2]);
      std::tie(p.k_batch, p.k_row, p.k_head) = std::make_tuple(strides[3], strides[4], strides[5]);
      std::tie(p.v_batch, p.v_row, p.v_head) = std::make_tuple(strides[6], strides[7], strides[8]);
      std::tie(p.o_batch, p.o_row, p.o_head) = std::make_tuple(strides[9], strides[10], strides[11]);
      // the result's axes from the innermost out: each has to step over what lies inside it
      std::array<std::pair<int64_t, int64_t>, 3> axes = {{{p.o_batch, batch}, {p.o_row, lq}, {p.o_head, heads}}};
      std::sort(axes.begin(), axes.end());
      int64_t extent = head_dim;
      for (const auto& a : axes) {
        if (a.second == 1) continue;
        if (a.first < extent) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_cross_attention: the result's rows overlap");
        if (a.first > (1ll << 50) / a.second) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_cross_attention: a stride is too large");
        extent = a.first * (a.second - 1) + extent;
      }
      for (int i = 0; i < 9; ++i)
        if (strides[i] > (1ll << 50) / std::max<int64_t>({batch, lq, lk, heads}))
          return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_cross_attention: a stride is too large");
    } else {
      p.q_head = p.o_head = p.k_head = p.v_head = head_dim;
      p.q_row = p.o_row = static_cast<long long>(heads) * head_dim;
      p.k_row = p.v_row = static_cast<long long>(kv_heads) * head_dim;
      p.q_batch = p.o_batch = p.q_row * lq;
      p.k_batch = p.v_batch = p.k_row * lk;
    }
    std::string why;
    const int device = op_common_device(kOp, {q, o, lk > 0 ? k : nullptr, lk > 0 ? v : nullptr, kv_lens, key_mask}, &why);
    if (device < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, why);
    DeviceGuard guard(device);
    if (lq > (1ll << 30) / (heads / kv_heads) || batch * lq * heads > (1ll << 33)) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_cross_attention: more than 2^33 rows");
    if (p.batch * static_cast<long long>(p.heads) > (1 << 30)) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_cross_attention: too many heads");
    const int sms = op_sm_count(device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type != NCNN_B200_F32 && p.lk > 0 && rows_of(p, 8, 2)) {
      if (few_queries(p, sms)) return type == NCNN_B200_F16 ? attend_few<__half>(p, device, sms, st) : attend_few<__nv_bfloat16>(p, device, sms, st);
      if (tma_strides(p)) {
        if (encode_tiled() == nullptr) return op_fail(NCNN_B200_STATUS_RUNTIME, "op_cross_attention: cuTensorMapEncodeTiled is not available from this driver");
        return type == NCNN_B200_F16 ? attend_tc<__half>(p, device, sms, st) : attend_tc<__nv_bfloat16>(p, device, sms, st);
      }
    }
    return op_by_type(type, [&](auto t) {
      using T = decltype(t);
      // (16-bit rows come here when they are not aligned: element by element)
      if constexpr (sizeof(T) == 4)
        if (rows_of(p, 4, sizeof(T))) return op_launched(kOp, attend_f32<T, true>(p, device, sms, st));
      return op_launched(kOp, attend_f32<T, false>(p, device, sms, st));
    });
  });
}
