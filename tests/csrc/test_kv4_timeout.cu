// GPU run: a wait of the 4-bit attention's ring that runs out ends, is reported and leaves the
// tracked weights alone. The copy that it waits for is never issued, by a kernel made for that.
#include <cuda_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../llm_fa_b200/csrc/kv4_attention.cuh"

using namespace llmfa;

constexpr int kPage = 64, kTokens = 50, kRows = 4, kWorkers = 8, kStages = 2;
using Ring = Kv4Ring<kStages, kv4_block_bytes(2)>;

__global__ void starved(Kv4Seqs seqs, unsigned long long limit_ns, int worker, uint8_t* gave_up,
                        uint32_t* pending) {
  __shared__ __align__(128) uint8_t tiles[kStages * Ring::kTileBytes];
  __shared__ uint64_t bar[kStages + 1];
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(ptx::smem_u32(&bar[s]), 1);
    bar[kStages] = 0;
    ptx::fence_mbar_init();
  }
  __syncwarp();
  Ring ring{ptx::smem_u32(tiles), ptx::smem_u32(bar)};
  ring.pending = kStages;  // as if both had been issued
  for (int s = 0; s < kStages; ++s) {
    ring.wait(limit_ns);
    ring.release();
  }
  ring.report(seqs);
  if (threadIdx.x == 0) {
    gave_up[worker] = ring.failed();
    *pending = ring.pending;
  }
}

#define CHECK(c) \
  do { \
    if (!(c)) { \
      std::printf("failed: %s (line %d), %s\n", #c, __LINE__, cudaGetErrorString(cudaGetLastError())); \
      std::exit(1); \
    } \
  } while (0)

template <typename T>
T* zeros(size_t n) {
  void* p = nullptr;
  CHECK(cudaMalloc(&p, n * sizeof(T)) == cudaSuccess && cudaMemset(p, 0, n * sizeof(T)) == cudaSuccess);
  return static_cast<T*>(p);
}
template <typename T>
std::vector<T> host(const T* p, size_t n) {
  std::vector<T> v(n);
  CHECK(cudaMemcpy(v.data(), p, n * sizeof(T), cudaMemcpyDeviceToHost) == cudaSuccess);
  return v;
}

int main() {
  // one page of one head: zero keys, queries and log-sum-exps, so that each row gives a token 1
  Kv4AttnParams p{};
  p.pool = Kv4Pool{zeros<uint8_t>(kPage / 16 * kv4_block_bytes(2)), zeros<int32_t>(kPage),
                   zeros<float>(kPage), 1, 1, 6, 2};
  const int32_t n = kTokens;
  int32_t* lengths = zeros<int32_t>(1);
  CHECK(cudaMemcpy(lengths, &n, 4, cudaMemcpyHostToDevice) == cudaSuccess);
  p.seqs = Kv4Seqs{zeros<int32_t>(1), 1, 1, 1, lengths, zeros<int>(1)};
  p.q = Kv4RowView{zeros<uint16_t>(kRows * 128), 0, 0, 128};
  p.row_lse = zeros<float>(kRows);
  p.scores = zeros<float>(kPage * kRows);
  p.gave_up = zeros<uint8_t>(kWorkers);
  p.heads_q = p.group = kRows;
  p.tokens = p.row_tiles = p.causal = 1;
  p.workers = kWorkers;
  p.page_stride = kPage / 16 * kv4_block_bytes(2);
  p.scale_log2 = 1.f;
  p.decay = 0.5f;
  p.timeout_ns = 1000000000ull;
  uint32_t* pending = zeros<uint32_t>(1);

  auto kept = [&] { kv4_sum_weights_kernel<<<1, kKv4SumThreads, kRows * sizeof(float)>>>(p); };
  auto again = [&] {
    constexpr auto kernel = kv4_weights_kernel<__nv_bfloat16, 1, 2, 8, 3, 2>;
    const int bytes = sizeof(Kv4WeightsSmem<1, 2, 8, 3>) + kv4_plan_bytes(1);
    CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess);
    kernel<<<2, 8 * 32, bytes>>>(p);
  };
  auto weights_are = [&](float w) {
    CHECK(cudaDeviceSynchronize() == cudaSuccess);
    const auto got = host(p.pool.weights, kPage);
    for (int i = 0; i < kPage; ++i) CHECK(got[i] == (i < kTokens ? w : 0.f));
  };
  kept();
  weights_are(4.f);
  again();
  weights_are(6.f);  // 0.5 * 4 + 4
  CHECK(host(p.seqs.status, 1)[0] == 0);
  for (int worker : {0, 5, kWorkers - 1}) {
    CHECK(cudaMemset(p.gave_up, 0, kWorkers) == cudaSuccess);
    CHECK(cudaMemset(p.seqs.status, 0, 4) == cudaSuccess);
    starved<<<1, 32>>>(p.seqs, 20000, worker, p.gave_up, pending);
    CHECK(cudaDeviceSynchronize() == cudaSuccess);
    CHECK(host(p.seqs.status, 1)[0] == kStatusTimeout + kSiteKv4Tile);
    CHECK(host(pending, 1)[0] == 0);
    const auto flags = host(p.gave_up, kWorkers);
    for (int i = 0; i < kWorkers; ++i) CHECK(flags[i] == (i == worker));
    kept();
    weights_are(6.f);
    again();
    weights_are(6.f);
  }
  CHECK(cudaMemset(p.gave_up, 0, kWorkers) == cudaSuccess);
  again();
  weights_are(7.f);
  std::printf("ok\n");
  return 0;
}
