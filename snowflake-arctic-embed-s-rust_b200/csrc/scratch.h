// Device scratch of calls that are asynchronous on a stream.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <map>
#include <memory>
#include <mutex>
#include <utility>
#include <vector>

namespace ae {

// Who may use a block, and until when:
//   A call that runs takes its stream's block. Only calls on that stream use it, one after the other, so it can be freed
//   once the stream has been waited for. Streams are told apart by their ids, which CUDA gives once: a handle can come
//   back for a new stream while the kernels of a destroyed one still run. (Asking for the capture and for the id takes
//   the host 73 ns a call.)
//   A call that is captured takes a block of the graph's own, whose address the graph replays at any time and on any
//   stream. The graph and what is instantiated from it hold the block as a user object; once the last of them is
//   gone it may serve another graph. It is not freed there, where CUDA allows no calls, but by release() or close().
class StreamScratch {
 public:
  StreamScratch() : kept_(std::make_shared<Kept>()) {}

  // At least `bytes` for a call on `st`, on the current device. May throw std::bad_alloc.
  cudaError_t take(cudaStream_t st, size_t bytes, uint8_t** out) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    cudaGraph_t graph = nullptr;
    cudaError_t e = cudaStreamGetCaptureInfo(st, &status, &id, &graph, nullptr, nullptr);
    if (e != cudaSuccess) return e;
    if (status == cudaStreamCaptureStatusInvalidated) return cudaErrorStreamCaptureInvalidated;
    Block b;
    if (status == cudaStreamCaptureStatusActive) e = take_captured({id, st}, graph, bytes, &b);
    else e = take_running(st, bytes, &b);
    *out = b.p;
    return e;
  }

  // Frees the block of `st`, which is not being captured, once its work is done, and the blocks of graphs that are gone.
  cudaError_t release(cudaStream_t st) {
    unsigned long long id = 0;
    cudaError_t e = cudaStreamGetId(st, &id);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return e;
    if (auto it = running_.find(id); it != running_.end()) {
      if (it->second.p) e = cudaFree(it->second.p);
      running_.erase(it);
    }
    std::vector<Block> gone;
    {
      std::lock_guard<std::mutex> lock(kept_->m);
      auto& all = kept_->all;
      for (const Block& b : kept_->idle) all.erase(std::find_if(all.begin(), all.end(), [&](const Block& o) { return o.p == b.p; }));
      gone.swap(kept_->idle);
    }
    for (const Block& b : gone)
      if (const cudaError_t f = cudaFree(b.p); f != cudaSuccess) e = f;
    return e;
  }

  // Frees everything. Graphs that hold a block must not run any more.
  void close() {
    for (auto& r : running_)
      if (r.second.p) cudaFree(r.second.p);
    running_.clear();
    std::vector<Block> all;
    {
      std::lock_guard<std::mutex> lock(kept_->m);
      all.swap(kept_->all);
      kept_->idle.clear();
      kept_->captured.clear();
      kept_->open = false;
    }
    for (const Block& b : all) cudaFree(b.p);
  }

 private:
  struct Block {
    uint8_t* p = nullptr;
    size_t bytes = 0;
  };
  using Capture = std::pair<unsigned long long, cudaStream_t>;  // a capture's id, and a stream that takes part in it

  // The blocks of graphs. Graphs may outlive the context, and are destroyed on any thread: the lock is held during no
  // CUDA call, which may itself be waiting for a thread that gives a block back.
  struct Kept {
    std::mutex m;
    bool open = true;
    std::vector<Block> all, idle;
    std::map<Capture, Block> captured;
  };
  struct Held {
    std::shared_ptr<Kept> kept;
    Block block;
  };

  // Allocations are no part of a capture, this thread's or another's.
  struct Relaxed {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
  };

  cudaError_t take_running(cudaStream_t st, size_t bytes, Block* out) {
    unsigned long long id = 0;
    cudaError_t e = cudaStreamGetId(st, &id);
    if (e != cudaSuccess) return e;
    Block& b = running_[id];
    if (b.bytes < bytes) {
      Relaxed relaxed;
      const size_t want = std::max(bytes, b.bytes + b.bytes / 2);
      if (b.p) {
        if ((e = cudaStreamSynchronize(st)) != cudaSuccess) return e;
        cudaFree(b.p);
        b = Block{};
      }
      if ((e = cudaMalloc(reinterpret_cast<void**>(&b.p), want)) != cudaSuccess) {
        b.p = nullptr;
        return e;
      }
      b.bytes = want;
    }
    *out = b;
    return cudaSuccess;
  }

  // Calls captured from one stream follow one another in the graph, so they share its block until one needs a larger one;
  // the graph then holds both.
  cudaError_t take_captured(const Capture& key, cudaGraph_t graph, size_t bytes, Block* out) {
    auto held = std::make_unique<Held>();
    held->kept = kept_;
    Block& b = held->block;
    size_t had = 0;
    {
      std::lock_guard<std::mutex> lock(kept_->m);
      const Block now = kept_->captured[key];
      if (now.bytes >= bytes) {
        *out = now;
        return cudaSuccess;
      }
      had = now.bytes;
      auto& idle = kept_->idle;
      auto best = idle.end();
      for (auto i = idle.begin(); i != idle.end(); ++i)
        if (i->bytes >= bytes && (best == idle.end() || i->bytes < best->bytes)) best = i;
      if (best != idle.end()) {
        b = *best;
        idle.erase(best);
      } else {  // room for one more, so that nothing below allocates
        kept_->all.reserve(kept_->all.size() + 1);
        idle.reserve(kept_->all.size() + 1);
      }
    }
    if (!b.p) {
      Relaxed relaxed;
      b.bytes = std::max(bytes, had + had / 2);
      if (const cudaError_t e = cudaMalloc(reinterpret_cast<void**>(&b.p), b.bytes); e != cudaSuccess) return e;
      std::lock_guard<std::mutex> lock(kept_->m);
      kept_->all.push_back(b);
    }
    *out = b;
    cudaUserObject_t object = nullptr;
    cudaError_t e = cudaUserObjectCreate(&object, held.get(), give_back, 1, cudaUserObjectNoDestructorSync);
    if (e != cudaSuccess) {
      give_back(held.release());
      return e;
    }
    held.release();  // the user object's
    // on failure the block stays with the object, which nothing releases: it is freed with the context
    if ((e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove)) != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(kept_->m);
    kept_->captured[key] = *out;
    return cudaSuccess;
  }

  static void CUDART_CB give_back(void* p) {
    std::unique_ptr<Held> held(static_cast<Held*>(p));
    Kept& k = *held->kept;
    std::lock_guard<std::mutex> lock(k.m);
    if (!k.open) return;
    for (auto i = k.captured.begin(); i != k.captured.end();)
      i = i->second.p == held->block.p ? k.captured.erase(i) : std::next(i);
    k.idle.push_back(held->block);
  }

  std::map<unsigned long long, Block> running_;
  std::shared_ptr<Kept> kept_;
};

}  // namespace ae
