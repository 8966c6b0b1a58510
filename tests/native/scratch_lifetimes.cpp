// Lifetimes of csrc/scratch.h on a stand-in for the CUDA runtime: every block that a graph or a running kernel may still
// use is one that was not freed and is nobody else's. Prints the first claim that does not hold and returns 1.
#include <cstdio>
#include <cstdlib>
#include <set>

#include "scratch.h"

// ------------------------------------------------------------------------------------- the stand-in
struct CUstream_st {
  unsigned long long id = 0, capture = 0;  // capture: 0 while nothing is captured
  cudaGraph_t graph = nullptr;
  int waits = 0;
};
struct CUuserObject_st {
  void* p;
  cudaHostFn_t destroy;
};
struct CUgraph_st {
  std::vector<cudaUserObject_t> objects;
  ~CUgraph_st() {
    for (auto o : objects) {
      o->destroy(o->p);
      delete o;
    }
  }
};

static std::set<void*> g_live;
static cudaStreamCaptureMode g_mode = cudaStreamCaptureModeGlobal;
static bool g_capturing = false, g_unsafe = false, g_no_memory = false, g_no_object = false;

static void unsafe() { g_unsafe |= g_capturing && g_mode != cudaStreamCaptureModeRelaxed; }

extern "C" {
cudaError_t cudaStreamGetCaptureInfo_v2(cudaStream_t s, cudaStreamCaptureStatus* status, unsigned long long* id,
                                        cudaGraph_t* graph, const cudaGraphNode_t**, size_t*) {
  *status = s->capture ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
  *id = s->capture;
  *graph = s->graph;
  return cudaSuccess;
}
cudaError_t cudaStreamGetId(cudaStream_t s, unsigned long long* id) { return *id = s->id, cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t s) { return unsafe(), ++s->waits, cudaSuccess; }
cudaError_t cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode* m) { return std::swap(*m, g_mode), cudaSuccess; }
cudaError_t cudaMalloc(void** p, size_t n) {
  unsafe();
  if (g_no_memory) return cudaErrorMemoryAllocation;
  g_live.insert(*p = std::malloc(n));
  return cudaSuccess;
}
cudaError_t cudaFree(void* p) {
  unsafe();
  if (!g_live.erase(p)) return cudaErrorInvalidValue;
  std::free(p);
  return cudaSuccess;
}
cudaError_t cudaUserObjectCreate(cudaUserObject_t* o, void* p, cudaHostFn_t destroy, unsigned, unsigned) {
  if (g_no_object) return cudaErrorMemoryAllocation;
  *o = new CUuserObject_st{p, destroy};
  return cudaSuccess;
}
cudaError_t cudaGraphRetainUserObject(cudaGraph_t g, cudaUserObject_t o, unsigned, unsigned) {
  return g->objects.push_back(o), cudaSuccess;
}
}

// ------------------------------------------------------------------------------------------ claims
static void claim(bool holds, const char* what) {
  if (holds) return;
  std::printf("%s\n", what);
  std::exit(1);
}

int main() {
  auto s = std::make_unique<ae::StreamScratch>();
  auto take = [&](CUstream_st& st, size_t n) {
    uint8_t* p = nullptr;
    claim(s->take(&st, n, &p) == cudaSuccess && g_live.count(p), "a block is given, and it is allocated");
    for (size_t i = 0; i < n; ++i) p[i] = 1;
    return p;
  };
  auto capture = [](CUstream_st& st, unsigned long long id) {
    st.capture = id;
    st.graph = new CUgraph_st;
    g_capturing = true;
    return std::unique_ptr<CUgraph_st>(st.graph);
  };
  auto end = [](CUstream_st& st) { st.capture = 0, st.graph = nullptr, g_capturing = false; };

  CUstream_st a{1}, b{2};
  uint8_t* pa = take(a, 1000);
  claim(take(a, 400) == pa, "smaller calls on a stream share its block");
  claim(take(b, 1000) != pa, "streams have blocks of their own");
  auto g1 = capture(a, 10);
  uint8_t* p1 = take(a, 800);
  claim(p1 != pa && take(a, 100) == p1, "a graph has a block of its own, which its calls share");
  uint8_t* p1_large = take(a, 5000);
  claim(p1_large != p1 && g_live.count(p1), "a captured call that needs more leaves the block of the ones before alone");
  CUstream_st fork{3, 10, g1.get()};
  claim(take(fork, 100) != p1_large, "a stream forked into a capture has a block of its own");
  end(a), fork.capture = 0;
  claim(!g_unsafe && a.waits == 0, "a capture is not disturbed");

  take(a, 100000);  // grows: waits for the stream, frees its old block
  claim(a.waits == 1 && g_live.count(p1) && g_live.count(p1_large), "growth leaves the blocks of graphs alone");
  auto g2 = capture(a, 11);
  uint8_t* p2 = take(a, 800);
  claim(p2 != p1 && p2 != p1_large, "two graphs of one stream share no block");
  end(a);
  claim(s->release(&a) == cudaSuccess && a.waits == 2 && g_live.count(p1) && g_live.count(p1_large) && g_live.count(p2),
        "release leaves the blocks of graphs alone");
  size_t live = g_live.size();
  g1.reset();
  claim(g_live.size() == live, "nothing is freed where a graph goes");
  auto g3 = capture(a, 12);
  claim(take(a, 700) == p1, "the block of a graph that is gone serves another, the smallest that is large enough");
  end(a);
  claim(s->release(&b) == cudaSuccess && !g_live.count(p1_large) && g_live.count(p1), "release frees what no graph holds");

  CUstream_st c{4};  // a new stream at a destroyed one's address
  uint8_t* old = take(a, 100);
  a.id = 5;
  claim(take(a, 100) != old && take(c, 100) != old, "a stream whose handle comes back has a block of its own");

  auto g4 = capture(a, 13);
  uint8_t* p = nullptr;
  live = g_live.size();
  g_no_memory = true;
  claim(s->take(&a, 1 << 20, &p) == cudaErrorMemoryAllocation, "no memory is an error");
  g_no_memory = false, g_no_object = true;
  claim(s->take(&a, 1 << 20, &p) == cudaErrorMemoryAllocation, "no user object is an error");
  g_no_object = false;
  uint8_t* p4 = take(a, 1 << 20);
  claim(g_live.size() == live + 1 && p4 == p, "a block that no graph took serves the next call");
  end(a);
  claim(!g_unsafe && g_mode == cudaStreamCaptureModeGlobal, "the thread's capture mode is as it was");

  s->close();
  claim(g_live.empty(), "close frees everything");
  s.reset();
  g2.reset(), g3.reset(), g4.reset();  // graphs that outlive it
  return 0;
}
