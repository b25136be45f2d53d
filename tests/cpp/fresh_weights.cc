// What FreshWeights (csrc/fresh_weights.h) answers over sequences of calls; streams are made-up handles.
#include "fresh_weights.h"

#include <cstdio>
#include <cstdlib>

static int g_checks = 0;
#define CHECK(x) do { ++g_checks; if (!(x)) { printf("line %d: %s\n", __LINE__, #x); exit(1); } } while (0)

int main() {
  using kge::FreshWeights;
  const void *A = (void*)0x1000, *B = (void*)0x2000, *legacy = (void*)1, *own = (void*)2;
  auto no = [] { return false; };
  auto yes = [] { return true; };
  auto elsewhere = [](auto fn) { std::thread(fn).join(); };
  FreshWeights f;
  CHECK(!f.take(A, no));
  // a launch on another stream in between, the product by another thread
  f.written(A);
  CHECK(!f.take(B, no));
  elsewhere([&] { CHECK(f.take(A, no)); });
  CHECK(!f.take(A, no));
  // written twice, one ordinary launch is enough; two streams apart
  f.written(A);
  f.written(B);
  f.written(A);
  CHECK(f.take(A, no));
  CHECK(!f.take(A, no));
  CHECK(f.take(B, no));
  CHECK(!f.take(B, no));
  // products recorded into a graph are ordinary, and so is the first one after the recording
  f.written(A);
  CHECK(f.take(A, yes));
  CHECK(f.take(A, yes));
  CHECK(f.take(A, no));
  CHECK(!f.take(A, no));
  // the two names of the legacy stream; a stream for each thread
  f.written(nullptr);
  CHECK(f.take(legacy, no));
  f.written(own);
  elsewhere([&] { CHECK(!f.take(own, no)); f.written(own); CHECK(f.take(own, no)); });
  CHECK(f.take(own, no));
  CHECK(!f.take(own, no));
  // many threads, a stream each
  std::vector<std::thread> threads;
  std::atomic<int> wrong{0};
  for (int t = 0; t < 8; ++t)
    threads.emplace_back([&, t] {
      const void* s = (void*)(uintptr_t)(0x10000 + t * 64);
      for (int i = 0; i < 2000; ++i) {
        f.written(s);
        if (!f.take(s, no) || f.take(s, no)) ++wrong;
      }
    });
  for (auto& t : threads) t.join();
  CHECK(wrong == 0);
  printf("%d checks\n", g_checks);
}
