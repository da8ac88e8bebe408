// The cluster-size rule of the few-rows tensor-core kernel with queries that fail: run by
// test_split_rule_cpu.py.  Prints what went wrong; exit status 0 when nothing did.
#include "split_rule.hpp"

#include <cstdio>
#include <thread>
#include <vector>

using namespace xvram::feed;

static int failures = 0;
#define CHECK(x)                                                                                   \
  do {                                                                                             \
    if (!(x)) {                                                                                    \
      std::printf("line %d: %s\n", __LINE__, #x);                                                  \
      ++failures;                                                                                  \
    }                                                                                              \
  } while (0)

int main() {
  { // a failed query is reported, not kept; an answer is, 0 included
    CapacityTable t;
    long long ctas = -1;
    int asked = 0;
    CHECK(t.ctas(0, 8, &ctas, [&](int*) { return ++asked, 700; }) == 700 && ctas == 0);
    CHECK(t.ctas(0, 8, &ctas, [&](int* c) { return ++asked, *c = 17, 0; }) == 0 && ctas == 136);
    CHECK(t.ctas(0, 8, &ctas, [&](int*) { return ++asked, 700; }) == 0 && ctas == 136);
    CHECK(asked == 2);
    CHECK(t.ctas(0, 4, &ctas, [&](int* c) { return ++asked, *c = 0, 0; }) == 0 && ctas == 0);
    CHECK(t.ctas(0, 4, &ctas, [&](int* c) { return ++asked, *c = 9, 0; }) == 0 && ctas == 0);
    CHECK(asked == 3);
    // sizes, devices and tables (kernels) are apart
    CHECK(t.ctas(0, 2, &ctas, [](int* c) { return *c = 70, 0; }) == 0 && ctas == 140);
    CHECK(t.ctas(63, 8, &ctas, [](int* c) { return *c = 3, 0; }) == 0 && ctas == 24);
    CHECK(t.ctas(64, 8, &ctas, [](int* c) { return *c = 3, 0; }) == 0 && ctas == 0);
    CapacityTable other;
    CHECK(other.ctas(0, 8, &ctas, [](int* c) { return *c = 5, 0; }) == 0 && ctas == 40);
    CHECK(t.ctas(0, 8, &ctas, [](int*) { return 1; }) == 0 && ctas == 136);
  }
  const auto all = [](int s, long long* c) { return *c = 144 / s * s, 0; };
  Split best;
  // a streamed A: one tile splits as far as it can, whole waves do not split
  CHECK(cheapest_split(1, 64, 148, 0, 0, all, &best) == 0 && best.splits == 8 && best.us > 0);
  CHECK(cheapest_split(148, 64, 148, 0, 0, all, &best) == 0 && best.splits == 1);
  // 2.5 + 3 x 0.45 = 3.85 alone against 2.5 + 2 x 0.45 + 1 = 4.4; 9.25 against 4.4 by 8
  CHECK(cheapest_split(1, 3, 148, 0, 0, all, &best) == 0 && best.splits == 1);
  CHECK(cheapest_split(1, 15, 148, 0, 0, all, &best) == 0 && best.splits == 8 && best.us < 5);
  // a held A needs the sizes under which it fits, and says when there is none
  CHECK(cheapest_split(100, 256, 148, 2048, 98304, all, &best) == 0 && best.splits == 8);
  const auto small = [](int s, long long* c) { return *c = s == 8 ? 0 : 144, 0; };
  CHECK(cheapest_split(100, 256, 148, 2048, 98304, small, &best) == 0 && best.splits == 0);
  // an error of the query is the rule's answer, and the next call may succeed
  const auto bad = [](int s, long long*) { return s == 8 ? 46 : 0; };
  CHECK(cheapest_split(100, 256, 148, 2048, 98304, bad, &best) == 46);
  CHECK(cheapest_split(100, 256, 148, 2048, 98304, all, &best) == 0 && best.splits == 8);
  // threads that ask at once agree
  CapacityTable shared;
  std::vector<std::thread> threads;
  std::atomic<int> wrong{0};
  for (int i = 0; i < 4; ++i)
    threads.emplace_back([&] {
      for (int k = 0; k < 1000; ++k) {
        long long ctas;
        if (shared.ctas(k % 64, 2, &ctas, [&](int* c) { return *c = k % 64, 0; }) || ctas != 2 * (k % 64))
          ++wrong;
      }
    });
  for (auto& th : threads)
    th.join();
  CHECK(wrong == 0);
  return failures != 0;
}
