// CPU test of the workspace blocks that belong to one captured graph
// (orator_amd/csrc/workspace_pool.hpp, WsKey::capture): two captures on one stream never share a
// block with each other or with the stream's eager calls; the calls of one capture do; a block is
// kept until the stream is released, also when its thread ends first.
#include <cstdio>
#include <cstdlib>
#include <set>
#include <thread>

#include "../../orator_amd/csrc/workspace_pool.hpp"

using orator_hip::WorkspacePool;
using orator_hip::WsKey;

static std::set<void*> g_live;
static int alloc(void** p, size_t n) {
  *p = std::malloc(n);
  g_live.insert(*p);
  return 0;
}
static void release(void* p) {
  g_live.erase(p);
  std::free(p);
}
static int sync(const void*) { return 0; }
static void* record(int, const void*) { return std::malloc(1); }
static int done(void*) { return 1; }
static void destroy(void* e) { std::free(e); }

#define REQUIRE(c)                                       \
  do {                                                   \
    if (!(c)) {                                          \
      std::fprintf(stderr, "line %d: %s\n", __LINE__, #c); \
      return 1;                                          \
    }                                                    \
  } while (0)

int main() {
  WorkspacePool pool(alloc, release, sync, record, done, destroy);
  int s = 0, other = 0;
  const auto me = std::this_thread::get_id();
  std::string err;
  auto get = [&](const void* stream, unsigned long long capture, size_t n, bool* fresh = nullptr) {
    return pool.get(WsKey{0, stream, me, 6, capture}, n, capture != 0, &err, fresh);
  };
  bool fresh = false;
  void* eager = get(&s, 0, 1000);
  void* a = get(&s, 1, 1000, &fresh);
  REQUIRE(fresh);
  REQUIRE(get(&s, 1, 900, &fresh) == a && !fresh);
  void* b = get(&s, 2, 1000);
  void* c = get(&other, 1, 1000);
  REQUIRE(eager != a && eager != b && a != b && c != a && c != b && c != eager);
  // a capture that needs more gets another block; the first stays for its earlier nodes
  void* a2 = get(&s, 1, 1 << 20, &fresh);
  REQUIRE(fresh && a2 != a && g_live.count(a));
  for (int i = 0; i < 50; ++i) REQUIRE(get(&s, 0, 1000) == eager);
  REQUIRE(g_live.count(a) && g_live.count(a2) && g_live.count(b) && g_live.count(c));
  std::thread t([&] {
    std::string e;
    const auto id = std::this_thread::get_id();
    (void)pool.get(WsKey{0, &s, id, 6, 9}, 1000, true, &e);
    pool.thread_exit(id);
  });
  t.join();
  pool.reap();
  REQUIRE(g_live.size() == 6);
  REQUIRE(pool.release_stream(0, &s) == 0);
  REQUIRE(g_live.size() == 1 && g_live.count(c));
  REQUIRE(pool.release_stream(0, &other) == 0);
  REQUIRE(g_live.empty() && pool.entries() == 0);
  std::printf("workspace capture OK\n");
  return 0;
}
