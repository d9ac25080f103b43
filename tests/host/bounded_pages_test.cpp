/* PagePool::trim and drop (include/battn_sched.h): the pages of bounded rows go back to the pool. */
#include <cstdio>
#include <cstdlib>

#include "battn_sched.h"

using battn_sched::PagePool;

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

int main() {
    PagePool p(16, 128, 3, 8);
    CHECK(p.reserve(0, 1000));                        /* 8 pages */
    CHECK(p.free_pages() == 8);
    p.take_dirty(0);
    /* an eviction to 300 positions keeps three pages; nothing happens when the row is short already */
    p.trim(0, 300);
    CHECK(p.pages_of(0) == 3 && p.free_pages() == 13 && p.row(0)[2] >= 0 && p.row(0)[3] == -1 && p.take_dirty(0));
    p.trim(0, 300);
    p.trim(0, 900);
    CHECK(p.pages_of(0) == 3 && !p.take_dirty(0));
    p.trim(0, 0);
    CHECK(p.pages_of(0) == 0 && p.free_pages() == 16);
    /* a shared prefix page stays with its other row */
    CHECK(p.reserve(0, 256) && p.share_prefix(0, 1, 256) == 256 && p.reserve(1, 500));
    const int shared = p.row(0)[1];
    p.trim(1, 100);
    CHECK(p.pages_of(1) == 1 && p.refcount(shared) == 1 && p.refcount(p.row(0)[0]) == 2);
    p.release(0);
    p.release(1);
    CHECK(p.free_pages() == 16);
    /* a stream with 4 sinks and a window of 256 that stands at position 900 sees [0, 4) and [645, 900]: pages 1 .. 4 go */
    CHECK(p.reserve(0, 901));
    p.take_dirty(0);
    p.drop(0, 4, 901 - 256);
    CHECK(p.free_pages() == 12 && p.row(0)[0] >= 0 && p.row(0)[5] >= 0 && p.take_dirty(0));
    for (int i = 1; i < 5; ++i) CHECK(p.row(0)[i] == -1);
    p.drop(0, 4, 901 - 256);                          /* again: nothing left to drop */
    CHECK(p.free_pages() == 12 && !p.take_dirty(0));
    p.drop(0, 130, 200);                              /* no whole page inside */
    p.drop(0, -5, 0);
    CHECK(p.free_pages() == 12);
    CHECK(p.share_prefix(0, 2, 900) == 128);          /* up to the first hole */
    int from, to;
    CHECK(!p.make_writable(0, 200, &from, &to) && from == -1 && to == -1);
    CHECK(p.reserve(0, 1024) && p.free_pages() == 12);
    p.release(0);
    p.release(2);
    CHECK(p.free_pages() == 16);
    std::printf("OK\n");
    return 0;
}
