// Reports of given-up waits by stream: everyone concerned is told once, whoever asks first.
#include <cstdio>
#include <thread>

#include "../../nvmai_b200/csrc/give_ups.h"

int main() {
    int bad = 0;
    auto expect = [&](const char *what, bool ok) { if (!ok) { std::printf("%s\n", what); ++bad; } };
    const void *a = reinterpret_cast<void *>(0x100), *b = reinterpret_cast<void *>(0x200), *c = reinterpret_cast<void *>(0x300);
    const void *legacy = nullptr, *own = reinterpret_cast<void *>(2);
    nvmai::GiveUps g;
    g.product(0, a);
    g.product(0, b);
    g.product(0, legacy);
    expect("nothing yet", !g.news(0, a, 0) && !g.news(0, b, 0));
    // a product on b gives up; a asks first
    expect("a is told", g.news(0, a, 1));
    expect("b still is", g.news(0, b, 1));
    expect("the legacy stream too", g.news(0, legacy, 1));
    expect("each of them once", !g.news(0, a, 1) && !g.news(0, b, 1) && !g.news(0, legacy, 1));
    // one that is given up between reading and answering is in the next answer
    expect("the second one", g.news(0, a, 2) && g.news(0, a, 3) && !g.news(0, a, 3) && g.news(0, b, 3));
    // a stream whose first product comes after a report does not hear of it, but of what comes then
    g.product(0, c);
    expect("old ones are not news for a new stream", !g.news(0, c, 3));
    g.product(0, c);
    expect("later ones are", g.news(0, c, 4));
    // ... and hears of one that nobody had read when its first product came
    const void *d = reinterpret_cast<void *>(0x400);
    g.product(0, d);                    // the last count read is 4; 5 is given up now, by d or by another
    expect("read by another one first", g.news(0, a, 5));
    expect("and still news here", g.news(0, d, 5));
    // without products: all there have been
    expect("a stream that only replays", g.news(0, reinterpret_cast<void *>(0x500), 5));
    // devices count for themselves
    g.product(1, a);
    expect("another device", !g.news(1, a, 0) && g.news(1, a, 1) && !g.news(0, a, 5));
    // the per-thread stream is another one in each thread
    g.product(0, own);
    std::thread([&] { g.product(0, own); expect("the thread's own", g.news(0, own, 6) && !g.news(0, own, 6)); }).join();
    expect("and this one's", g.news(0, own, 6));
    // another registry is not taken for this one
    nvmai::GiveUps h;
    h.product(0, own);
    expect("a registry of its own", !h.news(0, own, 0));
    // the count comes round
    expect("past the last count", g.news(0, a, 0xFFFFFFFFu) && g.news(0, a, 0));
    std::printf(bad ? "FAILED %d\n" : "PASSED\n", bad);
    return bad != 0;
}
