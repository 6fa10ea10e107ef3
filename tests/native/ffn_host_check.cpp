// Host build of the feed-forward operators' bookkeeping (tt_lazy_b200/csrc/ffn.cuh):
// prints a line "name=ok" for each part that behaves, exits 1 at the first that does not.
#include <cstdio>
#include <cstdlib>

#include "ffn.cuh"

static void expect(bool ok, const char* what) {
    if (ok) return;
    std::printf("failed: %s\n", what);
    std::exit(1);
}

static void copies_in_flight() {
    ttc::CopiesInFlight c;
    c.sent(0);
    c.sent(1);
    expect(c.on_its_way(0) && c.on_its_way(1) && c.parity(0) == 0 && c.parity(1) == 0, "two copies sent");
    expect(c.waited(0, true) && !c.on_its_way(0) && c.parity(0) == 1, "a copy that landed: its barrier's next phase");
    expect(c.on_its_way(1) && c.parity(1) == 0, "the other buffer is not touched");
    expect(!c.waited(1, false), "a wait that ran out says so");
    expect(c.on_its_way(1) && c.parity(1) == 0, "its copy is still on its way, in the same phase");
    expect(c.waited(1, true) && !c.on_its_way(1) && c.parity(1) == 1, "and is over once it has landed");
    std::printf("copies_in_flight=ok\n");
}

static void set_up_once() {
    ttc::OncePerDevice once;
    int calls = 0, answer = TTC_ERR_CUDA;
    auto prepare = [&] {
        ++calls;
        return answer;
    };
    expect(once(1, prepare) == TTC_ERR_CUDA && calls == 1, "a set-up that fails says so");
    answer = TTC_OK;
    expect(once(1, prepare) == TTC_OK && calls == 2, "and is tried again by the next call");
    expect(once(1, prepare) == TTC_OK && calls == 2, "one that succeeded is not");
    expect(once(0, prepare) == TTC_OK && calls == 3, "each device has its own");
    std::printf("set_up_once=ok\n");
}

int main() {
    copies_in_flight();
    set_up_once();
    return 0;
}
