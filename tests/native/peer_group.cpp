// TEST INFRASTRUCTURE ONLY: mml::PeerGroup's host barriers without a device (tests/test_peer_group.py
// builds and runs it against libmml_hip.so).  Prints one line per check; exit status 0 when all hold.
#include <atomic>
#include <chrono>
#include <cstdio>
#include <string>
#include <thread>
#include <vector>

#include "mml_internal.h"

namespace {
int failures = 0;
void check(bool ok, const char* what) {
    std::printf("%s: %s\n", ok ? "ok" : "FAILED", what);
    failures += !ok;
}
std::string thrown(mml::PeerGroup& g) {
    try {
        g.barrier();
    } catch (const std::exception& e) {
        return e.what();
    }
    return "";
}
}  // namespace

int main() {
    {  // every rank passes every barrier together
        constexpr int kRanks = 8, kTurns = 3000;
        mml::PeerGroup g(kRanks);
        std::atomic<int> before[kTurns]{};
        std::atomic<int> early{0};
        std::vector<std::thread> th;
        for (int r = 0; r < kRanks; ++r)
            th.emplace_back([&] {
                for (int t = 0; t < kTurns; ++t) {
                    ++before[t];
                    g.barrier();
                    early += before[t] != kRanks;
                }
            });
        for (auto& t : th) t.join();
        check(early == 0, "no rank leaves a barrier before all have come");
    }
    {  // a rank that fails releases the others; the group works again after a reset
        mml::PeerGroup g(3);
        std::string said[2];
        std::thread a([&] { said[0] = thrown(g); }), b([&] { said[1] = thrown(g); });
        std::this_thread::sleep_for(std::chrono::milliseconds(20));
        g.abort();
        a.join();
        b.join();
        check(said[0].find("failed") != said[0].npos && said[1].find("failed") != said[1].npos,
              "a failing rank releases the others");
        check(thrown(g).find("failed") != std::string::npos, "and whoever comes later");
        g.reset();
        std::string after[3];
        std::vector<std::thread> th;
        for (int r = 0; r < 3; ++r) th.emplace_back([&, r] { after[r] = thrown(g); });
        for (auto& t : th) t.join();
        check(after[0].empty() && after[1].empty() && after[2].empty(), "after a reset all pass");
    }
    {  // a rank that never comes: the others leave when the limit is over
        mml::PeerGroup g(3);
        g.limit_s = 0.2;
        std::string said[2];
        const auto t0 = std::chrono::steady_clock::now();
        std::thread a([&] { said[0] = thrown(g); }), b([&] { said[1] = thrown(g); });
        a.join();
        b.join();
        const double s = std::chrono::duration<double>(std::chrono::steady_clock::now() - t0).count();
        check(!said[0].empty() && !said[1].empty() && s >= 0.2, "a rank that never comes is not waited for");
        check((said[0] + said[1]).find("did not come") != std::string::npos, "with the reason");
        check(thrown(g).find("failed") != std::string::npos, "and is told when it comes late");
    }
    return failures != 0;
}
