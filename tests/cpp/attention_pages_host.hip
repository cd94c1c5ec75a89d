// Runs on the host what the kernels of attention over pages and their launches compute of positions and sizes.
// Reads a question a line from stdin, answers each with a line:
//   divide D N                               N / D as the kernels divide
//   window FRAME AHEAD BACK SINKS P N        what position P sees of N keys: sink lo hi of Window::at, then of span_of
#include <cstdio>
#include <cstring>

#include "dcn_attention_pages.hpp"

int main() {
    using namespace dcn;
    char what[16];
    while (std::scanf("%15s", what) == 1) {
        long long x[8] = {};
        const auto read = [&](int n) {
            for (int i = 0; i < n; ++i)
                if (std::scanf("%lld", &x[i]) != 1) return false;
            return true;
        };
        if (!std::strcmp(what, "divide") && read(2)) {
            std::printf("%d\n", fa::divide_by((int)x[0])((int)x[1]));
        } else if (!std::strcmp(what, "window") && read(6)) {
            AttentionArgs a{};
            a.frame = (int)x[0];
            a.ahead = (int)x[1];
            a.back = (int)x[2];
            a.sinks = (int)x[3];
            const fa::Span s = fa::window_of(a).at((int)x[4], (int)x[5]), t = fa::span_of(a, (int)x[4], (int)x[5]);
            std::printf("%d %d %d %d %d %d\n", s.sink, s.lo, s.hi, t.sink, t.lo, t.hi);
        } else {
            return 2;
        }
    }
    return 0;
}
