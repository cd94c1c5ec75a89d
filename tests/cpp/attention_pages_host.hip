// Runs on the host what the kernels of attention over pages and their launches compute of positions and sizes.
// Reads a question a line from stdin, answers each with a line:
//   divide D N                               N / D as the kernels divide
//   window FRAME AHEAD BACK SINKS P N        what position P sees of N keys: sink lo hi of Window::at, then of span_of
//   plan DIM BITS SEQUENCES KV_HEADS GROUP Q_TOKENS MAX_Q MAX_KV MAX_PREFIX FRAME BACK SINKS
//                                            shared both parts; rows waves blocks splits of own; of the prefix;
//                                            workgroups of the prefix, own; whether the launches fit
//   meet IN_AT TS HS HEADS OUT_AT TS HS HEADS TOKENS DIM SIZE
//                                            whether rows of an output lie on those of an input (places in bytes)
#include <cstdio>
#include <cstring>

#include "dcn_attention_host.hpp"
#include "dcn_attention_pages.hpp"
#include "dcn_attention_plan.hpp"

int main() {
    using namespace dcn;
    char what[16];
    while (std::scanf("%15s", what) == 1) {
        long long x[12] = {};
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
        } else if (!std::strcmp(what, "plan") && read(12)) {
            const fa::PlanOf p = fa::plan_of((int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)x[4], x[5], (int)x[6], (int)x[7], (int)x[8], (int)x[9],
                                             (int)x[10], (int)x[11]);
            fa::PagesGrid own{}, prefix{};
            const bool grids = fa::pages_grid(p.own.blocks, p.own.splits, p.own.per, (int)x[3], x[2], &own) &&
                               (!p.shared || fa::pages_grid(p.prefix.blocks, p.prefix.splits, p.prefix.per, (int)x[3], 1, &prefix));
            std::printf("%d %d %d %d %d %d %d %d %d %d %d %u %u %d\n", p.shared, p.both, p.parts, p.own.rows, p.own.waves, p.own.blocks, p.own.splits,
                        p.prefix.rows, p.prefix.waves, p.prefix.blocks, p.prefix.splits, prefix.grid, own.grid,
                        grids && fa::launches_fit(p, prefix.grid, own.grid, x[6] * x[3] * x[4]));
        } else if (!std::strcmp(what, "meet") && read(11)) {
            const int64_t in[2] = {x[1], x[2]}, out[2] = {x[5], x[6]};
            std::printf("%d\n", host::rows_meet((const void*)x[0], in, (int)x[3], (const void*)x[4], out, (int)x[7], x[8], (int)x[9], (int)x[10]));
        } else {
            return 2;
        }
    }
    return 0;
}
