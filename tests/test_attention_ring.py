"""The protocol of the tile kernel's ring of K and V steps (``rllama_b200/csrc/attention_long_ring.h``), on the host: a C++ program walks its roles (the fillers, the issuers of the
score and output products of one or two tiles, the softmax) over model barriers in random interleavings, with copies and products that complete whenever they like. A wait that returns
before its item is there, a stage that is filled before it is used up, and a standstill are errors. No GPU needed."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <deque>
#include <functional>
#include <random>
#include <vector>
#include "attention_long_ring.h"
using namespace attn_long;

struct Bar {
    int expected = 1, pending = 1, phase = 0;
    void init(int n) { expected = pending = n; phase = 0; }
    void arrive() { if (--pending == 0) { pending = expected; phase++; } }
    bool done(uint32_t parity) const { return (uint32_t)(phase & 1) != parity; }   // as mbarrier.try_wait.parity
};
struct Op { std::function<bool()> ready; std::function<void()> act; };
struct Role { std::vector<Op> ops; size_t at = 0; };

static const char* g_error = nullptr;
static void fail(const char* what) { if (!g_error) g_error = what; }

template <class Ring> int simulate(int n, int tiles, bool one_filler, const std::vector<std::vector<bool>>& any, std::mt19937& rng) {
    std::vector<Bar> full(Ring::STAGES), empty(Ring::STAGES), s_full(tiles), s_read(tiles), p_ready(2 * tiles), pv_done(2 * tiles);
    const int fillers = one_filler ? 1 : 4;
    for (auto& b : full) b.init(fillers);
    for (auto& b : empty) b.init(tiles);
    struct Stage { int item = -1; bool v = false; int filled = 0, used = 0; };
    std::vector<Stage> stage(Ring::STAGES);
    std::vector<std::deque<std::function<void()>>> later;   // queues of things that complete in order, each whenever it likes
    auto queue = [&](std::deque<std::function<void()>> q) { later.push_back(std::move(q)); };
    std::vector<Role> roles;
    const std::function<bool()> now = [] { return true; };

    auto begin = [&](bool v, int i) {   // the first filler's part of an item
        Stage& s = stage[Ring::at(v, i).stage];
        if (s.item >= 0 && s.used < tiles) fail("a stage was filled before it was used up");
        s = Stage{i, v, 0, 0};
    };
    if (one_filler) {   // copies complete in any order
        Role r;
        auto load = [&, fillers](bool v, int i) {
            return [&, v, i] { begin(v, i); queue({[&, v, i] { const int s = Ring::at(v, i).stage; stage[s].filled = 1; full[s].arrive(); }}); };
        };
        int k = 0, v = 0;
        const int mk = std::min(n, Ring::K), mv = std::min(n, Ring::V);
        while (k < mk || v < mv) {
            const bool is_v = v < mv && (k == mk || Ring::next_is_v(k, v, n));
            r.ops.push_back({now, load(is_v, is_v ? v : k)});
            (is_v ? v : k)++;
        }
        while (k < n || v < n) {
            const bool is_v = Ring::next_is_v(k, v, n);
            const auto slot = Ring::at(is_v, is_v ? v : k);
            if (!slot.used) fail("a first item waits");
            r.ops.push_back({[&, slot] { return empty[slot.stage].done(slot.parity ^ 1); }, load(is_v, is_v ? v : k)});
            (is_v ? v : k)++;
        }
        roles.push_back(r);
    } else {
        for (int w = 0; w < 2 * fillers; w++) {
            Role r;
            const bool v = w >= fillers;
            for (int i = 0; i < n; i++) {
                const auto slot = Ring::at(v, i);
                r.ops.push_back({[&, slot] { return !slot.used || empty[slot.stage].done(slot.parity ^ 1); },
                                 [&, v, i, slot] { if (stage[slot.stage].item != i || stage[slot.stage].v != v) begin(v, i); }});
                r.ops.push_back({now, [&, v, i, slot, fillers] { Stage& s = stage[slot.stage]; if (s.item != i || s.v != v) fail("a filler writes to another item"); s.filled += 1; full[slot.stage].arrive(); }});
            }
            roles.push_back(r);
        }
    }
    auto use = [&, fillers](bool v, int i) {
        const Stage& s = stage[Ring::at(v, i).stage];
        if (s.item != i || s.v != v || s.filled < fillers) fail("a step was used before it was there");
    };
    // a warp's products complete in order
    std::vector<std::deque<std::function<void()>>> issued(2 * tiles);
    for (int t = 0; t < tiles; t++) {
        Role s, p, m;
        int done = 0;
        for (int i = 0; i < n; i++) {
            const auto k = Ring::at(false, i), v = Ring::at(true, i);
            s.ops.push_back({[&, k] { return full[k.stage].done(k.parity); }, [&, i] { use(false, i); }});
            p.ops.push_back({[&, v] { return full[v.stage].done(v.parity); }, [&, i] { use(true, i); }});
            if (any[t][i]) {
                const int buf = done & 1;
                if (done > 0) s.ops.push_back({[&, t, done] { return s_read[t].done((done - 1) & 1); }, [] {}});
                p.ops.push_back({[&, t, buf, done] { return p_ready[2 * t + buf].done((done >> 1) & 1); }, [] {}});
                s.ops.push_back({now, [&, t, i] { issued[2 * t].push_back([&, t, i] { use(false, i); s_full[t].arrive(); }); }});
                p.ops.push_back({now, [&, t, i, buf] { issued[2 * t + 1].push_back([&, t, i, buf] { use(true, i); pv_done[2 * t + buf].arrive(); }); }});
                m.ops.push_back({[&, t, done] { return s_full[t].done(done & 1); }, [] {}});
                m.ops.push_back({now, [&, t] { s_read[t].arrive(); }});
                if (done >= 2) m.ops.push_back({[&, t, buf, done] { return pv_done[2 * t + buf].done(((done - 2) >> 1) & 1); }, [] {}});
                m.ops.push_back({now, [&, t, buf] { p_ready[2 * t + buf].arrive(); }});
                done++;
            }
            s.ops.push_back({now, [&, t, k] { issued[2 * t].push_back([&, k] { stage[k.stage].used++; empty[k.stage].arrive(); }); }});
            p.ops.push_back({now, [&, t, v] { issued[2 * t + 1].push_back([&, v] { stage[v.stage].used++; empty[v.stage].arrive(); }); }});
        }
        roles.push_back(s); roles.push_back(p); roles.push_back(m);
    }
    // some roles are much slower than others
    std::vector<double> speed;
    for (size_t i = 0; i < roles.size() + issued.size() + 1; i++) speed.push_back(rng() % 4 == 0 ? 0.02 : 1.0);
    std::uniform_real_distribution<double> u(0, 1);
    for (long idle = 0; !g_error;) {
        bool moved = false, left = false;
        for (size_t i = 0; i < roles.size(); i++) {
            Role& r = roles[i];
            if (r.at == r.ops.size()) continue;
            left = true;
            if (u(rng) > speed[i] || !r.ops[r.at].ready()) continue;
            r.ops[r.at++].act();
            moved = true;
        }
        for (size_t i = 0; i < issued.size(); i++)
            if (!issued[i].empty()) {
                left = true;
                if (u(rng) > 0.5 * speed[roles.size() + i]) continue;
                auto f = issued[i].front(); issued[i].pop_front(); f();
                moved = true;
            }
        for (size_t i = 0; i < later.size();)
            if (left = true, u(rng) < 0.3 * speed.back()) {
                auto f = later[i].front(); later.erase(later.begin() + i); f();
                moved = true;
            } else i++;
        if (!left) break;
        idle = moved ? 0 : idle + 1;
        if (idle > 20000) fail("nothing moves any more");
    }
    return g_error ? 1 : 0;
}

template <class Ring> int runs(const char* name, int tiles, bool one_filler, int seeds) {
    for (int seed = 0; seed < seeds; seed++) {
        std::mt19937 rng(seed);
        const int n = rng() % 30;
        std::vector<std::vector<bool>> any(tiles, std::vector<bool>(n, true));
        if (tiles == 2) {   // the second tile has no rows; or the first one ends earlier and the second one begins later
            if (rng() % 3 == 0) any[1].assign(n, false);
            else for (int t = 0; t < 2; t++) for (int i = 0, m = rng() % 4; i < m && i < n; i++) any[t][t ? i : n - 1 - i] = false;
        }
        if (simulate<Ring>(n, tiles, one_filler, any, rng)) { printf("%s, %d steps, seed %d: %s\n", name, n, seed, g_error); return 1; }
    }
    return 0;
}
"""
MAIN = """
int main() {
    return runs<KvRing<2, 2>>("2+2", 1, true, 800) | runs<KvRing<4, 4>>("4+4", 1, true, 400) | runs<KvRing<2, 1>>("2+1", 1, true, 800) | runs<KvRing<1, 2>>("1+2", 1, true, 800) |
           runs<KvRing<4, 4>>("4+4", 2, false, 400) | runs<KvRing<8, 8>>("8+8", 2, false, 300) | runs<KvRing<3, 3>>("3+3", 2, false, 800) | runs<KvRing<2, 2>>("2+2", 2, false, 800);
}
"""
# one ring for both kinds, K0 K1 V0 K2 V1 ...
SHARED = """
template <int N> struct Shared {
    static constexpr int K = N, V = N, STAGES = N;
    struct Slot { uint32_t stage, parity; bool used; };
    static int n;
    static bool next_is_v(int, int, int) { return false; }   // (its fillers are the eight warps)
    static Slot at(bool v, uint32_t i) {
        const uint32_t x = !v ? (i == 0 ? 0 : 2 * i - 1) : (int)i == n - 1 ? 2 * i + 1 : 2 * i + 2;
        return {x % N, x / N & 1, x >= (uint32_t)N};
    }
};
template <int N> int Shared<N>::n = 0;
int main() {
    for (int seed = 0; seed < 4000; seed++) {
        std::mt19937 rng(seed);
        const int n = 8 + rng() % 20;
        Shared<8>::n = n;
        std::vector<std::vector<bool>> any(2, std::vector<bool>(n, true));
        any[1].assign(n, false);
        if (simulate<Shared<8>>(n, 2, false, any, rng)) { printf("%s\\n", g_error); return 1; }
    }
}
"""


def run(tmp_path, main):
    (tmp_path / "ring.cpp").write_text(PROGRAM + main)
    exe = str(tmp_path / "ring")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-I" + os.path.join(ROOT, "rllama_b200", "csrc"), str(tmp_path / "ring.cpp"), "-o", exe], check=True)
    return subprocess.run([exe], capture_output=True, text=True, timeout=300)


def test_the_ring_keeps_its_order(tmp_path):
    r = run(tmp_path, MAIN)
    assert r.returncode == 0, r.stdout


def test_the_model_finds_what_stages_for_both_kinds_would_miss(tmp_path):
    """The issuer of a tile without rows waits for the last V step on a stage whose K steps it has not followed."""
    r = run(tmp_path, SHARED)
    assert r.returncode == 1 and "before it was there" in r.stdout
