"""How the CTAs of a cluster exchange a value per row and leave (csrc/row_exchange.hpp), compiled for the host: every thread of every CTA as a fiber, run
in random order; stores that land late, CTAs that stand still for longer than a wait lasts, copies that never come.  No wait is made to run out on a GPU."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama.cu_b200", "csrc")

MAIN = r"""
#include <ucontext.h>
#include <cstdio>
#include <cstdlib>
#include <memory>
#include <random>
#include <vector>
#include "row_exchange.hpp"

// Mistakes that the simulation has to find: exchanges go on behind one that failed, and CTAs leave at once.
struct LeavesAtOnce : lcu::RowExchange {
    template <class Port> void leave(Port &port) { port.together(); }
};
struct SendsOn : lcu::RowExchange {
    template <class Port> bool exchange(Port &port) {
        if (row == 0) port.started();
        port.send(turn());
        if (port.wait(turn(), parity())) return true;
        port.give_up();
        return false;
    }
};
struct Careless : SendsOn {
    template <class Port> void leave(Port &port) { port.together(); }
};

constexpr int LATENCY = 25;
int polls = 40;

struct Sim {
    struct Bar { int pending = 1, tx = 0; unsigned phase = 0; void settle() { if (!pending && !tx) { pending = 1; ++phase; } } };
    struct Cta {
        int slot[2][8];
        Bar bar[2];
        bool flag = false;
        int arrived = 0, exited = 0;   // at the CTA's barrier, in all
        unsigned generation = 0;
        long still_from = -1, still_to = -1;
    };
    struct Store { long at; int to, turn, from, row; };
    struct Fiber { ucontext_t ctx; std::unique_ptr<char[]> stack; int cta, thread, cluster_phase = 0; bool done = false; };
    std::mt19937 rng;
    int size, threads, rows;
    long step = 0, limit = 3000000;
    std::vector<Cta> cta;
    std::vector<Store> flying;
    std::vector<std::unique_ptr<Fiber>> fibers;
    ucontext_t home;
    Fiber *now = nullptr;
    long left = 0, foreign = 0, failed = 0, done_rows = 0;  // stores to a CTA that has left; rows read with another row's value

    int below(int n) { return (int)(rng() % (unsigned)n); }
    void yield() { swapcontext(&now->ctx, &home); }
    bool gone(int c) { return cta[c].exited == threads; }
    void land() {
        for (size_t i = 0; i < flying.size();) {
            if (flying[i].at > step) { ++i; continue; }
            Store s = flying[i];
            flying[i] = flying.back();
            flying.pop_back();
            if (gone(s.to)) { ++left; continue; }
            cta[s.to].slot[s.turn][s.from] = s.row;
            cta[s.to].bar[s.turn].tx -= 8;
            cta[s.to].bar[s.turn].settle();
        }
    }
    bool all_in(int phase) {
        for (auto &f : fibers)
            if (!f->done && f->cluster_phase < phase) return false;
        return true;
    }
};

struct Port {
    Sim &s;
    int c, t, row;
    void started() { while (!s.all_in(1)) s.yield(); }
    void send(uint32_t turn) {
        s.yield();
        Sim::Bar &b = s.cta[c].bar[turn];
        if (t == 0) { --b.pending; b.tx += 8 * s.size; b.settle(); }
        s.yield();
        if (t < s.size) {
            if (s.gone(t)) ++s.left;
            s.flying.push_back({s.step + 1 + s.below(LATENCY), t, (int)turn, c, row});
        }
    }
    bool wait(uint32_t turn, uint32_t parity) {
        for (int i = 0; i < polls; ++i) {
            s.yield();
            if ((s.cta[c].bar[turn].phase & 1u) != parity) return true;
            if (i % 8 == 7 && s.cta[c].flag) return false;
        }
        return false;
    }
    bool gave_up() { s.yield(); return s.cta[c].flag; }
    void give_up() { s.cta[c].flag = true; }
    void together() {
        Sim::Cta &x = s.cta[c];
        const unsigned g = x.generation;
        if (++x.arrived == s.threads) { x.arrived = 0; ++x.generation; }
        while (x.generation == g) s.yield();
    }
    void others() { s.now->cluster_phase = 2; while (!s.all_in(2)) s.yield(); }
    void landed() { for (const long t0 = s.step; s.step < t0 + 2 * LATENCY;) s.yield(); }
};

template <class Exchange> struct Run {
    static Sim *sim;
    static int lost_cta, lost_row, lost_thread;
    static void body() {
        Sim &s = *sim;
        Sim::Fiber *me = s.now;
        Port port{s, me->cta, me->thread, 0};
        me->cluster_phase = 1;
        Exchange ex;
        bool had_failed = false;
        for (int r = 0; r < s.rows; ++r, ex.next_row()) {
            if (me->cta == lost_cta && r == lost_row && me->thread == lost_thread) port.give_up();  // its copy of the row never came
            port.together();
            port.row = r;
            const bool ok = ex.exchange(port);
            if (ok && had_failed) ++s.foreign;  // (nothing was sent for it)
            if (ok) {
                bool own = true;
                for (int c = 0; c < s.size; ++c) {
                    s.yield();
                    own = own && s.cta[me->cta].slot[ex.turn()][c] == r;
                }
                if (!own) ++s.foreign;
                ++s.done_rows;
            } else {
                ++s.failed;
                had_failed = true;
            }
        }
        ex.leave(port);
        me->done = true;
        ++s.cta[me->cta].exited;
        s.yield();
    }
    // kind 0: everyone in time; 1: CTAs stand still for a while; 2: and a copy never comes
    static void once(unsigned seed, int kind, long *total) {
        const auto own = std::make_unique<Sim>();
        Sim &s = *own;
        s.rng.seed(seed);
        s.size = 1 << s.below(4);
        if (s.size == 8) s.size = 4;
        s.threads = s.size + 1;
        s.rows = 1 + s.below(7);
        s.cta.resize(s.size);
        for (auto &c : s.cta) {
            for (auto &turn : c.slot) for (int &x : turn) x = -1;
            if (kind && s.below(2)) {
                c.still_from = s.below(60 * s.size * s.rows + 200);
                c.still_to = c.still_from + (1L << s.below(16));
            }
        }
        lost_cta = kind == 2 ? s.below(s.size) : -1;
        lost_row = s.below(s.rows);
        lost_thread = s.below(s.threads);
        sim = &s;
        polls = kind ? 40 : 100000;
        for (int c = 0; c < s.size; ++c)
            for (int t = 0; t < s.threads; ++t) {
                auto f = std::make_unique<Sim::Fiber>();
                f->cta = c;
                f->thread = t;
                f->stack.reset(new char[65536]);
                getcontext(&f->ctx);
                f->ctx.uc_stack.ss_sp = f->stack.get();
                f->ctx.uc_stack.ss_size = 65536;
                f->ctx.uc_link = &s.home;
                makecontext(&f->ctx, body, 0);
                s.fibers.push_back(std::move(f));
            }
        int open = (int)s.fibers.size();
        while (open && s.step < s.limit) {
            ++s.step;
            s.land();
            Sim::Fiber *f = s.fibers[s.below((int)s.fibers.size())].get();
            const Sim::Cta &c = s.cta[f->cta];
            if (f->done || (s.step >= c.still_from && s.step < c.still_to)) continue;
            s.now = f;
            swapcontext(&s.home, &f->ctx);
            if (f->done) --open;
        }
        for (; !s.flying.empty(); ++s.step) s.land();
        const long found[5] = {s.left, s.foreign, s.failed, s.done_rows, open};
        for (int i = 0; i < 5; ++i) total[i] += found[i];
    }
};
template <class E> Sim *Run<E>::sim;
template <class E> int Run<E>::lost_cta;
template <class E> int Run<E>::lost_row;
template <class E> int Run<E>::lost_thread;

int main(int argc, char **argv) {
    const int which = atoi(argv[1]), kind = atoi(argv[2]), runs = atoi(argv[3]);
    long total[5] = {};
    for (int i = 0; i < runs; ++i) {
        if (which == 0) Run<lcu::RowExchange>::once(i, kind, total);
        if (which == 1) Run<Careless>::once(i, kind, total);
        if (which == 2) Run<LeavesAtOnce>::once(i, kind, total);
        if (which == 3) Run<SendsOn>::once(i, kind, total);
    }
    printf("%ld %ld %ld %ld %ld\n", total[0], total[1], total[2], total[3], total[4]);
}
"""


@pytest.fixture(scope="module")
def simulate(tmp_path_factory):
    d = tmp_path_factory.mktemp("exchange")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(d / "main.cpp"), "-o", str(d / "main")], check=True)

    def run(which, kind, runs=1500):
        """Stores to CTAs that have left, rows read with values of other rows, threads' rows that failed and that came, threads that never ended."""
        out = subprocess.run([str(d / "main"), str(which), str(kind), str(runs)], capture_output=True, text=True, check=True, timeout=120).stdout
        return list(map(int, out.split()))
    return run


def test_everyone_in_time(simulate):
    left, foreign, failed, came, open_ = simulate(0, 0)
    assert left == foreign == failed == open_ == 0 and came > 10000


@pytest.mark.parametrize("kind", [1, 2])
def test_late_and_missing_peers(simulate, kind):
    """Rows come whole or fail; nobody is sent anything behind its end; everyone ends."""
    left, foreign, failed, came, open_ = simulate(0, kind)
    assert left == foreign == open_ == 0 and failed > 1000 and came > 1000


@pytest.mark.parametrize("which,kind,leaves,reads", [(1, 1, True, True), (2, 1, True, False), (3, 1, False, True)])
def test_the_simulation_finds_careless_exchanges(simulate, which, kind, leaves, reads):
    """Planted: the order of steps without its precautions, and without either of them."""
    left, foreign, _, _, _ = simulate(which, kind)
    assert (left > 0) >= leaves and (foreign > 0) >= reads
