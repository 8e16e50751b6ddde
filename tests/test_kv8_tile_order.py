"""The waits of the attention tiles' f32 rows, walked through in every order in
which the parts of a CTA can run.

The kernel's barriers are told apart by parity, so a wait is only right if it is
made between the end of the phase before and the end of the phase after the one
it means.  The model has the softmax's warps, the warp that issues the products,
the tensor cores that complete them, and the warps that add the tiles up; which
barrier and parity each wait takes comes from the kernel's own header."""
import ctypes as C
import os
import subprocess

import pytest

from conftest import PKG

SHIM = """
#include "kv8_order.h"
extern "C" int o_full(int split, int half, int n) {
  const qtts::TileTurn t = qtts::o_full_turn(split, half, n);
  return t.bar * 2 + (int)t.parity;
}
extern "C" int o_free(int n) {
  const qtts::TileTurn t = qtts::o_free_turn(n);
  return t.bar * 2 + (int)t.parity;
}
extern "C" int summed(int n) { return (int)qtts::summed_parity(n); }
"""


@pytest.fixture(scope="module")
def order(tmp_path_factory):
    d = tmp_path_factory.mktemp("order")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.check_call(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(PKG, "csrc"), "-o",
                           str(d / "shim.so"), str(d / "shim.cpp")])
    return C.CDLL(str(d / "shim.so"))


def walk(agents, counts):
    """Every reachable state of `agents` (lists of steps) and barriers of
    `counts` arrivals a phase.  Steps: ("arrive", bar); ("give", sem) and
    ("take", sem), a semaphore; ("wait", bar, parity, k), which the barrier lets
    through by parity and which means its k-th phase; ("order", bar, k), a wait
    that is right by itself.  Returns what is wrong, or None."""
    start = (tuple(0 for _ in agents), tuple(0 for _ in counts), ())
    seen, todo = {start}, [start]
    while todo:
        at, arrived, sems = todo.pop()
        sem = dict(sems)
        moved = finished = 0
        for a, steps in enumerate(agents):
            if at[a] == len(steps):
                finished += 1
                continue
            step = steps[at[a]]
            arr, left = arrived, sem
            if step[0] == "arrive":
                arr = arrived[:step[1]] + (arrived[step[1]] + 1,) + arrived[step[1] + 1:]
            elif step[0] == "give":
                left = dict(sem, **{step[1]: sem.get(step[1], 0) + 1})
            elif step[0] == "take":
                if not sem.get(step[1]):
                    continue
                left = dict(sem, **{step[1]: sem[step[1]] - 1})
            else:
                done = arrived[step[1]] // counts[step[1]]  # phases that have ended
                k = step[-1]
                if step[0] == "wait":
                    through = (done - 1) & 1 == step[2]
                    if through and done != k + 1:
                        return f"part {a} passes its wait for phase {k} of barrier {step[1]} after {done} phases"
                    if not through and done > k:
                        return f"part {a} misses phase {k} of barrier {step[1]}: {done} phases have ended"
                if done <= k:
                    continue
            nxt = (at[:a] + (at[a] + 1,) + at[a + 1:], arr, tuple(sorted(left.items())))
            moved += 1
            if nxt not in seen:
                seen.add(nxt)
                todo.append(nxt)
        if not moved and finished < len(agents):
            return f"nobody goes on at {at}"
    return None


S_FULL, P_FULL, O_FULL, O_FREE, SUMMED = 0, 1, 2, 4, 6


def f32_rows(order, segments, who=2, end=None):
    """The parts of a CTA with f32 rows over `segments` of so many tiles each,
    `who` threads standing for the 128 of the softmax and of the sums.  end: the
    softmax's step before it reads a segment's sums, of (segment, last tile)."""
    full = lambda n: (O_FULL + order.o_full(1, 0, n) // 2, order.o_full(1, 0, n) % 2)  # noqa: E731
    free = lambda n: (O_FREE + order.o_free(n) // 2, order.o_free(n) % 2)  # noqa: E731
    phase = lambda turn, n: sum(turn(i)[0] == turn(n)[0] for i in range(n))  # noqa: E731
    total = sum(segments)
    last = [sum(segments[:i + 1]) - 1 for i in range(len(segments))]
    issue, cores, softmax, sums = [], [], [], []
    for n in range(total):
        if n:  # score(n): P of the tile before lies where S goes
            issue.append(("wait", *full(n - 1), phase(full, n - 1)))
        issue += [("give", "s"), ("arrive", S_FULL)]
        cores += [("take", "s"), ("arrive", S_FULL)]
        issue.append(("wait", P_FULL, n & 1, n))  # weigh(n)
        if n > 1:
            issue.append(("wait", *free(n - 2), phase(free, n - 2)))
        issue += [("give", "o"), ("arrive", full(n)[0])]
        cores += [("take", "o"), ("arrive", full(n)[0])]
        softmax += [("wait", S_FULL, n & 1, n), ("arrive", P_FULL)]
        sums += [("wait", *full(n), phase(full, n)), ("arrive", free(n)[0])]
        if n in last:  # the segment's sums are read
            sums.append(("arrive", SUMMED))
            softmax.append(end(last.index(n), n) if end else ("order", free(n)[0], phase(free, n)))
    counts = [2, who, 2, 2, who, who, who]
    return [issue, cores] + [softmax] * who + [sums] * who, counts


@pytest.mark.parametrize("segments", [[1], [2], [5], [7], [1, 1, 1], [3, 1, 2], [2, 5]])
def test_no_wait_of_products_and_sums_is_left_to_timing(order, segments):
    assert walk(*f32_rows(order, segments)) is None


@pytest.mark.parametrize("segments", [[1], [2], [3], [6], [1, 1, 1], [3, 1, 2], [2, 5]])
def test_the_sums_are_read_when_all_tiles_are_in_them(order, segments):
    end = lambda i, n: ("wait", SUMMED, order.summed(i), i)  # noqa: E731
    assert walk(*f32_rows(order, segments, end=end)) is None


def test_the_walk_finds_sums_read_by_the_last_buffer_alone(order):
    # the order that was there before: the wait for o_free of the last tile
    end = lambda i, n: ("wait", O_FREE + (n & 1), (n >> 1) & 1, n >> 1)  # noqa: E731
    assert "of barrier %d" % O_FREE in walk(*f32_rows(order, [3], end=end))


def test_sixteen_bit_halves_have_a_barrier_each(order):
    for n in range(6):
        for half in (0, 1):
            assert order.o_full(0, half, n) == half * 2 + (n & 1)


def test_the_walk_finds_one_barrier_for_both_buffers(order):
    # the order that was there before: o_full by the tile's parity alone
    class One:
        o_free = staticmethod(order.o_free)

        @staticmethod
        def o_full(split, half, n):
            return n & 1

    assert "of barrier %d" % O_FULL in walk(*f32_rows(One, [5]))


def halves(order, segments, who):
    """The parts of a CTA with 16-bit rows: `segments` of (tiles, whether the
    first half holds rows of it, whether the second does); `who` threads of each
    group that arrives together."""
    k_full, v_full, k_free, v_free, s_full, p_full, o_full = (2 * i for i in range(7))
    full = lambda h, n: (o_full + order.o_full(0, h, n) // 2, order.o_full(0, h, n) % 2)  # noqa: E731
    convert, issue, cores, softmax = [], [], [], ([], [])
    done = [0, 0]

    def buffer(bar, it):  # the use of a pair of buffers by tile `it`
        return ("wait", bar + (it & 1), (it >> 1) & 1, it >> 1)

    def score(h, b, last):
        if done[h]:
            issue.append(("wait", *full(h, done[h] - 1), done[h] - 1))
        issue.extend([("give", "m"), ("arrive", s_full + h)])
        cores.extend([("take", "m"), ("arrive", s_full + h)] + ([("arrive", k_free + b)] if last else []))

    def weigh(h, b, last):
        n = done[h]
        done[h] += 1
        issue.extend([("wait", p_full + h, n & 1, n), ("give", "m")])
        cores.extend([("take", "m"), ("arrive", full(h, n)[0])] + ([("arrive", v_free + b)] if last else []))

    it = 0
    for tiles, one, two in segments:
        first, begin = it, list(done)
        for t in range(tiles):
            b = it & 1
            if it > 1:
                convert.append(buffer(k_free, it - 2))
            convert.append(("arrive", k_full + b))
            if it > 1:
                convert.append(buffer(v_free, it - 2))
            convert.append(("arrive", v_full + b))
            issue.append(buffer(k_full, it))
            if one:
                score(0, b, not two)
            if two and t:
                weigh(1, b ^ 1, True)
            if two:
                score(1, b, True)
            issue.append(buffer(v_full, it))
            if one:
                weigh(0, b, not two)
            it += 1
        if two and it > first:
            weigh(1, (it - 1) & 1, True)
        for h, here in ((0, one), (1, two)):
            for n in range(begin[h], done[h]):
                softmax[h].extend([("wait", s_full + h, n & 1, n), ("arrive", p_full + h)])
            if here and done[h] > begin[h]:
                softmax[h].append(("wait", *full(h, done[h] - 1), done[h] - 1))
    counts = [who] * 4 + [1] * 4 + [2] * 2 + [who] * 2 + [1] * 2
    return [issue, cores] + [convert] * who + [softmax[0]] * who + [softmax[1]] * who, counts


@pytest.mark.parametrize("who,segments", [(1, [(5, True, True)]), (1, [(3, True, False), (2, True, True), (3, False, True)]),
                                          (1, [(1, True, True)] * 3), (1, [(2, False, True), (1, True, False), (2, True, True)]),
                                          (2, [(3, True, True)]), (2, [(4, True, False)]), (2, [(2, True, False), (1, False, True)])])
def test_no_wait_of_two_halves_is_left_to_timing(order, who, segments):
    assert walk(*halves(order, segments, who)) is None
