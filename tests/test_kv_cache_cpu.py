"""Paged key-value cache, what needs no device: the record layout is a bijection within its bounds, the work units of an
append cover every record once, and bad arguments are refused before a device is touched."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

LAYOUT_CHECK = r"""
#include <cstdio>
#include <vector>
#include "kv_cache.cuh"
using namespace eosb;
int main() {
    const int dims[] = {32, 64, 96, 128, 192, 256};
    for (int format = 0; format < 4; ++format)
        for (int dim : dims) {
            const int nb = dim / 32, kp = kv_key_piece(format), vp = kv_value_piece(format), total = kv_record_bytes(format, nb);
            if (total % 16 || kv_value_offset(format, nb) % 16 || kv_key_scale_offset(format, nb) % 16 ||
                kv_value_scale_offset(format, nb) % 16) return 1;
            std::vector<int> seen(total, 0);
            auto piece = [&](int base, int bytes, int lane, int p, int size) {   // one access of `size` bytes
                const int at = base + kv_lane_offset(bytes, lane, p);
                if (at % (size < 16 ? size : 16) != 0) return false;
                for (int i = 0; i < size; ++i) {
                    if (base + kv_lane_offset(bytes, lane, p + i) != at + i || at + i >= total) return false;
                    seen[at + i]++;
                }
                return true;
            };
            for (int lane = 0; lane < 32; ++lane)
                for (int b = 0; b < nb; ++b) {
                    if (format <= kKvBf16) {   // both tokens' words in turn
                        for (int j = 0; j < 2; ++j)
                            for (int i = 0; i < 4; ++i)
                                if (!piece(0, 2 * nb * kp, lane, 32 * b + 16 * (i >> 1) + 8 * (i & 1) + 4 * j, 4)) return 2;
                    } else {
                        for (int j = 0; j < 2; ++j)
                            if (!piece(j * 32 * nb * kp, nb * kp, lane, b * kp, kp)) return 2;
                    }
                    const int step = vp < 16 ? vp : 16;
                    for (int p = 0; p < vp; p += step)
                        if (!piece(kv_value_offset(format, nb), nb * vp, lane, b * vp + p, step)) return 3;
                }
            for (int i = 0; i < kv_key_scale_offset(format, nb); ++i)
                if (seen[i] != 1) return 4;
            if (format >= kKvMx8) {   // scales of 16 tokens behind the codes
                if (kv_scale_stride(nb) < nb || kv_scale_bytes(format, nb) != 16 * kv_scale_stride(nb)) return 5;
                if (kv_value_top_offset(format, nb) != kv_value_scale_offset(format, nb) + 16 * kv_scale_stride(nb)) return 6;
                if (kv_value_top_offset(format, nb) + 32 != total) return 6;
            } else if (kv_key_scale_offset(format, nb) != total) return 7;
        }
    std::puts("ok");
}
"""


def test_record_layout_is_a_bijection(tmp_path):
    src = tmp_path / "layout.cpp"
    src.write_text(LAYOUT_CHECK)
    exe = tmp_path / "layout"
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.check_call(["g++", "-std=c++17", "-I", os.path.join(ROOT, "eos_b200", "csrc"), "-I", os.path.join(cuda, "include"),
                           str(src), "-o", str(exe)])
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout == "ok\n"


def run_cpp(tmp_path, body):
    """Compiles a main() with the cache's host-side header and runs it; it prints ok."""
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text("#include <climits>\n#include <cstdio>\n#include <cstdlib>\n#include <set>\n#include <utility>\n#include <vector>\n"
                   '#include "kv_cache.cuh"\nusing namespace eosb;\n' + body)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.check_call(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                           os.path.join(ROOT, "eos_b200", "csrc"), "-I", os.path.join(cuda, "include"), str(src), "-o", str(exe)])
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout == "ok\n"


def test_records_of_a_span_up_to_the_largest_position(tmp_path):
    run_cpp(tmp_path, r"""
int main() {
    const int ends[] = {0, 1, 15, 16, 17, 31, 32, 1000, 65536, INT_MAX - 33, INT_MAX - 17, INT_MAX - 16, INT_MAX - 15, INT_MAX - 14, INT_MAX - 1, INT_MAX};
    for (int lo : ends)
        for (int hi : ends) {
            const long long want = hi > lo ? ((long long)hi + 15) / 16 - lo / 16 : 0;
            if (kv_records(lo, hi) != want) return 1;
        }
    std::puts("ok");
}
""")


def test_work_units_cover_every_record_once():
    """The unit arithmetic of an append / read: sequence b starts at unit cu[b] // 16 + 2 b, unit i of a sequence is its
    i-th touched record, and tokens // 16 + 2 batch units are enough."""
    rng = random.Random(5)
    for _ in range(300):
        batch = rng.randrange(1, 40)
        counts = [rng.choice([0, 1, 2, 15, 16, 17, 31, rng.randrange(0, 200)]) for _ in range(batch)]
        starts = [rng.randrange(0, 100) for _ in range(batch)]
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        spare = rng.randrange(0, 20)                      # rows behind the last sequence
        units = (cu[-1] + spare) // 16 + 2 * batch
        done = {}
        for u in range(units):
            b = max(i for i in range(batch) if i == 0 or cu[i] // 16 + 2 * i <= u)
            rec = starts[b] // 16 + u - (cu[b] // 16 + 2 * b)
            if counts[b] and rec >= starts[b] // 16 and rec * 16 < starts[b] + counts[b]:
                done[b, rec] = done.get((b, rec), 0) + 1
        want = {(b, r) for b in range(batch) if counts[b]
                for r in range(starts[b] // 16, (starts[b] + counts[b] - 1) // 16 + 1)}
        assert set(done) == want and set(done.values()) <= {1}


def test_split_and_join_cover_every_record_once():
    """The cut of the attention's work: ranges of CTAs and teams, which of their units are whole, begun or continued, and
    the CTAs that a unit's parts are gathered from."""
    rng = random.Random(6)
    for _ in range(300):
        batch, per_seq = rng.randrange(1, 30), rng.choice([1, 2, 5, 8])
        n = [rng.choice([0, 0, 1, 2, 7, rng.randrange(0, 400)]) for _ in range(batch)]
        ctas, teams, least = rng.choice([1, 3, 148]), rng.choice([1, 2, 4, 8]), rng.choice([1, 8])
        units = [(b, hu) for b in range(batch) if n[b] for hu in range(per_seq)]
        flat = [(u, r) for u in units for r in range(n[u[0]])]
        total = len(flat)
        part = max(-(-total // ctas), least)
        parts, whole, more = {}, set(), {}
        for c in range(ctas):
            c0 = min(c * part, total)
            c1 = min(c0 + part, total)
            step = -(-(c1 - c0) // teams)
            entries = []
            for t in range(teams):
                t0 = min(c0 + t * step, c1)
                t1 = min(t0 + step, c1)
                while t0 < t1:
                    u, r = flat[t0]
                    seg = min(n[u[0]] - r, t1 - t0)
                    begins, ends = r == 0, r + seg == n[u[0]]
                    if begins and ends:
                        assert u not in whole
                        whole.add(u)
                    else:
                        entries.append((2 * t + begins, u, begins + 2 * ends, seg))
                    t0 += seg
            assert len({e[0] for e in entries}) == len(entries)          # a slot is used once
            assert [e[0] for e in entries] == sorted(e[0] for e in entries)
            i = 0
            while i < len(entries):                                      # runs of equal units
                j, ends, count = i, 0, 0
                while j < len(entries) and entries[j][1] == entries[i][1]:
                    ends |= entries[j][2]
                    count += entries[j][3]
                    j += 1
                u = entries[i][1]
                if ends == 3:
                    assert u not in whole and count == n[u[0]]
                    whole.add(u)
                else:
                    which = ends & 1
                    assert (c, which) not in parts
                    parts[c, which] = (u, count)
                    if which:
                        end = flat.index((u, 0)) + n[u[0]]
                        more[c] = (end - 1) // part - c
                i = j
        for c, k in more.items():
            u = parts[c, 1][0]
            got = [parts[c, 1]] + [parts[c + i, 0] for i in range(1, k + 1)]
            assert all(g[0] == u for g in got) and sum(g[1] for g in got) == n[u[0]] and u not in whole
            whole.add(u)
        assert whole == set(units) and sum(1 + k for k in more.values()) == len(parts)


def test_cuts_between_units_cover_every_unit_once():
    """The cut where units are left whole: CTA i begins with the first record of unit i * whole."""
    rng = random.Random(8)
    for _ in range(500):
        batch, per_seq, ctas = rng.randrange(1, 60), rng.choice([1, 2, 5, 8]), rng.choice([1, 3, 148])
        n = [rng.choice([0, 1, rng.randrange(0, 60)]) for _ in range(batch)]
        before = [sum(n[:b]) for b in range(batch)]
        total, units = sum(n) * per_seq, batch * per_seq
        whole = -(-units // ctas)

        def begin(cta):
            u = cta * whole
            return total if u >= units else before[u // per_seq] * per_seq + u % per_seq * n[u // per_seq]

        starts, at = set(), 0
        for b in range(batch):
            for _ in range(per_seq):
                starts.add(at)
                at += n[b]
        cuts = [begin(c) for c in range(ctas + 1)]
        assert cuts[0] == 0 and cuts[-1] == total and cuts == sorted(cuts) and set(cuts) <= starts | {total}
        assert all(b - a <= whole * max(n) for a, b in zip(cuts, cuts[1:]))


def test_refusals_without_a_device():
    import eos_b200
    from eos_b200 import _lib
    with pytest.raises(ValueError, match="format"):
        eos_b200.KvCache(None, 1, 16, 1, 64, "fp3")
    for name, args in (("eos_b200_kv_cache_create", (None, 1, 16, 1, 64, 0, C.byref(C.c_void_p()))),
                       ("eos_b200_kv_cache_append_device", (None, None, None, 0, 0, None, 0, None, 0, None, None, None, None)),
                       ("eos_b200_kv_cache_read_device", (None, None, None, 0, 0, None, 0, None, 0, None, None, None, None)),
                       ("eos_b200_kv_cache_attend_device", (None, None, 0, 1, 0, 0, 0, None, 0, None, 1.0, 0, None, None, None, None)),
                       ("eos_b200_kv_cache_sync", (None, None))):
        with pytest.raises(eos_b200.EosB200Error, match="null"):
            _lib.call(name, *args)
    assert _lib.lib().eos_b200_kv_cache_page_bytes(None) == 0
    _lib.lib().eos_b200_kv_cache_destroy(None)


class FakeLibrary:
    """Entry points that wait for another call in flight before they answer: with the token count as launches, or an error."""

    def __init__(self):
        import threading
        self.both = threading.Barrier(2, timeout=20)
        self.freed = []

    def eos_b200_kv_cache_create(self, *args):
        return 0

    def eos_b200_kv_cache_destroy(self, handle):
        pass

    def eos_b200_free_cstring(self, p):
        self.freed.append(p)

    def _rows(self, handle, key, value, type_, tokens, strides, batch, *rest):
        stats, err = (r._obj for r in rest[-2:])
        stats.kernel_launches = tokens
        if batch < 0:
            err.value = b"refused %d" % tokens
        self.both.wait()       # both have written
        self.both.wait()
        return 1 if batch < 0 else 0

    eos_b200_kv_cache_append_device = eos_b200_kv_cache_read_device = _rows

    def eos_b200_kv_cache_attend_device(self, handle, query, type_, q_heads, *rest):
        return self._rows(handle, None, None, type_, q_heads, None, rest[2], *rest)


def fake_cache(monkeypatch):
    from types import SimpleNamespace

    import eos_b200
    from eos_b200 import _lib
    fake = FakeLibrary()
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    return eos_b200.KvCache(SimpleNamespace(handle=None, _adopt=lambda child: None), 1, 16, 1, 64), fake


def test_calls_of_two_threads_keep_their_results_apart(monkeypatch):
    """ctypes lets other threads run during a call: launches and errors are those of the thread's own call."""
    from concurrent.futures import ThreadPoolExecutor

    import eos_b200
    cache, fake = fake_cache(monkeypatch)
    calls = [lambda n, b: cache.append_device(1, 1, "f16", n, b, 1, 1, 1), lambda n, b: cache.read_device(1, 1, "f16", n, b, 1, 1, 1),
             lambda n, b: cache.attend_device(1, "f16", n, b, 1, 1, 1, 1, 1.0)]
    with ThreadPoolExecutor(2) as pool:
        for one in calls:
            for two in calls:
                got = [pool.submit(one, 3, 1), pool.submit(two, 5, 1)]
                assert [g.result(30) for g in got] == [3, 5]
                got = [pool.submit(one, 7, -1), pool.submit(two, 9, -1)]
                errors = [g.exception(30) for g in got]
                assert all(isinstance(e, eos_b200.EosB200Error) for e in errors) and [str(e) for e in errors] == ["refused 7", "refused 9"]
    assert len(fake.freed) == 2 * len(calls) ** 2


def test_strides_of_the_wrong_count_are_refused(monkeypatch):
    cache, _ = fake_cache(monkeypatch)
    for call in (cache.append_device, cache.read_device):
        for strides in ((64, 64), (64, 64, 64), (64,) * 5, ()):
            with pytest.raises(ValueError, match="strides"):
                call(1, 1, "f16", 1, 1, 1, 1, 1, strides=strides)
    for strides in ((64,), (64, 64, 64), ()):
        with pytest.raises(ValueError, match="strides"):
            cache.attend_device(1, "f16", 1, 1, 1, 1, 1, 1, 1.0, query_strides=strides)


def test_divisions_by_constants_of_a_launch(tmp_path):
    run_cpp(tmp_path, r"""
#include "kv_split.cuh"
int main() {
    std::srand(1);
    const long long fixed[] = {0, 1, 2, 15, 16, 147, 148, 149, (1ll << 31) - 2, (1ll << 31) - 1, 1ll << 31, (1ll << 31) + 1, 1ll << 40};
    for (int i = 0; i < 3000; ++i) {
        const uint32_t d = i < 2000 ? i + 1 : i < 2030 ? 1u << (i - 2000) : 1u + (uint32_t)std::rand();
        const KvDiv by(d);
        for (long long a : fixed)
            if (by(a) != a / d || kv_div(a, d) != a / d) return 1;
        for (int j = 0; j < 200; ++j) {
            const long long r = std::rand(), k = r / d * d;   // and next to multiples
            for (long long a : {r, k, k + d - 1, k ? k - 1 : 0})
                if (by(a) != a / d || kv_div(a, d) != a / d) return 2;
        }
    }
    std::puts("ok");
}
""")


def test_work_units_place_every_row_once(tmp_path):
    """The kernels' own arithmetic: every position of every sequence is in one unit, with the row that belongs to it."""
    run_cpp(tmp_path, r"""
#include "kv_split.cuh"
int main() {
    std::srand(2);
    const int some[] = {0, 1, 2, 15, 16, 17, 31};
    for (int round = 0; round < 400; ++round) {
        const int batch = 1 + std::rand() % 40;
        std::vector<int> n(batch), start(batch), cu(1, 0);
        for (int b = 0; b < batch; ++b) {
            n[b] = std::rand() % 3 ? some[std::rand() % 7] : std::rand() % 200;
            start[b] = std::rand() % 4 ? std::rand() % 100 : INT_MAX - n[b] - std::rand() % 20;
            cu.push_back(cu.back() + n[b]);
        }
        const int tokens = cu.back() + std::rand() % 20;   // rows behind the last sequence
        std::set<std::pair<int, int>> seen;
        for (int64_t u = 0; u < kv_units(true, tokens, batch); ++u) {
            int b = 0;
            for (int i = 1; i < batch; ++i)
                if (kv_unit_start(cu[i], i) <= u) b = i;
            KvUnit w{};
            if (n[b] == 0 || !kv_place(w, cu[b], n[b], start[b], u - kv_unit_start(cu[b], b))) continue;
            if (w.lo >= w.hi || w.lo / 16 != w.rec || (w.hi - 1) / 16 != w.rec) return 1;
            for (int64_t p = w.lo; p < w.hi; ++p) {
                const int64_t row = w.row0 + p;
                if (row < cu[b] || row >= cu[b + 1] || p != start[b] + (row - cu[b])) return 2;
                if (!seen.insert({b, (int)row}).second) return 3;
            }
        }
        if ((int)seen.size() != cu.back()) return 4;
        for (int b = 0; b < batch; ++b) {   // without row offsets: a unit a sequence
            KvUnit w{};
            if (start[b] == INT_MAX) continue;
            if (!kv_place(w, b, 1, start[b], 0) || w.lo != start[b] || w.hi != start[b] + 1 || w.row0 + w.lo != b) return 5;
        }
        if (kv_units(false, batch, batch) != batch) return 6;
    }
    std::puts("ok");
}
""")


def test_parts_of_a_unit_are_joined_once(tmp_path):
    """The kernel's own ranges and joins: what teams and CTAs hold of every unit, who joins it and which count says so."""
    run_cpp(tmp_path, r"""
#include <map>
#include "kv_split.cuh"
struct Part { int unit, records, which; KvHolders held; };
int main() {
    std::srand(3);
    for (int round = 0; round < 1500; ++round) {
        const int all_ctas[] = {1, 3, 24, 25, 49, 148, 744}, all_teams[] = {1, 2, 3, 4, 8, 12, 16};
        const int ctas = all_ctas[std::rand() % 7], teams = all_teams[std::rand() % 7], units = 1 + std::rand() % 60;
        std::vector<int64_t> n(units), from(units + 1, 0);
        const int kind = std::rand() % 3;
        for (int u = 0; u < units; ++u) {
            n[u] = kind == 0 ? 1 + std::rand() % 9 : kind == 1 ? 1 + std::rand() % 400 : u == units / 2 ? 1 + std::rand() % 20000 : 1 + std::rand() % 50;
            from[u + 1] = from[u] + n[u];
        }
        const int64_t total = from[units];
        const KvDiv by_ctas(ctas), by_teams(teams);
        const int64_t part = kv_part(by_ctas, total);
        if (part * ctas < total || part < kKvMinRecords) return 1;
        std::vector<int64_t> whole(units, 0);
        std::map<std::pair<int, int>, Part> parts;   // (cta, which)
        for (int c = 0; c < ctas; ++c) {
            const int64_t c0 = kv_least(c * part, total), c1 = kv_least((c + 1) * part, total);
            struct Entry { int unit; bool begins, ends; int records; int64_t from; };
            std::vector<Entry> entries;
            int64_t reached = c0;
            for (int t = 0; t < teams; ++t) {
                const KvRange r = kv_team_range(by_teams, c0, c1, t);
                if (r.begin != reached || r.end < r.begin) return 2;
                reached = r.end;
                for (int64_t at = r.begin; at < r.end;) {
                    int u = 0;
                    while (from[u + 1] <= at) ++u;
                    const int64_t end = kv_least(from[u + 1], r.end);
                    const bool begins = at == from[u], ends = end == from[u + 1];
                    if (begins && ends) whole[u] += n[u];
                    else entries.push_back({u, begins, ends, (int)(end - at), from[u]});
                    at = end;
                }
            }
            if (reached != c1) return 3;
            for (size_t i = 0; i < entries.size();) {   // runs of equal units
                size_t j = i;
                bool begun = false, ended = false;
                int records = 0;
                for (; j < entries.size() && entries[j].unit == entries[i].unit; ++j) {
                    begun |= entries[j].begins, ended |= entries[j].ends;
                    records += entries[j].records;
                }
                const int u = entries[i].unit;
                if (begun && ended) whole[u] += records;
                else {
                    if (begun ? j != entries.size() : i != 0) return 4;   // only the first and the last run are open
                    if (parts.count({c, begun ? 1 : 0})) return 5;
                    parts[{c, begun ? 1 : 0}] = {u, records, begun ? 1 : 0, kv_holders(from[u], n[u], part)};
                }
                i = j;
            }
        }
        std::map<int, std::pair<int, int>> counts;   // count -> (unit, lead)
        std::map<int, int> arrivals;
        for (auto& [key, p] : parts) {
            const int c = key.first, u = p.unit;
            if (c < p.held.owner || c >= p.held.owner + p.held.parts || p.which != (c == p.held.owner ? 1 : 0)) return 6;
            whole[u] += p.records;
            const KvJoin a = kv_join(p.held, c, 1, ctas);
            if (c < a.lead || c >= a.lead + a.n * a.step || a.n > kKvGroup || a.n > 31) return 7;
            for (int i = 0; i < a.n; ++i) {
                auto q = parts.find({a.lead + i * a.step, a.lead + i * a.step == p.held.owner ? 1 : 0});
                if (q == parts.end() || q->second.unit != u) return 8;
            }
            if (a.count < 0 || a.count >= 2 * ctas || !counts.emplace(a.count, std::make_pair(u, a.lead)).second && counts[a.count] != std::make_pair(u, a.lead)) return 9;
            if (++arrivals[a.count] > a.n) return 10;
            if (arrivals[a.count] == a.n && p.held.parts > kKvGroup) {   // this group is joined: phase 2
                const KvJoin g = kv_join(p.held, c, 2, ctas);
                if (g.lead != p.held.owner || g.n > 31 || g.count < 2 * ctas || g.count >= 3 * ctas) return 11;
                if (!counts.emplace(g.count, std::make_pair(u, -1)).second && counts[g.count] != std::make_pair(u, -1)) return 12;
                bool leads = false;
                for (int i = 0; i < g.n; ++i) leads |= g.lead + i * g.step == a.lead;
                if (!leads || ++arrivals[g.count] > g.n) return 13;
            }
        }
        for (auto& [key, p] : parts) {   // every count is reached
            const KvJoin a = kv_join(p.held, key.first, 1, ctas);
            if (arrivals[a.count] != a.n) return 14;
            const KvJoin g = kv_join(p.held, key.first, 2, ctas);
            if (p.held.parts > kKvGroup && arrivals[g.count] != g.n) return 15;
        }
        for (int u = 0; u < units; ++u)
            if (whole[u] != n[u]) return 16;
        // whole units: those that fit a little more than an equal range
        if (!kv_keep_whole(1, part + kKvWhole, part) || kv_keep_whole(1, part + kKvWhole + 1, part)) return 17;
    }
    std::puts("ok");
}
""")


def test_scales_of_a_live_token_beside_one_that_is_being_written(tmp_path):
    """An attention may read a record while the token behind the last is appended: whatever bytes that one has at the moment, the live
    token's come out as they are."""
    run_cpp(tmp_path, r"""
int main() {
    std::srand(4);
    for (int round = 0; round < 2000000; ++round) {
        const int live = std::rand() % 3;   // the first, the second, both
        uint32_t top[2], e[2][2];
        for (int i = 0; i < 2; ++i) {
            top[i] = std::rand() % 255;
            for (int b = 0; b < 2; ++b) {
                const int down = std::rand() % (kKvNear + 1);
                e[b][i] = live == i || live == 2 ? (top[i] > (uint32_t)down ? top[i] - down : 0) : std::rand() % 256;
            }
        }
        const uint32_t mask = kv_live_bytes(live != 1, live != 0);
        const uint32_t scales = e[0][0] | e[0][1] << 8 | e[1][0] << 16 | e[1][1] << 24, pair = top[0] | top[1] << 8;
        const uint32_t got = kv_relative_scales(scales & mask, (pair | pair << 16) & mask);
        for (int i = 0; i < 2; ++i)
            for (int b = 0; b < 2; ++b)
                if ((live == i || live == 2) && (got >> (16 * b + 8 * i) & 255) != 60 - 4 * (top[i] - e[b][i])) return 1;
    }
    std::puts("ok");
}
""")
