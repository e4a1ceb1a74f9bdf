// How the work of the key-value cache's kernels is cut: plain arithmetic, for the device and for the host (the tests run it there).
#pragma once
#include "kv_cache.cuh"

namespace eosb {

#define EOSB_HD __host__ __device__ __forceinline__

EOSB_HD int64_t kv_least(int64_t a, int64_t b) { return a < b ? a : b; }
EOSB_HD int64_t kv_most(int64_t a, int64_t b) { return a > b ? a : b; }

__host__ __device__ __attribute__((noinline)) inline int64_t kv_div64(int64_t a, int64_t b) { return a / b; }

// Division of a number that is not negative by a constant of the launch: below 2^31 floor(a / d) = a m >> s with
// s = 31 + ceil(log2 d), m = ceil(2^s / d) -- the excess a (m d - 2^s) / (d 2^s) is below 2^31 / 2^s <= 1 / d.
struct KvDiv {
    uint32_t d, m;
    int s;
    KvDiv() = default;
    explicit KvDiv(uint32_t by) : d(by), s(31) {
        while ((1ull << (s - 31)) < by) ++s;
        m = (uint32_t)(((s < 63 ? 1ull << s : 0) + by - 1) / by);
    }
    EOSB_HD int64_t operator()(int64_t a) const { return a >> 31 ? kv_div64(a, d) : (int64_t)((uint64_t)(uint32_t)a * m >> s); }
};
EOSB_HD int64_t kv_div(int64_t a, int64_t b) {   // not negative; the 32-bit division is far shorter
    return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : kv_div64(a, b);
}

// ---------------------------------------------------------------- append and read
// Work units of a call of `tokens` rows: one for each (sequence, record).  Sequence b, whose first row is `row`, starts at unit
// row / 16 + 2 b: n tokens that start anywhere in a record touch at most floor((n + 30) / 16) records, and the gap to sequence
// b + 1 is at least that.  (Without row offsets: one token, and unit, a sequence.)  Rows behind the last sequence belong to no unit.
EOSB_HD int64_t kv_unit_start(int row, int64_t b) { return (int64_t)(row >> 4) + 2 * b; }
EOSB_HD int64_t kv_units(bool offsets, int64_t tokens, int64_t batch) { return offsets ? (tokens >> 4) + 2 * batch : tokens; }

struct KvUnit {
    int b, rec;       // sequence, record index within the sequence
    int lo, hi;       // positions [lo, hi) of the record that the call covers
    int64_t row0;     // row of position 0 of the sequence (may be negative: rows are row0 + position)
    bool ok;
};
// The `first`-th unit of a sequence with n rows from `row` on, written from position `start` on; false: it has none such.
EOSB_HD bool kv_place(KvUnit& u, int64_t row, int64_t n, int64_t start, int64_t first) {
    const int64_t rec = (start >> 4) + first;
    if (first < 0 || rec * kKvRecord >= start + n) return false;
    u.rec = (int)rec;
    u.lo = (int)kv_most(start, rec * kKvRecord);
    u.hi = (int)kv_least(start + n, (rec + 1) * kKvRecord);
    u.row0 = row - start;
    return true;
}

// ---------------------------------------------------------------- attention
// Units are (sequence, key head, chunk of query heads); the records of all units, one unit after the other, are cut into equal
// ranges, one for each CTA and within it for each team, wherever the cuts fall -- or, where whole units make ranges that are
// hardly longer, the CTAs' cuts are between units.  kKvWhole is a number of records whatever their bytes.  Measured at both ends of
// it: 96 units of 32 to 64 records of 16 KB (23 more than an equal range) 30 us whole, 35 cut; 8 units of 125 records (117 more)
// 19.5 us whole, 13 cut.
constexpr int kKvMinRecords = 8;    // records of a CTA, at least
constexpr int kKvWhole = 24;        // records more than an equal range that a CTA may take to keep its units whole
// Neighbouring CTAs whose parts of a unit are joined first (at most 31 groups of it, for 744 SMs).  (Groups of 12: one sequence of 2000
// tokens and 8 heads, 16 CTAs a unit, 14.4 us instead of 12.9, of 131071 56.5 instead of 55.3.)
constexpr int kKvGroup = 24;

// Records of an equal range (of `total`, none of it empty but the last).  (At least 16 instead of 8: 1000 tokens 14.6 us instead of 12.2.)
EOSB_HD int64_t kv_part(const KvDiv& by_ctas, int64_t total) { return kv_most(by_ctas(total + by_ctas.d - 1), kKvMinRecords); }
// Whether `whole` units a CTA, of at most `longest` records, are left whole.
EOSB_HD bool kv_keep_whole(int64_t whole, int64_t longest, int64_t part) { return whole * longest <= part + kKvWhole; }

// A team's records of its CTA's [c0, c1).
struct KvRange {
    int64_t begin, end, part;
};
EOSB_HD KvRange kv_team_range(const KvDiv& by_teams, int64_t c0, int64_t c1, int team) {
    KvRange r;
    r.part = by_teams(c1 - c0 + by_teams.d - 1);
    r.begin = kv_least(c0 + team * r.part, c1);
    r.end = kv_least(r.begin + r.part, c1);
    return r;
}

// The CTAs that hold parts of a unit of `records` records from `from` on, among all, where ranges are equal: `parts` from `owner` on.
struct KvHolders {
    int owner, parts;
};
EOSB_HD KvHolders kv_holders(int64_t from, int64_t records, int64_t part) {
    KvHolders h;
    h.owner = (int)kv_div(from, part);
    h.parts = (int)kv_div(from + records - 1, part) - h.owner + 1;
    return h;
}
// What `cta` may join: of kKvGroup neighbours the parts (phase 1), then what the groups have joined (phase 2).  n results, with
// the CTAs lead, lead + step, ...; the joined one is left with `lead`.  `count`: the count of those that are done.
struct KvJoin {
    int lead, n, step, count;
};
EOSB_HD KvJoin kv_join(const KvHolders& h, int cta, int phase, int ctas) {
    KvJoin j;
    if (phase == 1) {
        const int group = (cta - h.owner) / kKvGroup, rest = h.parts - group * kKvGroup;
        j.lead = h.owner + group * kKvGroup;
        j.n = rest < kKvGroup ? rest : kKvGroup;
        j.step = 1;
        j.count = 2 * j.lead + (j.lead == h.owner ? 1 : 0);   // (a CTA leads at most a unit that begins in it and a group of an earlier one's)
    } else {
        j.lead = h.owner;
        j.n = (h.parts + kKvGroup - 1) / kKvGroup;
        j.step = kKvGroup;
        j.count = 2 * ctas + h.owner;
    }
    return j;
}

}  // namespace eosb
