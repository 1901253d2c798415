// Host program of tests/test_attend_plan.py: the sizes of plans (attend_sizes) whose arguments come on lines of standard input:
// rows B Hq Hkv T shared shared_T max_rows; tiles, joins, units, partial rows and the parts' places in the workspace go out.
#include <cstdio>

#include "../kvskip_amd/csrc/attend_plan.hip"

int main() {
  kvskip_attend_plan_args p{};
  while (std::scanf("%d %d %d %d %d %d %d %d", &p.rows, &p.B, &p.Hq, &p.Hkv, &p.T, &p.shared, &p.shared_T, &p.max_rows) == 8) {
    const kvs::AttendSizes z = kvs::attend_sizes(p);
    std::printf("%lld %lld %lld %lld %lld %lld %lld %lld %lld\n", (long long)z.tiles, (long long)z.joins, (long long)z.units,
                (long long)z.part_rows, (long long)z.at_units, (long long)z.at_joins, (long long)z.at_tiles, (long long)z.at_rows,
                (long long)z.total);
  }
  return 0;
}
