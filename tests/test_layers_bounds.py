"""Plans that are none, and memory that is not there: what the layers' operators read and take then."""
import os
import subprocess

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_on_host(tmp_path, text, *arguments):
    """The output of a C++ program over the kernels' own headers, in numbers."""
    source, program = tmp_path / "program.cpp", tmp_path / "program"
    source.write_text(text)
    include = os.path.join(ROOT, "mops_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", include, "-o", str(program), str(source)], check=True)
    done = subprocess.run([str(program), *map(str, arguments)], check=True, capture_output=True, text=True)
    return np.array([[int(x) for x in line.split()] for line in done.stdout.splitlines()], dtype=np.int64)


PLACES = """
#include <cstdio>
#include <cstdlib>
#include "plan_bounds.hpp"
using namespace mops::amd;
// (what overflows is no constant expression: these lines would not compile)
static_assert(places_between(2147483647, 2147483647, 200000).begin == 200000, "");
static_assert(chunks_inside(places_between(2147483647, -2147483647 - 1, 2147418111), 8192).begin == 262136, "");
static_assert(chunks_inside(places_between(-2147483647 - 1, 2147483647, 2147418111), 8192).end == 262135, "");
int main(int n, char** a) {
    for (int i = 1; i + 3 < n; i += 4) {
        const Range places = places_between(atoi(a[i]), atoi(a[i + 1]), atoi(a[i + 2]));
        const Range chunks = chunks_inside(places, atoi(a[i + 3]));
        printf("%d %d %d %d\\n", places.begin, places.end, chunks.begin, chunks.end);
    }
}
"""


def test_offsets_that_are_none_stay_within_the_rows(tmp_path):
    """The places and chunks that the gradient of the embedding and the products count from two neighbouring offsets:
    within the rows for every pair of offsets, near the ends of 32 bits, negative and decreasing ones among them."""
    low, high = np.iinfo(np.int32).min, np.iinfo(np.int32).max
    rng = np.random.default_rng(0)
    points = []
    for n_rows in (0, 1, 63, 64, 257, 200_000, high - 65536):
        near = [low, low + 1, -1, 0, 1, 63, n_rows // 2, n_rows - 1, n_rows, n_rows + 1, high - 8192, high - 1, high]
        near = [int(np.clip(x, low, high)) for x in near] + rng.integers(low, high, 3).tolist()
        points += [(a, b, n_rows, chunk) for a in near for b in near for chunk in (32, 64, 8192)]
    got = np.concatenate(
        [run_on_host(tmp_path, PLACES, *np.ravel(points[i : i + 1000])) for i in range(0, len(points), 1000)]
    )
    a, b, n_rows, chunk = np.array(points, dtype=np.int64).T
    begin = np.clip(a, 0, n_rows)
    end = np.maximum(np.minimum(b, n_rows), begin)
    np.testing.assert_array_equal(got, np.stack([begin, end, -(-begin // chunk), end // chunk], 1))
    # nothing that a workgroup counts past a place leaves 32 bits: 256 teams with eight rows on their way each
    assert (got[:, :2] + 256 * 64).max() <= high and (got * np.array([1, 1, 0, 0])).min() >= 0
    inside = got[:, 2] < got[:, 3]
    assert ((got[:, 3] * chunk)[inside] <= n_rows[inside]).all()
