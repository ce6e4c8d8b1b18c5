"""What running the paged kernels cannot show, because it only matters once a bounded wait has given up: read from the
source. A wait may end differently in the lanes of a warp (one sees the barrier complete, another that a role has failed),
so its result is voted on before any lane goes by it."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nekochat_b200", "csrc")


def lines(name):
    with open(os.path.join(CSRC, name)) as f:
        return [re.sub(r"//.*", "", x).strip() for x in f]


def test_waits_of_a_role_are_voted_on():
    src = lines("k_paged_prompt.cu")
    at = [i for i, x in enumerate(src) if re.search(r"\bok = .*wait_on\(", x)]
    assert len(at) >= 6
    for i in at:
        after = src[i + 1]
        assert after.startswith("ok = __all_sync(0xffffffffu, ok);"), f"line {i + 1}: {src[i]} / {after}"


def test_a_loader_that_gives_up_waits_for_its_copies():
    """After the loop that starts tensor copies, the warp that started them waits, with a limit, for those in flight."""
    src = lines("k_paged_prompt.cu")
    start = next(i for i, x in enumerate(src) if "copy_box(base" in x)
    end = next(i for i, x in enumerate(src) if i > start and "} else if (warp == kMmaWarp)" in x)
    rest = " ".join(src[start:end])
    given_up = rest.partition("if (!ok && warp == kLoadWarp)")[2]
    assert "wait_out(&ms.full[" in given_up and "wait_out(&ms.land" in given_up


def test_what_lanes_write_is_ordered_before_the_arrival_that_publishes_it():
    """Several lanes of the loader store a tile's scales and lane 0 arrives: a warp barrier stands between."""
    src = lines("k_paged_prompt.cu")
    stores = [i for i, x in enumerate(src) if "ms.ks[i % kRing][lane] =" in x]
    assert len(stores) == 2
    for i in stores:
        rest = src[i:]
        one = next(j for j, x in enumerate(rest) if re.search(r"mbar_arrive(_expect_tx)?\(", x))
        alone = "lane == 0" in rest[one]
        assert not alone or any("__syncwarp()" in x for x in rest[:one])


def test_what_is_asked_once_is_asked_once_per_device():
    """Clusters that run at once: kept by device, like the number of SMs beside it (one GPU cannot show the difference)."""
    src = " ".join(lines("k_paged_prompt.cu"))
    body = src[src.index("int clusters_at_once(int log) {"):]
    assert "cudaGetDevice(&dev)" in body[:300] and "[dev & 63]" in body[:400]
