"""GPU tests of draws from rows whose cut goes through very many columns that weigh next to nothing each: the definition in numbers of
64 bits of mantissa, as sums of millions of them beside a peak of 1 would lose what they are about in fewer."""
import numpy as np
import pytest

from test_gpu_sample import as_setting, call, lib, torch  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -53


def definition(x, temperature, top_k, top_p):
    """(weights of all columns, place in the order of each, how many are kept, their running sums by column, weight at the cut)"""
    order = np.argsort(-x, kind="stable")
    some, which = np.unique(x, return_inverse=True)
    each = np.exp((some.astype(np.longdouble) - x.max()) / np.longdouble(np.float32(temperature)))
    w = each[which]
    w[x == x.max()] = 1
    falling = w[order]
    if top_k:
        falling = falling[:top_k]
    upto = np.cumsum(falling)
    count = min(int(np.searchsorted(upto, np.longdouble(np.float32(top_p)) * upto[-1])) + 1, len(falling))
    place = np.empty(len(x), np.int64)
    place[order] = np.arange(len(x))
    return w, place, count, np.cumsum(np.where(place < count, w, 0)), falling[count - 1]


def check(lib, x, kind, rows, temperature=1.0, top_k=0, top_p=1.0, draws=500):  # noqa: F811
    """One row in 64 bits, given `rows` times."""
    n = len(x)
    dev = torch.from_numpy(x).to({"f32": torch.float32, "bf16": torch.bfloat16}[kind]).cuda()
    x = dev.double().cpu().numpy()
    w, place, count, run, least = definition(x, temperature, top_k, top_p)
    # numbers that fall on what is not the best column's, and on that too
    best = int(np.argmax(x))
    tail = float((run[-1] - w[best]) / run[-1])
    u = ((np.arange(draws) + 0.5) / draws * tail).astype(np.float32) if best == n - 1 else (np.arange(draws) / draws).astype(np.float32)
    u[-3:] = [0.0, 0.5, 1 - 2.0 ** -24]
    uniform = torch.from_numpy(u).repeat(rows, 1).cuda()
    s = {"temperature": as_setting(temperature, rows, torch.float32), "top_p": as_setting(top_p, rows, torch.float32),
         "top_k": as_setting(top_k, rows, torch.int32) if top_k else None}
    labels, probs, _ = call(lib, dev.repeat(rows, 1), kind, uniform, **s)
    labels, probs = labels[:rows].cpu().numpy(), probs[:rows].double().cpu().numpy()
    assert (labels == labels[:1]).all() and (probs == probs[:1]).all()
    # What sums in 64 bits lose: a lane adds up to eight columns of each block of its segment (n / 2^18 blocks of 512 in one of 512
    # segments, four at least) to a 1, a few dozen additions of segments follow; twice, for the whole and for what lies above the cut.
    # The exponentials are off by 4e-14 of themselves, of all but the best column's, which is 1.
    adds = 8 * max(4, n / 2 ** 18) + 100
    off = float(run[-1]) * 2 * adds * U + 4e-14 * float(w.sum() - 1)
    near = off + 2 * float(least)                       # the cut comes a column sooner or later
    more = off / max(float(least), 1e-300) + 1
    for d in range(draws):
        l = int(labels[0, d])
        target = float(u[d]) * run[-1]
        assert 0 <= l < n, f"draw {d} ({u[d]}): label {l}, probability {probs[0, d]}; {count} columns are left"
        assert place[l] < count + more, f"draw {d} ({u[d]}): column {l} is the {place[l]}th of {count} that are left"
        assert run[l] > target - near and run[l] - w[l] <= target + near, \
            f"draw {d} ({u[d]}): column {l} ends at {float(run[l])}, {float((run[l] - target) / least):.1f} columns from {float(target)}"
        assert abs(probs[0, d] - w[l] / run[-1]) <= 2.0 ** -23 * w[l] / run[-1] + near * w[l], (d, probs[0, d], float(w[l] / run[-1]))


def peak_and_tail(n, low, high, seed, last=True):
    x = np.random.default_rng(seed).uniform(low, high, n)
    x[n - 1 if last else 0] = 0.0
    return x


@pytest.mark.parametrize("rows,n,low,high,top_p", [
    (2, 131_072, -27.75, -27.73, 1 - 2.0 ** -24), (130, 131_072, -27.75, -27.73, 1 - 2.0 ** -24), (1, 2 ** 21, -29.0, -28.9, 0.9999999),
    (1, 2 ** 22, -28.51, -28.49, 0.9999995), (1, 2 ** 24 - 3, -27.01, -26.99, 0.99999), (129, 300_001, -26.0, -25.95, 0.9999999),
    (3, 1_000_003, -29.0, -25.0, 0.9999999), (130, 60_000, -24.02, -24.0, 0.9999997), (2, 60_000, -24.02, -24.0, 0.9999997)])
@pytest.mark.parametrize("last", [True, False])
def test_a_peak_over_a_flat_tail(lib, rows, n, low, high, top_p, last):  # noqa: F811
    check(lib, peak_and_tail(n, low, high, n, last), "f32", rows, top_p=top_p)


@pytest.mark.parametrize("rows", [1, 130])
def test_a_cut_in_a_short_list_of_small_weights(lib, rows):  # noqa: F811
    """The list holds all that lie around the cut: their sums go to the segments."""
    check(lib, peak_and_tail(2 ** 20, -36.7, -27.7, 3), "f32", rows, top_p=1 - 2.0 ** -24)
    check(lib, peak_and_tail(131_072, -36.0, -25.0, 4), "f32", rows, top_p=1 - 2.0 ** -24)


@pytest.mark.parametrize("rows", [2, 130])
@pytest.mark.parametrize("temperature,distance", [(0.25, 6.9), (40.0, 1100.0), (1e4, 2.75e5)])
def test_other_temperatures(lib, rows, temperature, distance):  # noqa: F811
    x = peak_and_tail(200_000, -distance - 0.02 * temperature, -distance, 5)
    check(lib, x, "f32", rows, temperature=temperature, top_p=0.9999999)


@pytest.mark.parametrize("rows", [2, 130])
def test_scores_of_few_steps_of_their_type(lib, rows):  # noqa: F811
    """Neither bins nor brackets can tell them apart: the row is gone through as a whole, from the best score to the lowest."""
    rng = np.random.default_rng(6)
    x = 1e8 - 8.0 * (100 + rng.integers(0, 3, 200_000))
    x[-1] = 1e8
    check(lib, x, "f32", rows, temperature=29.0, top_p=0.9999999)
    x = 1e8 - 8.0 * rng.integers(0, 40, 200_000)
    x[-1] = 1.001e8
    for top_p in (0.5, 0.999, 0.9999999):
        check(lib, x, "f32", rows, temperature=4000.0, top_p=top_p)


@pytest.mark.parametrize("rows", [2, 130])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_all_scores_and_few_of_them_far_apart(lib, rows, kind):  # noqa: F811
    """Wide rows of many sizes: the cut lies in the middle, near the end, and behind a count."""
    rng = np.random.default_rng(7)
    x = np.concatenate((rng.uniform(-12, -8, 50_000), rng.uniform(-300, -12, 100_000), np.full(30_000, -11.25), [0.0]))
    x = x[np.concatenate((rng.permutation(len(x) - 1), [len(x) - 1]))]
    for top_p in (0.3, 0.9, 0.99999, 1 - 2.0 ** -24):
        check(lib, x, kind, rows, top_p=top_p)
        check(lib, x, kind, rows, top_p=top_p, top_k=70_000)
