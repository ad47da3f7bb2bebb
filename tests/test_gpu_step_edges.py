"""Tokens from logits and plans at the edges of what their calls take, against the plain forms of tests/step_ref.py (see test_gpu_step.py for how near is equal)."""
import pytest
import torch

from gevva_b200 import step
from tests.test_gpu_step import DEV, compare, generator, ints

pytestmark = pytest.mark.gpu


def f32(values):
    return torch.tensor(values, dtype=torch.float32, device=DEV)


# ---- low temperatures, no cap

def rows_with_ties(gen, vocabulary, dtype):
    """Largest values of several sizes, some several times, some with the next floats below beside them, and a bulk further down."""
    largest = [10.0, 10.0, 20.0, 0.1, -20.0, 17.3, 1000.0, 0.0]
    x = torch.randn(len(largest), vocabulary, generator=gen, device=DEV) * 2.5
    for r, most in enumerate(largest):
        x[r] = most - 1.0 - x[r].abs() * max(1.0, abs(most) / 16)
        at = torch.randperm(vocabulary, generator=gen, device=DEV)
        top = torch.tensor(most, dtype=dtype, device=DEV)
        x[r, at[:r % 4 + 1]] = top.float()
        if r % 2:
            x[r, at[8:11]] = torch.nextafter(top, torch.full_like(top, -1e9)).float()
    return x.to(dtype)


@pytest.mark.parametrize("vocabulary", [100, 9000, 70001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1e-4, 1e-6, 1e-7, 1e-8, 3e-9, 1e-9, 1e-10, 1e-12, 1e-15, 1e-20, 1e-29])
def test_low_temperatures(vocabulary, dtype, temperature):
    """A step of 32 bits is many temperatures there: what is next to the largest has next to no share, and the largest ones have equal ones."""
    gen = generator(vocabulary + 11)
    logits = rows_with_ties(gen, vocabulary, dtype)
    rows = len(logits)
    cold = torch.full((rows,), temperature, device=DEV)
    for rules in ({}, dict(top_p=f32([0.35] * rows)), dict(top_p=f32([0.999] * rows)), dict(top_k=ints([2] * rows)), dict(top_k=ints([400] * rows)),
                  dict(min_p=f32([0.1] * rows)), dict(top_k=ints([400] * rows), top_p=f32([0.6] * rows), min_p=f32([0.01] * rows)),
                  dict(top_p=f32([-1.0] * rows))):
        for _ in range(2):
            compare(logits, torch.rand(rows, generator=gen, device=DEV), dict(rules, temperature=cold))


# ---- values so near one another that bins of equal width between them are too narrow for numbers of 32 bits

@pytest.mark.parametrize("vocabulary", [100, 500, 900, 5000, 70001])
@pytest.mark.parametrize("spread", [1e-45, 1e-38, 1e-37, 3e-36, 1e-30])
def test_first_of_a_narrow_range(vocabulary, spread):
    gen = generator(vocabulary + 12)
    rows = 7
    one = torch.zeros(rows, vocabulary, device=DEV)
    one[torch.arange(rows), torch.randint(0, vocabulary, (rows,), generator=gen, device=DEV)] = spread
    some = torch.randint(0, 5, (rows, vocabulary), generator=gen, device=DEV).float() * spread
    for logits in (one, some, some - 3 * spread):
        for k in (1, 3, 70, 200, 300, 1000):
            compare(logits, torch.rand(rows, generator=gen, device=DEV), dict(top_k=ints([k] * rows)))
        compare(logits, torch.rand(rows, generator=gen, device=DEV), dict(top_p=f32([0.37, 0.811, 0.123, 0.59, 0.99, 0.9999, 0.001])))


@pytest.mark.parametrize("temperature", [5e-38, 1e-37, 1e-36])
@pytest.mark.parametrize("vocabulary", [5000, 7001])
def test_borders_at_temperatures_next_to_nothing(temperature, vocabulary):
    """By top_p far down: the many values 24.5 temperatures below the largest are together more than what it leaves out.  The largest is the vocabulary's
    last, so that small random numbers find them.  (The plain form adds so many shares to one or less: each rounding is at most 2^-53.  The border
    by top_p is 2.56e-12 from the next one, which 2^-40 and twice those of up to 7400 values stay below; of more no token could be told.)"""
    gen = generator(vocabulary + 13)
    u = f32([0.0, 1e-9, 1e-8, 3e-8, 4.5e-8, 5.5e-8, 8e-8, 1e-7, 0.5])
    rows = len(u)
    logits = torch.full((rows, vocabulary), -24.5 * temperature, device=DEV)
    logits[:, torch.randint(0, vocabulary - 1, (2,), generator=gen, device=DEV)] = -20.0 * temperature
    logits[:, -1] = 0.0
    given = dict(temperature=torch.full((rows,), temperature, device=DEV), top_p=f32([1 - 2.0 ** -24] * rows))
    compare(logits, u, given, off=vocabulary * 2.0 ** -53, most_near=0.6)


# ---- many infinite values

@pytest.mark.parametrize("vocabulary", [5000, 70001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("infinite", [3, 200, 1100, 3000])
def test_many_infinite_values(vocabulary, dtype, infinite):
    """Each has the same share and the others none, also where they are more than a top_k that is more than a list is made for."""
    gen = generator(vocabulary + infinite)
    rows = 4
    logits = torch.randn(rows, vocabulary, generator=gen, device=DEV) * 2.5
    logits[1] *= 1e37
    logits[2, ::3] = torch.finfo(dtype).max
    logits[3] = logits[3].round()
    logits = logits.to(dtype)
    for r in range(rows):
        logits[r, torch.randperm(vocabulary, generator=gen, device=DEV)[:infinite]] = float("inf")
    for k in (1, 2, 70, 150, 300, 1000, 1024, 2000, 4000):
        compare(logits, torch.rand(rows, generator=gen, device=DEV), dict(top_k=ints([k] * rows)), most_near=0.5)
    for p in (0.37, 0.811):
        compare(logits, torch.rand(rows, generator=gen, device=DEV), dict(top_p=f32([p] * rows)), most_near=0.5)
        compare(logits, torch.rand(rows, generator=gen, device=DEV), dict(top_p=f32([p] * rows), top_k=ints([700] * rows)), most_near=0.5)
    compare(logits, torch.rand(rows, generator=gen, device=DEV), dict(min_p=f32([0.3] * rows)), most_near=0.5)


# ---- caps and temperatures next to nothing

@pytest.mark.parametrize("vocabulary", [4, 100, 5000])
@pytest.mark.parametrize("temperature", [2e-30, 1e-29, 1e-28, 1e-27, 1e-24])
def test_capped_values_next_to_zero(vocabulary, temperature):
    """Values about the smallest normal number, zeros among them, at temperatures of which they are a part that counts: a random number of a half
    falls into the second half of the row, whose shares' sum is larger by (2 * 2e-38 - 3.7e-38) / temperature of a quarter."""
    x = torch.zeros(2, vocabulary, device=DEV)
    quarter = vocabulary // 4
    x[:, quarter:2 * quarter] = 3.7e-38
    x[:, 2 * quarter:] = 2e-38
    x[1] = -x[1]  # (and by as much into the first)
    for cap in (temperature, 30 * temperature):
        for rules in ({}, dict(top_k=ints([vocabulary - 1] * 2))):
            compare(x, f32([0.5, 0.5]), dict(rules, temperature=f32([temperature] * 2)), softcap=cap, most_near=1.0 if temperature > 5e-28 else 0.0)


@pytest.mark.parametrize("vocabulary", [5000, 70001])
@pytest.mark.parametrize("softcap", [30.0, 1e4])
def test_many_infinite_values_capped(vocabulary, softcap):
    """An infinite value is capped to the cap, and ranks before others that are."""
    gen = generator(vocabulary + 14)
    logits = torch.randn(4, vocabulary, generator=gen, device=DEV) * torch.tensor([2.5, 1e37, 40.0, 1e4], device=DEV)[:, None]
    for r, infinite in enumerate((3, 200, 1100, 3000)):
        logits[r, torch.randperm(vocabulary, generator=gen, device=DEV)[:infinite]] = float("inf")
    for rules in ({}, dict(top_k=ints([150] * 4)), dict(top_k=ints([1000] * 4)), dict(top_p=f32([0.37, 0.811, 0.937, 0.123])), dict(min_p=f32([0.3] * 4)),
                  dict(top_k=ints([2000] * 4), top_p=f32([0.37, 0.811, 0.937, 0.123]))):
        compare(logits, torch.rand(4, generator=gen, device=DEV), rules, softcap, off=2 * softcap * 2.0 ** -51, most_near=0.5)


# ---- plans in place

def test_a_plan_in_place_goes_on_from_what_a_trim_returned():
    """The lengths and the count that trim_step made take the place of those that the plan began with: no page is handed out twice."""
    from tests import step_ref
    from tests.test_gpu_step import requests
    rng, lengths, table, free, taken = requests(4, 30, 16, 60, width=20)
    pool, rows, state = step.PagePool(ints(free), ints([taken])), ints(table), ints(lengths)
    plan = step.StepPlan.in_place(state, rows, pool, 300)
    held, first, count = plan.batch, state, pool.taken
    for turn in range(6):
        news = [int(x) for x in rng.integers(0, 10, 30)]
        want = step_ref.plan(lengths, news, table, free, taken, 16, 300)
        assert step.plan_step(state, ints(news), rows, pool, 16, 300, out=plan) is plan
        lengths, taken, table = want[1], want[4], want[5]
        assert state.tolist() == lengths and pool.taken.tolist() == [taken] and rows.tolist() == table and plan.slots.tolist() == want[2]
        assert plan.lengths is state and plan.taken is pool.taken and plan.batch is held and held.lengths is state
        live = [row[i] for row, n in zip(table, lengths) for i in range(-(-n // 16))]
        assert len(set(live)) == len(live)
        if turn % 2 == 0:
            keep = [max(0, n - int(rng.integers(0, 30))) for n in lengths]
            lengths, free, taken = step_ref.trim(lengths, keep, table, free, taken, 16)
            trimmed = step.trim_step(state, ints(keep), rows, pool, 16)
            state, pool.taken = trimmed.lengths, trimmed.taken
    pool.check()
    assert first is not state and count is not pool.taken


def test_a_captured_plan_in_place_keeps_its_tensors():
    pool, table, state, news = step.PagePool.whole(20, DEV), torch.full((2, 5), -1, dtype=torch.int32, device=DEV), ints([0, 0]), ints([1, 20])
    plan = step.StepPlan.in_place(state, table, pool, 30)
    step.plan_step(state, news, table, pool, 16, 30, out=plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.plan_step(state, news, table, pool, 16, 30, out=plan)
    count, pool.taken, other = pool.taken, ints([7]), ints([5, 5])
    step.plan_step(other, news, table, pool, 16, 30, out=plan)
    assert other.tolist() == [6, 25] and pool.taken.item() == 8 and state.tolist() == [1, 20] and plan.batch.lengths is other
    graph.replay()
    assert state.tolist() == [2, 40] and other.tolist() == [6, 25] and pool.taken.item() == 8 and count.item() == 4  # (1 + 2 pages, and one more)
    pool.check()


def test_the_batch_of_a_plan_has_the_plans_tensors():
    pool, table = step.PagePool.whole(20, DEV), torch.full((2, 5), -1, dtype=torch.int32, device=DEV)
    plan = step.plan_step(ints([0, 0]), ints([1, 20]), table, pool, 16, 21)
    batch = plan.batch
    plan.lengths, plan.table = plan.lengths.clone(), plan.table.clone()
    assert plan.batch is batch and batch.lengths is plan.lengths and batch.table is plan.table


# ---- layers

@pytest.mark.parametrize("prompt", [False, True])
def test_a_layer_of_no_rows(prompt):
    from gevva_b200 import attention as attn
    from tests.test_gpu_step import attention_layer
    layer = attention_layer(generator(71))
    pool, table = step.PagePool.whole(8, DEV), torch.full((2, 4), -1, dtype=torch.int32, device=DEV)
    plan = step.plan_step(ints([0, 0]), ints([0, 0]), table, pool, 16, 0)
    hidden = torch.zeros(0, 256, dtype=torch.bfloat16, device=DEV)
    for batch in (plan, plan.batch, attn.PagedBatch(ints([0, 0, 0]), ints([5, 0]), ints([[0], [1]]))):
        assert layer.forward(hidden, batch, prompt).shape == (0, 256)
    pool.check()
    layer.cache.check()


def test_a_stack_with_a_row_without_a_token():
    """The other rows get what they get beside any token, and what the row leaves in the cache is finite."""
    from gevva_b200.synthetic import SyntheticAttention, SyntheticStack
    gen = generator(72)
    stack = SyntheticStack(2, 16, DEV, distinct_experts=False, attention=SyntheticAttention(window=24, whole_every=2, pages=16, page_size=16), vocabulary=1201)
    pool, table, lengths = step.PagePool.whole(16, DEV), torch.full((3, 4), -1, dtype=torch.int32, device=DEV), ints([0, 0, 0])
    u = torch.rand(3, generator=gen, device=DEV)
    got = []
    for middle in (-1, 5):
        plan = step.plan_step(lengths, ints([1, 1, 1]), table, pool, 16, 3)
        got.append(stack.decode(ints([7, middle, 1200]), plan, u, probability=True))
        for layer in stack.attention:
            assert layer.cache.k.isfinite().all() and layer.cache.v.isfinite().all()
    (without, shares), (beside, others) = got
    assert without.tolist() == [beside[0], -1, beside[2]] and shares.tolist() == [others[0], 0, others[2]] and (beside >= 0).all()


@pytest.mark.parametrize("temperature", [5e-38, 1e-37])
def test_borders_of_wide_bins(temperature):
    """At temperatures of which a bin is a part that counts: values at the upper ends of their bins, whose shares' sum is more than their middles say by
    up to exp of half a bin.  The border is just in front of the last of a bin."""
    width = 1.0 / 1.7014118e38  # of the bins in use, at most as many as a number of 32 bits says
    at = torch.arange(1, 86, dtype=torch.float64).repeat_interleave(50)
    row = torch.cat([torch.zeros(1, dtype=torch.float64), -(at - 0.499) * width])
    row = row[torch.randperm(len(row), generator=torch.Generator().manual_seed(3))].float()
    degrees = float(torch.tensor(temperature))
    shares = torch.exp(row.double() / degrees).sort(descending=True).values.cumsum(0)
    bins = torch.arange(24, 64)
    p = shares[50 * bins] / shares[-1] * 0.9995
    for u in (0.97, 0.73, 0.41):
        compare(row.expand(len(bins), -1).to(DEV), f32([u] * len(bins)), dict(temperature=f32([temperature] * len(bins)), top_p=p.float().to(DEV)), off=1e-12)


@pytest.mark.parametrize("vocabulary", [7, 300, 5000])
@pytest.mark.parametrize("size", [1e-31, 1e-35, 1e-38])
def test_capped_values_of_next_to_nothing(vocabulary, size):
    """Logits, cap and temperature that are all below 1e-30: what counts is how large they are to one another.  (Subnormal temperatures are read as they are
    on both sides; softened values are off by 2^-50 of the smaller of cap and value.)"""
    gen = generator(vocabulary + 15)
    for cap in f32([3 * size, 100 * size, 1e-6, 30.0]).tolist():  # (a call's cap is a number of 32 bits)
        logits = torch.randn(5, vocabulary, generator=gen, device=DEV) * 2.5 * size
        for part in (0.1, 1.0, 3.0):
            for rules in ({}, dict(top_k=ints([4] * 5)), dict(top_p=f32([0.83] * 5)), dict(min_p=f32([0.05] * 5))):
                given = dict(rules, temperature=f32([part * size] * 5))
                compare(logits, torch.rand(5, generator=gen, device=DEV), given, cap, off=vocabulary * 2.0 ** -53 + 4 * 12 / part * 2.0 ** -50)


@pytest.mark.parametrize("vocabulary", [7, 300, 5000])
@pytest.mark.parametrize("cap", [4e29, 2e30, 1e31, 1e32])
def test_large_caps(vocabulary, cap):
    """Caps and temperatures far apart from ordinary ones, of which the cap is a few or many."""
    gen = generator(vocabulary + 16)
    cap = f32([cap]).item()
    logits = torch.randn(5, vocabulary, generator=gen, device=DEV) * torch.tensor([0.3, 1.0, 5.0, 30.0, 300.0], device=DEV)[:, None] * cap
    for parts in (1.5, 15.0, 110.0):
        for rules in ({}, dict(top_k=ints([4] * 5)), dict(top_p=f32([0.83] * 5)), dict(top_p=f32([1 - 2.0 ** -23] * 5)), dict(min_p=f32([0.05] * 5))):
            given = dict(rules, temperature=f32([cap / parts] * 5))
            compare(logits, torch.rand(5, generator=gen, device=DEV), given, cap, off=vocabulary * 2.0 ** -53 + parts * 2.0 ** -50, most_near=0.4)


@pytest.mark.parametrize("vocabulary", [1810, 20001])
@pytest.mark.parametrize("temperature", [3e36, 1e38, 3e38])
def test_values_over_the_whole_range(vocabulary, temperature):
    """From the lowest numbers to the largest, further apart than a number of 32 bits says, at temperatures at which all of them have a share."""
    gen = generator(vocabulary + 17)
    rows = 12
    logits = (torch.randn(rows, vocabulary, generator=gen, device=DEV) * 1.4).clamp(-3.3, 3.3) * 1e38
    logits[::3] = (logits[::3] / 4e36).round() * 4e36
    for cap in f32([0.0, 1e38, 3e38]).tolist():
        for _ in range(3):
            given = dict(temperature=f32([temperature] * rows), top_p=torch.rand(rows, generator=gen, device=DEV))
            off = vocabulary * 2.0 ** -53 + 4e38 / temperature * 2.0 ** -50
            compare(logits, torch.rand(rows, generator=gen, device=DEV), given, cap, off=off, most_near=0.4)
            compare(logits, torch.rand(rows, generator=gen, device=DEV), dict(given, top_k=ints([vocabulary // 2] * rows)), cap, off=off, most_near=0.4)
