"""The gated delta rule where the sizes of a column's numbers change along a request: both forms against the formula in 64 bits.

What is behind a change of size is measured against its own size, rows chunk by chunk and columns one by one.  The tolerance
is that of test_gpu_delta_rule.py, whose derivation asks for nothing about sizes: a token's errors are units of what the
state holds at that token, and they fade as fast as the state does."""
import pytest
import torch

from test_gpu_delta_rule import CROWD, FEW, MANY, Case, near

pytestmark = pytest.mark.gpu
CHUNK = 32


def check_parts(case, longest, cuts):
    """Rows between two of `cuts` by themselves, from the last cut on by chunks and by columns, and the states by columns."""
    (out, state), (want_out, want_state) = case.run(longest), case.want()
    assert torch.isfinite(out).all() and torch.isfinite(state).all()
    edges = [0] + cuts + list(range(cuts[-1] // CHUNK * CHUNK + CHUNK, case.tokens, CHUNK)) + [case.tokens]
    for a, b in zip(edges, edges[1:]):
        near(out[a:b], want_out[a:b])
    for col in range(case.heads * case.vdim):
        near(out[cuts[-1]:, col], want_out[cuts[-1]:, col])
    size = case.heads * case.dim * case.vdim
    got, want = (s[case.slots[0], :size].view(case.heads, case.dim, case.vdim) for s in (state, want_state))
    for head in range(case.heads):
        for col in range(case.vdim):
            near(got[head, :, col], want[head, :, col])


def values(case):
    return case.qkv[:, case.offs[2]:case.offs[2] + case.heads * case.vdim]


FORMS = pytest.mark.parametrize("longest", [FEW, MANY, CROWD])
TYPES = pytest.mark.parametrize("dtype,dim,vdim", [(torch.bfloat16, 128, 64), (torch.float32, 64, 48)])


@FORMS
@TYPES
@pytest.mark.parametrize("ratio", [1e2, 1e3, 1e4, 1e5, 1e6, 1e8])
def test_a_large_state_that_is_forgotten(ratio, dtype, dim, vdim, longest):
    case = Case([512], 2, 1, dim, vdim, dtype)
    case.state *= 10 * ratio
    case.decay[3] = -1e4
    check_parts(case, longest, [3])


@FORMS
@TYPES
@pytest.mark.parametrize("ratio", [1e2, 1e3, 1e4, 1e5, 1e6, 1e8])
def test_a_large_first_value_that_is_forgotten(ratio, dtype, dim, vdim, longest):
    case = Case([512], 2, 1, dim, vdim, dtype)
    values(case)[0] *= ratio
    case.decay[3] = -1e4
    check_parts(case, longest, [3])


@FORMS
@TYPES
@pytest.mark.parametrize("ratio", [1e4, 1e8])
def test_a_large_value_that_fades(ratio, dtype, dim, vdim, longest):
    """Half a unit of log-decay a token: the value is of the others' size again some 20 or 40 tokens later."""
    case = Case([300], 2, 1, dim, vdim, dtype)
    values(case)[40] *= ratio
    case.decay.fill_(-0.5)
    check_parts(case, longest, [40, 50, 64, 80, 90])


@FORMS
@TYPES
@pytest.mark.parametrize("ratio", [1e4, 1e6, 1e9])
def test_a_large_value_changes_no_token_before_it(ratio, dtype, dim, vdim, longest):
    case = Case([100], 2, 1, dim, vdim, dtype)
    values(case)[90] *= ratio
    check_parts(case, longest, [64, 70, 80, 90])


@FORMS
@TYPES
@pytest.mark.parametrize("ratio", [1e5, 1e9])
def test_values_that_fall_behind_the_first_chunk(ratio, dtype, dim, vdim, longest):
    case = Case([700], 2, 1, dim, vdim, dtype)
    values(case)[:CHUNK] *= ratio
    case.decay.clamp_(max=-0.1)
    check_parts(case, longest, [32])


@FORMS
@TYPES
def test_values_that_fall_all_the_time(dtype, dim, vdim, longest):
    """Every chunk's values are a fiftieth of those before, and a token forgets a fifth of the state."""
    case = Case([260], 2, 1, dim, vdim, dtype)
    values(case).mul_(50.0 ** -(torch.arange(case.tokens, device="cuda") // CHUNK)[:, None])
    case.decay.fill_(-0.22)
    check_parts(case, longest, [32])


@FORMS
@TYPES
def test_steps_of_almost_nothing(dtype, dim, vdim, longest):
    """Values of which next to nothing is stored, beside a state of that size."""
    case = Case([90], 2, 1, dim, vdim, dtype)
    case.beta *= 1e-8
    case.state *= 1e-7
    check_parts(case, longest, [32])


@FORMS
@TYPES
def test_a_small_state_that_is_only_read(dtype, dim, vdim, longest):
    """Nothing is stored in front of token 20, where a large value comes."""
    case = Case([70], 2, 1, dim, vdim, dtype)
    case.state *= 1e-6
    case.beta[:20] = 0.0
    values(case)[20] *= 1e4
    check_parts(case, longest, [20, 32])


@FORMS
@pytest.mark.parametrize("v_scale", [1e-33, 1e33])
def test_sizes_near_the_ends_of_the_type(v_scale, longest):
    check_parts(Case([70], 2, 1, 64, 48, torch.float32, v_scale=v_scale), longest, [32])


@FORMS
def test_one_column_among_others(longest):
    """Only one column has a large first value: its neighbours of the same warp as exactly as ever."""
    case = Case([100], 1, 1, 64, 32, torch.float32)
    values(case)[0, 13] *= 1e7
    case.decay[3] = -1e4
    check_parts(case, longest, [3])


@FORMS
@TYPES
def test_columns_of_zeros(dtype, dim, vdim, longest):
    """Columns whose values are zero for a while, over a state of zeros: zero outputs as long as both are, and right ones when
    values come, of whatever size."""
    case = Case([300], 2, 1, dim, vdim, dtype)
    v = values(case)
    case.state.zero_()
    v[:, 5] = 0.0
    v[:150, 9] = 0.0
    v[:100, 16:19] = 0.0
    v[100:, 16], v[100:, 17] = v[100:, 16] * 1e-28, v[100:, 17] * 1e9
    v[40:260] *= (torch.arange(case.heads * vdim, device="cuda") != 20)      # zeros in between
    v[:64, vdim:] = 0.0                                        # the second head's first chunks
    case.beta[130:140] = 0.0
    check_parts(case, longest, [32, 64])
    out, state = case.run(longest)
    assert (out[:, 5] == 0).all() and (out[:100, 16:19] == 0).all() and (out[:64, vdim:] == 0).all()


@FORMS
def test_values_that_come_to_columns_of_zeros_without_a_step(longest):
    """Nothing is stored (beta = 0) of values over a state of zeros: the outputs are zero."""
    case = Case([200], 2, 1, 64, 48, torch.float32)
    case.state.zero_()
    v = values(case)
    v[:64] = 0.0
    case.beta[:130] = 0.0
    out, state = case.run(longest)
    want_out, want_state = case.want()
    assert (out[:130] == 0).all()
    near(out, want_out)
    near(state, want_state)
