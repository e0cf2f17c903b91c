"""What moe_layer's streaming kernels make of a call: runs of units a workgroup and passes over them, from the launch that describe() names
and the tokens of each expert."""
import libr3d_amd as R


def launch(ops):
    """describe()'s numbers; the call needs no scratch to be described."""
    scratch = ops.args.scratch, ops.args.scratch_bytes
    ops.args.scratch, ops.args.scratch_bytes = 1 << 20, R.row_scratch_bytes("moe_layer", ops)
    rc, text = R.describe("moe_layer", ops)
    ops.args.scratch, ops.args.scratch_bytes = scratch
    assert rc == R.RAD_OK, text
    return {k: int(v) for k, _, v in (w.partition("=") for w in text.split()) if v.isdigit()}


def passes(tokens, units, width, rows, cap=1 << 30, blocks=256):
    """Of a kernel with `units` units a job: (the most passes a workgroup takes, whether a pass begins inside a job, whether one
    ends at `cap` units)."""
    job, slot = [], 0
    for n in tokens:
        for at in range(0, n, width):
            job.append((slot + at, min(width, n - at)))
        slot += n
    total = len(job) * units
    most, inside, capped = 0, False, False
    for g in range(blocks):
        u, end_of_run = total * g // blocks, total * (g + 1) // blocks
        count = 0
        while u < end_of_run:
            count += 1
            inside |= count > 1 and u % units != 0
            j = u // units
            base, end = job[j][0], u
            while end < end_of_run and end - u < cap:
                if job[j][0] + job[j][1] - base > rows:
                    break
                end = min((j + 1) * units, end_of_run)
                j += 1
            if end - u > cap:
                end, capped = u + cap, True
            u = end
        most = max(most, count)
    return most, inside, capped
