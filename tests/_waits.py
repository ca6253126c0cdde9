"""Loads on their way through a kernel's listing, along every path of its branches."""
import re

LOADS = ("buffer_load", "global_load", "scratch_load", "flat_load")


def instructions(lines):
    """Lines of llvm-objdump -> [(address, operation, text, branch target or None)]; the first line names the kernel."""
    start, found = int(lines[0].split()[0], 16), []
    for line in lines[1:]:
        text, _, rest = line.partition("//")
        op = text.split()
        if op and rest:
            target = re.search(r"\+0x([0-9a-f]+)>", rest) if op[0].startswith(("s_branch", "s_cbranch")) else None
            found.append((int(rest.split(":")[0], 16), op[0], text.strip(), start + int(target[1], 16) if target else None))
    return found


def barriers_met_early(code, ahead=2):
    """A kernel whose window w of loads to LDS is asked for `ahead` barriers before barrier w, behind which it is read (the first
    `ahead` windows in front of all barriers), four loads a window.  -> ({barriers that a window's own load may reach still on its
    way}, {barriers of windows})

    Loads come back in the order they were asked for, so a wait for n of them leaves the newest n.  Stores are not counted, though
    the hardware counts them: fewer loads may be on their way than this takes for possible, not more."""
    at = {address: i for i, (address, *_) in enumerate(code)}
    first = next(i for i, (_, op, text, _) in enumerate(code) if op.startswith(LOADS) and text.endswith(" lds"))
    # a state: the next instruction; pending loads, the oldest first, as the number of barriers until their data are read (None: not
    # to LDS); loads to LDS since the last barrier; whether a barrier has been met
    todo, seen, early, barriers = [(first, (), 0, False)], set(), set(), set()
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        i, pending, asked, inside = state
        address, op, text, target = code[i]
        if op == "s_endpgm":
            continue
        if op.startswith(LOADS):
            lds = text.endswith(" lds")
            window = (ahead - 1 if inside else asked // 4) if lds else None
            pending, asked = (*pending, window)[-63:], asked + lds
        elif op == "s_waitcnt" and "vmcnt" in text:
            left = int(text.split("vmcnt(")[1].split(")")[0])
            pending = pending[max(len(pending) - left, 0):]
        elif op == "s_barrier":
            if 0 in pending:
                early.add(address)
            if asked:
                assert asked == (4 if inside else 4 * ahead), (hex(address), asked)
                barriers.add(address)
            pending, asked, inside = tuple(w if w is None else w - 1 for w in pending), 0, True
        if target is not None:
            todo.append((at[target], pending, asked, inside))
        if op != "s_branch":
            todo.append((i + 1, pending, asked, inside))
    return early, barriers
