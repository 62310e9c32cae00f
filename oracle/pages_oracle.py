"""Oracle of pages: the rules of allocate_pages and release_pages one request, page and token at a time, on lists."""


def allocate(table, seqlens, new_lens, free_pages, num_free, page, num_tokens):
    """(table, slots, cu_seqlens, seqlens, num_free) after the call; the arguments are left as they are."""
    table = [list(row) for row in table]
    cols = len(table[0]) if table else 0
    stack = list(free_pages[:min(max(num_free, 0), len(free_pages))])
    wanted = 0  # pages of this request and those before it, refused ones for want of pages among them
    available = len(stack)
    slots, cu, lens, token = [-1] * num_tokens, [0], [], 0
    for b, (n, m) in enumerate(zip(seqlens, new_lens)):
        n, m = max(n, 0), max(m, 0)
        begin, token = token, token + m
        cu.append(min(token, num_tokens))
        need = -(-(n + m) // page) - -(-n // page)
        room = n + m <= min(cols * page, 2 ** 31 - 1) and token <= num_tokens
        if room:
            wanted += need
        if not room or (need > 0 and wanted > available):
            lens.append(n)
            continue
        lens.append(n + m)
        for j in range(need):
            table[b][-(-n // page) + j] = stack.pop()
        for i in range(m):
            entry = table[b][(n + i) // page]
            slots[begin + i] = entry * page + (n + i) % page if entry >= 0 else -1
    return table, slots, cu, lens, len(stack)


def release(table, seqlens, done, free_pages, num_free, page, keep_lens=None):
    """(free_pages, seqlens, num_free) after the call."""
    pages = list(free_pages)
    cols = len(table[0]) if table else 0
    count = min(max(num_free, 0), len(pages))
    room, wanted, lens = len(pages) - count, 0, []
    for b, n in enumerate(seqlens):
        n = max(n, 0)
        if not done[b]:
            lens.append(n)
            continue
        given = range(0 if keep_lens is None else max(keep_lens[b], 0) // page, min(-(-n // page), cols))
        wanted += len(given)
        if len(given) and wanted > room:
            lens.append(n)
            continue
        lens.append(0)
        for col in given:
            pages[count] = table[b][col]
            count += 1
    return pages, lens, count
